// Where the values of a dense product's tiles lie, in memory and in LDS: plain arithmetic, for the kernels and for
// checks on the host.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dense_plan.hpp"

namespace moe {

#define MOE_INDEX static __host__ __device__ __forceinline__

// One operand's tile: R rows (of M or N) x 64 k, W wavefronts loading it. TR: the operand is stored with its k as rows.
template <int R, int W, bool TR>
struct DenseIndex {
  static constexpr int kBytes = R * 128;
  static constexpr int kDmas = R / 8;                 // LDS-DMAs of 1 KB
  static constexpr int kLoads = (kDmas + W - 1) / W;  // per wavefront; past the last one again (the same bytes)
  static constexpr int kPairs = R / 16;               // 32-byte pieces of a transposed row

  // Transposed: piece of a row that holds the logical piece q in row k. The transposing load's 16 lanes
  // take 4 rows k: their pieces go to different banks. (Only within groups of 4 pieces, so that the
  // fragments of 16 rows lie at 4 addresses and constant distances from them.)
  MOE_INDEX int piece(int q, int k) {
    const int mask = kPairs >= 4 ? ((q | 3) < kPairs ? 3 : 0) : kPairs >= 2 ? 1 : 0;
    return q ^ (k & mask);
  }

  MOE_INDEX int dma(int i, int wave) {
    const int d = i * W + wave;
    return kDmas % W == 0 ? d : d % kDmas;
  }
  // chunk c of the tile: the first k of its values if K-contiguous, its row's k if transposed
  MOE_INDEX int k_of(int c) { return TR ? c / (R / 8) : ((c & 7) ^ ((c >> 3) & 7)) * 8; }
  // Byte offset of a lane's 16 bytes of load i from the tile's base. rows: valid rows from the tile's first; ld: bytes
  // between stored rows; after every `skip_every` rows (of planes stacked from every other slot) as many are left
  // out, none if it is 0.
  MOE_INDEX uint32_t offset(int i, int wave, int lane, int rows, uint32_t ld, int skip_every) {
    const int c = dma(i, wave) * 64 + lane, k = k_of(c);
    if constexpr (!TR) {
      int row = (c >> 3) < rows - 1 ? c >> 3 : rows - 1;
      if (skip_every) row += row / skip_every * skip_every;
      return (uint32_t)row * ld + k * 2;
    } else {
      const int pos = c % (R / 8);
      int col = piece(pos >> 1, k) * 16 + (pos & 1) * 8;  // the permutation is its own inverse
      if (col >= rows) col = 0;
      return (uint32_t)k * ld + col * 2;
    }
  }
  // of a step with fewer k values left than its 64: how far that offset goes back to a valid place (what is loaded past
  // them is cleared)
  MOE_INDEX uint32_t behind(int i, int wave, int lane, uint32_t ld, int left) {
    const int k = k_of(dma(i, wave) * 64 + lane);
    return k < left ? 0u : TR ? (uint32_t)(k - (left - 1)) * ld : (uint32_t)k * 2;
  }
  // Where a lane's MFMA operand lies in the step at lds, 16 rows from row0, half h: its 16 bytes, or (transposed) the
  // 8 bytes of its first and second 4 k values that the transposing load reads. (Added to the address one by one: as
  // one offset the main loop computed more of them.)
  MOE_INDEX const uint8_t *frag_at(const uint8_t *lds, int row0, int h, int lane, int part) {
    if constexpr (!TR) {
      const int row = row0 + (lane & 15), ch = h * 4 + (lane >> 4);
      return lds + row * 128 + ((ch ^ (row & 7)) << 4);
    } else {
      const int i = lane & 15, k = (lane >> 4) * 8 + (i >> 2) + 4 * part;
      return lds + (h * kDenseHalf + k) * (R * 2) + piece(row0 >> 4, k) * 32 + (i & 3) * 8;
    }
  }
};

// The tile of workgroup b: 8 XCDs take the workgroups in turn, so each gets a contiguous share of the
// order; in it, 8 tiles along n, then along m, so that the 32 workgroups of an XCD share the rows of
// about 4 x 8 tiles in its L2.
MOE_INDEX void dense_tile_of(int b, int tiles_m, int tiles_n, int &tm, int &tn) {
  const int total = tiles_m * tiles_n, x = b & 7, q = total >> 3, r = total & 7;
  const int t = x * q + (x < r ? x : r) + (b >> 3);
  const int group = t / (tiles_m * 8), n0 = group * 8, width = tiles_n - n0 < 8 ? tiles_n - n0 : 8, in = t - group * tiles_m * 8;
  tm = in / width;
  tn = n0 + in % width;
}

#undef MOE_INDEX

}  // namespace moe
