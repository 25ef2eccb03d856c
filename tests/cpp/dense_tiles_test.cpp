// The index arithmetic of the dense products' tiles (csrc/dense_index.hpp, the code that the kernels run) replayed on the
// host for every tile shape of the plan and of both operands' layouts: every LDS-DMA reads inside the operand, and the
// fragments read back from LDS are the rows and k values that the product needs, zeros past K.
//   dense_tiles_test            all of it; prints the shapes
//   dense_tiles_test clamp      the same without the last step's clamp: must find a read outside
//   dense_tiles_test pieces     the same with the pieces of a transposed row not permuted back: must find a wrong value
#include <cstdio>
#include <cstring>
#include <set>
#include <string>
#include <tuple>
#include <vector>

#include "../../silentotithrandousha_amd/csrc/dense_index.hpp"

using namespace moe;

static bool g_no_clamp, g_no_pieces;
static long g_outside, g_wrong, g_checked;

// One operand's tile of R rows loaded by W wavefronts: `rows_all` rows of K values, from row r0 and value k0.
// `skip`: the rows are three planes of `skip` rows each, in every other slot.
template <int R, int W, bool TR>
void step(const std::vector<float> &mem, size_t ld, int rows_all, int K, int r0, int k0, int skip) {
  using At = DenseIndex<R, W, TR>;
  const size_t base = TR ? (size_t)k0 * ld + r0 : (size_t)r0 * ld + k0;
  const int left = K - k0, rows = rows_all - r0;
  std::vector<float> lds(R * kDenseStep, -1.0f);  // (2 bytes a value there)
  static const uint8_t first[R * 128] = {};  // for its addresses
  for (int wave = 0; wave < W; wave++)
    for (int i = 0; i < At::kLoads; i++)
      for (int lane = 0; lane < 64; lane++) {
        uint32_t off = At::offset(i, wave, lane, rows, (uint32_t)ld * 2, skip);
        if (left < kDenseStep && !g_no_clamp) off -= At::behind(i, wave, lane, (uint32_t)ld * 2, left);
        const size_t at = base + off / 2;
        if (off % 16 || at + 8 > mem.size()) {
          g_outside++;
          continue;
        }
        memcpy(&lds[At::dma(i, wave) * 512 + lane * 8], &mem[at], 8 * sizeof(float));
      }
  for (float v : lds) g_outside += v == -1.0f;  // a chunk that no wavefront loaded
  if (left < kDenseStep)
    for (int c = 0; c < R * 8; c++)
      if (At::k_of(c) >= left) memset(&lds[c * 8], 0, 8 * sizeof(float));
  for (int row0 = 0; row0 < R; row0 += 16)
    for (int h = 0; h < 2; h++)
      for (int lane = 0; lane < 64; lane++) {
        float got[8];
        if (!TR) {
          memcpy(got, &lds[(At::frag_at(first, row0, h, lane, 0) - first) / 2], sizeof(got));
        } else {
          for (int part = 0; part < 2; part++)
            for (int j = 0; j < 4; j++) {  // lane l gets element l % 4 of the lane 4 j + l / 4 of its 16
              const int src = (lane & 48) + j * 4 + ((lane & 15) >> 2);
              int at = (int)(At::frag_at(first, row0, h, src, part) - first);
              if (g_no_pieces) at += 32 * ((row0 >> 4) - At::piece(row0 >> 4, at / (R * 2)));
              got[part * 4 + j] = lds[at / 2 + (lane & 3)];
            }
        }
        const int r = r0 + row0 + (lane & 15), k = k0 + h * kDenseHalf + (lane >> 4) * 8;
        if (r >= rows_all) continue;
        // (K-contiguous values between K and its next multiple of 8 are the operand's own)
        const int top = TR ? K : (int)ld;
        const size_t stored = skip ? (size_t)(r / skip * 2 * skip + r % skip) : (size_t)r;
        for (int j = 0; j < 8; j++) {
          const float want = k + j >= top ? 0.0f : TR ? mem[(size_t)(k + j) * ld + r] : mem[stored * ld + k + j];
          g_wrong += got[j] != want;
          g_checked++;
        }
      }
}

template <int R, int W, bool TR>
void operand() {
  static std::set<std::tuple<int, int, bool>> done;
  if (!done.insert({R, W, TR}).second) return;
  printf("%d %d %d\n", R, W, TR);
  unsigned seed = 1;
  auto fill = [&](std::vector<float> &m) {
    for (float &v : m) v = (float)((seed = seed * 1664525u + 1013904223u) >> 9) + 1.0f;
  };
  for (int rows : {1, 7, 8, R - 3, R, R + 5, 2 * R + 9})
    for (int K : {1, 8, 31, 32, 56, 64, 72, 130}) {
      const size_t ld = ((TR ? rows : K) + 7) / 8 * 8;
      std::vector<float> mem((TR ? K : rows) * ld);
      fill(mem);
      for (int r0 = 0; r0 < rows; r0 += R)
        for (int k0 = 0; k0 < K; k0 += kDenseStep) step<R, W, TR>(mem, ld, rows, K, r0, k0, 0);
    }
  if (!TR && R <= 64)  // stacked planes in every other slot (the right operand's slots 1, 3, 5)
    for (int n : {1, 2, 5, 10, 21})
      if (3 * n <= R)
        for (int K : {8, 40, 130}) {
          const size_t ld = (K + 7) / 8 * 8;
          std::vector<float> mem(5 * n * ld);
          fill(mem);
          for (int k0 = 0; k0 < K; k0 += kDenseStep) step<R, W, false>(mem, ld, 3 * n, K, 0, k0, n);
        }
}

int main(int argc, char **argv) {
  g_no_clamp = argc > 1 && std::string(argv[1]) == "clamp";
  g_no_pieces = argc > 1 && std::string(argv[1]) == "pieces";
#define X(bm, bn, wm, wn, ns, planes, wgs, rate) \
  operand<bm, wm * wn, false>();                 \
  operand<bm, wm * wn, true>();                  \
  operand<bn, wm * wn, false>();                 \
  operand<bn, wm * wn, true>();
  MOE_DENSE_TILES(X)
#undef X
  long twice = 0;
  for (auto t : {std::pair<int, int>{1, 1}, {3, 2}, {15, 16}, {1048, 3}, {7, 9}, {23, 17}, {2, 100}, {8, 8}}) {
    std::set<std::pair<int, int>> seen;
    for (int b = 0; b < t.first * t.second; b++) {
      int m, n;
      dense_tile_of(b, t.first, t.second, m, n);
      if (m < 0 || n < 0 || m >= t.first || n >= t.second || !seen.insert({m, n}).second) twice++;
    }
  }
  printf("checked %ld outside %ld wrong %ld tiles %ld\n", g_checked, g_outside, g_wrong, twice);
  return g_outside ? 3 : g_wrong ? 4 : twice ? 5 : 0;
}
