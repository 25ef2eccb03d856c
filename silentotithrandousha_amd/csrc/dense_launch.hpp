// Tile shapes of the dense products and the rule that picks one.
#pragma once
#include "dense_gemm.hpp"

namespace moe {

// X(rows, columns, wavefronts along each, LDS slots, B's planes, workgroups of a CU, TFLOP/s of the device
// full of them, planes counted). The rates are those of 2880 k values (loss over 201088 rows, 512 tokens and
// more), with planes those of 2048 (loss of 100 and 333 rows over 50257).
#define MOE_DENSE_TILES(X)            \
  X(288, 256, 2, 4, 2, 1, 1, 1180.0)  \
  X(256, 256, 2, 4, 2, 1, 1, 1290.0)  \
  X(192, 256, 2, 4, 2, 1, 1, 1190.0)  \
  X(128, 128, 2, 2, 2, 1, 2, 1000.0)  \
  X(128, 64, 2, 2, 3, 1, 2, 800.0)    \
  X(64, 64, 2, 2, 4, 1, 2, 600.0)     \
  X(32, 64, 2, 2, 6, 1, 2, 430.0)     \
  X(32, 32, 2, 2, 8, 1, 2, 300.0)     \
  X(32, 16, 2, 1, 8, 1, 3, 220.0)     \
  X(128, 16, 4, 1, 4, 1, 2, 220.0)    \
  X(64, 16, 4, 1, 8, 1, 2, 210.0)     \
  X(16, 16, 1, 1, 16, 1, 2, 110.0)    \
  X(256, 128, 4, 2, 2, 3, 1, 1280.0)  \
  X(128, 128, 2, 4, 2, 3, 1, 1150.0)  \
  X(128, 64, 2, 2, 2, 3, 2, 1200.0)   \
  X(64, 64, 2, 2, 2, 3, 2, 980.0)     \
  X(64, 32, 2, 2, 4, 3, 2, 780.0)     \
  X(32, 32, 2, 2, 5, 3, 2, 480.0)

struct DenseTileDims {
  int bm, bn, wm, wn, ns, planes, wgs;
  double rate;
};
constexpr DenseTileDims kDenseTiles[] = {
#define X(bm, bn, wm, wn, ns, planes, wgs, rate) {bm, bn, wm, wn, ns, planes, wgs, rate},
    MOE_DENSE_TILES(X)
#undef X
};
constexpr int kDenseTileCount = sizeof(kDenseTiles) / sizeof(kDenseTiles[0]);

int dense_tile(const DenseShape &s, const DenseArgs &a);  // index of the tile that the plan takes

template <int I, bool AT, bool BT, int EPI>
hipError_t launch_dense_tile(int tile, const DenseArgs &a, hipStream_t st) {
  if constexpr (I < kDenseTileCount) {
    constexpr DenseTileDims d = kDenseTiles[I];
    if constexpr (((AT && EPI == DENSE_STORE) || d.bm <= 256) && !(BT && d.planes > 1))
      if (tile == I) return launch_dense_as<d.bm, d.bn, d.wm, d.wn, d.ns, d.planes, AT, BT, EPI>(a, st);
    return launch_dense_tile<I + 1, AT, BT, EPI>(tile, a, st);
  }
  return hipErrorInvalidValue;
}
template <bool AT, bool BT, int EPI>
hipError_t launch_dense_shape(const DenseArgs &a, hipStream_t st) {
  return launch_dense_tile<0, AT, BT, EPI>(dense_tile(DenseShape{AT, BT, (DenseEpi)EPI}, a), a, st);
}

template <int I>
hipError_t launch_dense_pair_tile(int tile, const DenseArgs &a, const DenseArgs &b, hipStream_t st) {
  if constexpr (I < kDenseTileCount) {
    constexpr DenseTileDims d = kDenseTiles[I];
    if constexpr (d.planes == 1)
      if (tile == I) return launch_dense_pair_as<d.bm, d.bn, d.wm, d.wn, d.ns>(a, b, st);
    return launch_dense_pair_tile<I + 1>(tile, a, b, st);
  }
  return hipErrorInvalidValue;
}
hipError_t launch_dense_tt_pair(int tile, const DenseArgs &a, const DenseArgs &b, hipStream_t st);
bool dense_few_fits(const DenseShape &s, const DenseArgs &a);
hipError_t launch_dense_few(const DenseShape &s, const DenseArgs &a, hipStream_t st);
hipError_t launch_dense_nt(const DenseShape &s, const DenseArgs &a, hipStream_t st);
hipError_t launch_dense_tn(const DenseShape &s, const DenseArgs &a, hipStream_t st);

}  // namespace moe
