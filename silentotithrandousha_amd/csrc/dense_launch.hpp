// Tile shapes of the dense products and the rule that picks one.
#pragma once
#include "dense_gemm.hpp"

namespace moe {

// X(name, rows, columns, wavefronts along each, LDS slots, workgroups of a CU, TFLOP/s of the device full of
// them). The rates are those of 2880 k values (loss over 201088 rows, 512 tokens and more).
#define MOE_DENSE_TILES(X)                   \
  X(288x256, 288, 256, 2, 4, 2, 1, 1180.0)   \
  X(256x256, 256, 256, 2, 4, 2, 1, 1290.0)   \
  X(192x256, 192, 256, 2, 4, 2, 1, 1190.0)   \
  X(128x128, 128, 128, 2, 2, 2, 2, 1000.0)    \
  X(128x64, 128, 64, 2, 2, 3, 2, 800.0)      \
  X(64x64, 64, 64, 2, 2, 4, 2, 600.0)        \
  X(32x64, 32, 64, 2, 2, 6, 2, 430.0)        \
  X(32x32, 32, 32, 2, 2, 8, 2, 300.0)        \
  X(32x16, 32, 16, 2, 1, 8, 3, 220.0)        \
  X(128x16, 128, 16, 4, 1, 4, 2, 220.0)      \
  X(64x16, 64, 16, 4, 1, 8, 2, 210.0)        \
  X(16x16, 16, 16, 1, 1, 16, 2, 110.0)

enum DenseTileShape {
#define X(name, bm, bn, wm, wn, ns, wgs, rate) TILE_##name,
  MOE_DENSE_TILES(X)
#undef X
};

DenseTileShape dense_tile(const DenseShape &s, const DenseArgs &a);

template <bool AT, bool BT, int EPI>
hipError_t launch_dense_shape(const DenseArgs &a, hipStream_t st) {
  switch (dense_tile(DenseShape{AT, BT, (DenseEpi)EPI}, a)) {
#define X(name, bm, bn, wm, wn, ns, wgs, rate) \
  case TILE_##name:                 \
    if constexpr ((AT && EPI == DENSE_STORE) || bm <= 256)  \
      return launch_dense_as<bm, bn, wm, wn, ns, AT, BT, EPI>(a, st); \
    break;
    MOE_DENSE_TILES(X)
#undef X
  }
  return hipErrorInvalidValue;
}

struct DenseTileDims {
  int bm, bn, wm, wn, ns, wgs;
  double rate;
};
constexpr DenseTileDims kDenseTiles[] = {
#define X(name, bm, bn, wm, wn, ns, wgs, rate) {bm, bn, wm, wn, ns, wgs, rate},
    MOE_DENSE_TILES(X)
#undef X
};

bool dense_few_fits(const DenseShape &s, const DenseArgs &a);
hipError_t launch_dense_few(const DenseShape &s, const DenseArgs &a, hipStream_t st);
hipError_t launch_dense_nt(const DenseShape &s, const DenseArgs &a, hipStream_t st);
hipError_t launch_dense_tn(const DenseShape &s, const DenseArgs &a, hipStream_t st);

}  // namespace moe
