// Tile shapes of the dense products and the rule that picks one.
#pragma once
#include "dense_gemm.hpp"

namespace moe {

enum DenseTileShape { TILE_128x16, TILE_128x128 };

inline DenseTileShape dense_tile(const DenseArgs &a) { return a.N <= 16 ? TILE_128x16 : TILE_128x128; }

template <bool AT, bool BT, int EPI>
hipError_t launch_dense_shape(const DenseArgs &a, hipStream_t st) {
  switch (dense_tile(a)) {
    case TILE_128x16: return launch_dense_as<128, 16, 4, 1, AT, BT, EPI>(a, st);
    default: return launch_dense_as<128, 128, 2, 2, AT, BT, EPI>(a, st);
  }
}

// rows and columns of a tile, and its wavefronts along each
struct DenseTileDims {
  int bm, bn, wm, wn;
};
inline DenseTileDims dense_tile_dims(DenseTileShape s) {
  switch (s) {
    case TILE_128x16: return {128, 16, 4, 1};
    default: return {128, 128, 2, 2};
  }
}

hipError_t launch_dense_nt(const DenseShape &s, const DenseArgs &a, hipStream_t st);
hipError_t launch_dense_tn(const DenseShape &s, const DenseArgs &a, hipStream_t st);

}  // namespace moe
