// The launch of a tile shape that the plan took.
#pragma once
#include "dense_gemm.hpp"
#include "dense_plan.hpp"

namespace moe {

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
hipError_t launch_dense_few(const DenseShape &s, const DenseArgs &a, hipStream_t st);
hipError_t launch_dense_nt(const DenseShape &s, const DenseArgs &a, hipStream_t st);
hipError_t launch_dense_tn(const DenseShape &s, const DenseArgs &a, hipStream_t st);

}  // namespace moe
