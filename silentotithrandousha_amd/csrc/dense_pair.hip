// Pairs of weight gradients over the same rows in one launch.
#include "dense_gemm.hpp"
#include "dense_launch.hpp"

namespace moe {
hipError_t launch_dense_tt_pair(int tile, const DenseArgs &a, const DenseArgs &b, hipStream_t st) {
  return launch_dense_pair_tile<0>(tile, a, b, st);
}
}  // namespace moe
