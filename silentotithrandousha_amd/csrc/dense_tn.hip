// Dense products with a transposed operand: the gradients of activations (A transposed) and of
// weights (both).
#include "dense_gemm.hpp"
#include "dense_launch.hpp"

namespace moe {
hipError_t launch_dense_tn(const DenseShape &s, const DenseArgs &a, hipStream_t st) {
  if (s.bt) return s.epi == DENSE_STORE ? launch_dense_shape<true, true, DENSE_STORE>(a, st) : hipErrorInvalidValue;
  switch (s.epi) {
    case DENSE_STORE: return launch_dense_shape<true, false, DENSE_STORE>(a, st);
    case DENSE_DGATE: return launch_dense_shape<true, false, DENSE_DGATE>(a, st);
    default: return hipErrorInvalidValue;
  }
}
}  // namespace moe
