// Dense products with both operands K-contiguous: the forward projections and the logits.
#include "dense_gemm.hpp"
#include "dense_launch.hpp"

namespace moe {
hipError_t launch_dense_nt(const DenseShape &s, const DenseArgs &a, hipStream_t st) {
  switch (s.epi) {
    case DENSE_STORE: return launch_dense_shape<false, false, DENSE_STORE>(a, st);
    case DENSE_GATE: return launch_dense_shape<false, false, DENSE_GATE>(a, st);
    case DENSE_STATS: return launch_dense_shape<false, false, DENSE_STATS>(a, st);
    case DENSE_DLOGITS: return launch_dense_shape<false, false, DENSE_DLOGITS>(a, st);
    default: return hipErrorInvalidValue;
  }
}
}  // namespace moe
