// Rows quantised to MXFP4: E2M1 codes with one E8M0 scale per 32 values, in the checkpoint's layout.
//
// e = floor(log2 max |x|) - 2, at least -126: the largest value of a block comes to lie in [4, 8), codes are x 2^-e
// rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code, at most 6.
#include <algorithm>

#include "act8.hpp"
#include "serve.hpp"

namespace moe {
namespace {

// v of the lane whose number differs in bit 0 (1) of the lane's within a quad
template <int XOR>
__device__ __forceinline__ float quad_xor(float v) {
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), XOR == 1 ? 0xB1 : 0x4E, 0xF, 0xF, true));
}

// Four lanes a block of 32 values (which leave together).
template <class S>
__global__ __launch_bounds__(256) void k_mx4_quantize(const S *x, size_t blocks, uint8_t *codes, uint8_t *scales) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i / 4 < blocks; i += (size_t)gridDim.x * 256) {
    float v[8];
    act8_load(x + i * 8, v);
    uint32_t m = 0;  // the largest magnitude's bits: above those of infinity if there is a NaN
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    m = max(m, __float_as_uint(quad_xor<1>(__uint_as_float(m))));
    m = max(m, __float_as_uint(quad_xor<2>(__uint_as_float(m))));
    const bool bad = m >= 0x7F800000u;
    const int byte = max((int)(m >> 23) - 2, 1), e = byte - 127;  // (subnormal: 2^-126, too)
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, ldexpf(v[0], -e), ldexpf(v[1], -e), 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, ldexpf(v[2], -e), ldexpf(v[3], -e), 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, ldexpf(v[4], -e), ldexpf(v[5], -e), 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, ldexpf(v[6], -e), ldexpf(v[7], -e), 1.0f, 3);
    *(uint32_t *)(codes + i * 4) = bad ? 0u : w;
    if (i % 4 == 0) scales[i / 4] = (uint8_t)(bad ? 255 : byte);
  }
}

}  // namespace

hipError_t launch_mx4_quantize(const void *x, bool bf16, size_t n, size_t cols, uint8_t *blocks, uint8_t *scales, hipStream_t s) {
  const size_t nb = n * cols / 32;
  if (!nb) return hipSuccess;
  if (cols % 32) return hipErrorInvalidValue;
  // (a launch has less than 2^32 threads)
  const unsigned grid = (unsigned)std::min<size_t>((nb * 4 + 255) / 256, (size_t)1 << 23);
  return bf16 ? launch_own(k_mx4_quantize<uint16_t>, grid, 256, 0, s, (const uint16_t *)x, nb, blocks, scales)
              : launch_own(k_mx4_quantize<float>, grid, 256, 0, s, (const float *)x, nb, blocks, scales);
}

}  // namespace moe
