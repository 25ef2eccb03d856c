// Rows quantised to MXFP4: E2M1 codes with one E8M0 scale per 32 values, in the checkpoint's layout; and such rows read back.
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

// Four lanes a block of 32 values (which leave together): a lane reads 16 bytes of bf16, or 32 of f32, and writes 4. Bound by memory:
// 23040 x 2880 bf16 (133 MB read, 35 written) take 25 us, 6.7 TB/s; one row 1.9 us, the latency of its loads.
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

// The values of MXFP4 rows, as the reference decodes them (weights.rs:350-371): a code's value times f32_from_bits(byte << 23),
// so that byte 0 is 0 and byte 255 infinity. A thread takes 4 values and 4 further on, so that a
// wavefront's stores lie side by side; bound by the bytes written (one thread a block, whose stores lay 128 bytes apart, took 100 us
// for 23040 x 2880; this 45).
__global__ __launch_bounds__(256) void k_dequant_hf(const uint16_t *codes, const uint8_t *scales, size_t n, f32x4 *out) {
  for (size_t i = (size_t)blockIdx.x * 512 + threadIdx.x; i < n; i += (size_t)gridDim.x * 512) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const size_t k = i + 256 * h;
      if (k >= n) break;
      const uint32_t w = codes[k];
      const float sc = __uint_as_float((uint32_t)scales[k / 8] << 23);
      f32x4 v;
#pragma unroll
      for (int x = 0; x < 4; x++) v[x] = canon_nan(e2m1_to_f32(w >> 4 * x & 15u) * sc);
      __builtin_nontemporal_store(v, out + k);
    }
  }
}

}  // namespace

hipError_t launch_dequant_hf(const uint8_t *blocks, const uint8_t *scales, size_t rows, size_t cols, float *out, hipStream_t s) {
  if (cols % 32) return hipErrorInvalidValue;
  const size_t n = rows * (cols / 32) * 8;
  if (!n) return hipSuccess;
  const unsigned grid = (unsigned)std::min<size_t>((n + 511) / 512, (size_t)1 << 23);
  return launch_own(k_dequant_hf, grid, 256, 0, s, (const uint16_t *)blocks, scales, n, (f32x4 *)out);
}

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
