// Activation checkpoints in 8 bits (MXFP8): e4m3 codes with one power-of-two scale per 32 values.
//
// e: the smallest exponent (at least -127) with max |x| <= 448 * 2^e, so that nothing saturates and
// every code is within half a step of its value: 2^-4 relative in e4m3's normal range, 2^(e - 10)
// below it. Scale byte e + 127. A block that holds a value that is not finite has scale byte 255 and
// reads back as NaN. A code times its scale has 4 significant bits: exact in bf16.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "dense.hpp"
#include "device.hpp"

namespace moe {
namespace {

__device__ __forceinline__ void load8(const float *x, float (&v)[8]) {
  const float4 a = *(const float4 *)x, b = *(const float4 *)(x + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const uint16_t *x, float (&v)[8]) {
  const uint4 u = *(const uint4 *)x;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// Four lanes a block of 32 values; bound by the bytes read and written.
template <class S>
__global__ __launch_bounds__(256) void k_act8_pack(const S *x, size_t blocks, uint8_t *codes, uint8_t *scales) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, b = i / 4;
  if (b >= blocks) return;  // (whole quads leave)
  float v[8];
  load8(x + i * 8, v);
  float m = 0.0f;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    m = fmaxf(m, fabsf(v[j]));
    bad |= !isfinite(v[j]);
  }
  if (bad) m = INFINITY;
  m = fmaxf(m, __shfl_xor(m, 1));
  m = fmaxf(m, __shfl_xor(m, 2));
  int e = -127;
  if (m > 0.0f && isfinite(m)) {
    const float f = frexpf(m, &e);  // m = f 2^e, f in [1/2, 1); 448 = 0.875 * 2^9
    e = max(e - 9 + (f > 0.875f ? 1 : 0), -127);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(v[4 * h], -e), ldexpf(v[4 * h + 1], -e), 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(v[4 * h + 2], -e), ldexpf(v[4 * h + 3], -e), p, true);
    w[h] = isfinite(m) ? (uint32_t)p : 0x7F7F7F7Fu;
  }
  *(uint2 *)(codes + i * 8) = uint2{w[0], w[1]};
  if (i % 4 == 0) scales[b] = (uint8_t)(isfinite(m) ? e + 127 : 255);
}

template <class D>
__global__ __launch_bounds__(256) void k_act8_unpack(const uint8_t *codes, const uint8_t *scales, size_t blocks, D *out, int copies) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, b = i / 4;
  if (b >= blocks) return;
  const uint2 u = *(const uint2 *)(codes + i * 8);
  const int sc = scales[b], e = sc - 127;
  const uint32_t w[2] = {u.x, u.y};
  float v[8];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    v[4 * h + 0] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(w[h], 0), e);
    v[4 * h + 1] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(w[h], 1), e);
    v[4 * h + 2] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(w[h], 2), e);
    v[4 * h + 3] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(w[h], 3), e);
  }
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (sc == 255) v[j] = NAN;
  for (int c = 0; c < copies; c++, out += blocks * 32) {
    if constexpr (sizeof(D) == 4) {
      float4 *o = (float4 *)(out + i * 8);
      o[0] = make_float4(v[0], v[1], v[2], v[3]);
      o[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint16_t q[8];
#pragma unroll
      for (int j = 0; j < 8; j++) q[j] = __builtin_bit_cast(uint16_t, (__bf16)v[j]);
      *(uint4 *)(out + i * 8) = __builtin_bit_cast(uint4, q);
    }
  }
}

}  // namespace

hipError_t launch_act8_pack(const void *x, bool bf16, size_t n, size_t cols, uint8_t *packed, hipStream_t s) {
  const size_t blocks = n * cols / 32;
  if (!blocks) return hipSuccess;
  const size_t grid = (blocks * 4 + 255) / 256;
  if (cols % 32 || grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  uint8_t *scales = packed + n * cols;
  if (bf16)
    k_act8_pack<<<(unsigned)grid, 256, 0, s>>>((const uint16_t *)x, blocks, packed, scales);
  else
    k_act8_pack<<<(unsigned)grid, 256, 0, s>>>((const float *)x, blocks, packed, scales);
  return hipGetLastError();
}

hipError_t launch_act8_unpack(const uint8_t *packed, size_t n, size_t cols, void *out, bool bf16, int copies, hipStream_t s) {
  const size_t blocks = n * cols / 32;
  if (!blocks) return hipSuccess;
  const size_t grid = (blocks * 4 + 255) / 256;
  if (cols % 32 || grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  const uint8_t *scales = packed + n * cols;
  if (bf16)
    k_act8_unpack<<<(unsigned)grid, 256, 0, s>>>(packed, scales, blocks, (uint16_t *)out, copies);
  else
    k_act8_unpack<<<(unsigned)grid, 256, 0, s>>>(packed, scales, blocks, (float *)out, copies);
  return hipGetLastError();
}

}  // namespace moe
