// 8-bit checkpoints on the device: what act8.hip's kernels and the preparation of the gated block's rows do with
// a block of 32 values.
#pragma once
#include <hip/hip_runtime.h>

#include "device.hpp"

namespace moe {

__device__ __forceinline__ void act8_load(const float *x, float (&v)[8]) {
  const float4 a = *(const float4 *)x, b = *(const float4 *)(x + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void act8_load(const uint16_t *x, float (&v)[8]) {
  const uint4 u = *(const uint4 *)x;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// Values 8 i to 8 i + 7 of x: four lanes share a block of 32, and come here together.
template <class S>
__device__ __forceinline__ void act8_pack8(const S *x, size_t i, uint8_t *codes, uint8_t *scales) {
  const size_t b = i / 4;
  float v[8];
  act8_load(x + i * 8, v);
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
__device__ __forceinline__ void act8_unpack8(const uint8_t *codes, const uint8_t *scales, size_t i, size_t blocks, D *out, int copies) {
  const size_t b = i / 4;
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

}  // namespace moe
