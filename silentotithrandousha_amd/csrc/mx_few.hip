// Products of a few rows with a resident MXFP4 matrix (mx_gemm.hpp's operands and arithmetic): bound by the weights, which a
// workgroup's 8 wavefronts stream through registers, each every eighth step of K, and by the latency of its loads.
// There is no barrier before the wavefronts' sums meet in LDS, where they are added in order.
#include "device.hpp"
#include "serve.hpp"

namespace moe {
namespace {

constexpr int kFewWaves = 8;

// RT row tiles a workgroup, CT tiles of 16 tokens.
template <int FMT, int TERMS, int RT, int CT>
__global__ __launch_bounds__(64 * kFewWaves) void k_mx_few(MxGemmArgs a) {
  constexpr int kChunk = FMT == 4 ? 1024 : FMT == 6 ? 1536 : 2048;
  __shared__ f32x4 s_sum[kFewWaves][RT * CT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  const uint32_t m0 = blockIdx.x * RT, n0 = blockIdx.y * CT, nb = a.d.nb, ns = a.d.ns, nq = a.d.nq;
  const uint32_t *wsc = (const uint32_t *)(a.w + pack_weight_bytes(a.d));
  f32x4 acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; i++)
#pragma unroll
    for (int j = 0; j < CT; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
  for (uint32_t s = wave; s < ns; s += kFewWaves) {
    u32x4 A[RT];
    uint32_t sa[RT], sb[CT];
    const uint32_t in_tile = min((s * 64 + lane) * 16, 256 * nb - 16);  // (a last step may be short: its scales are 0)
#pragma unroll
    for (int i = 0; i < RT; i++) {
      const uint32_t m = min(m0 + i, a.d.tiles - 1);
      A[i] = __builtin_nontemporal_load((const u32x4 *)(a.w + (size_t)m * 256 * nb + in_tile));
      sa[i] = wsc[((size_t)m * nq + s / 4) * 64 + lane];
    }
    const uint8_t *row[CT];
#pragma unroll
    for (int j = 0; j < CT; j++) {
      const uint32_t n = min(n0 + j, a.r.tiles - 1);
      sb[j] = a.scales[((size_t)n * nq + s / 4) * 64 + lane];
      row[j] = a.codes + ((size_t)n * ns + s) * TERMS * kChunk + lane * 16;
    }
    i32x8 B[TERMS][CT];
#pragma unroll
    for (int t = 0; t < TERMS; t++)
#pragma unroll
      for (int j = 0; j < CT; j++) {
        const uint8_t *p = row[j] + t * kChunk;
        const uint4 v = *(const uint4 *)p;
        B[t][j] = i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
        if constexpr (FMT == 6) {
          const uint2 u = *(const uint2 *)(p - lane * 8 + 1024);
          B[t][j][4] = (int)u.x, B[t][j][5] = (int)u.y;
        } else if constexpr (FMT == 8) {
          const uint4 u = *(const uint4 *)(p + 1024);
          B[t][j][4] = (int)u.x, B[t][j][5] = (int)u.y, B[t][j][6] = (int)u.z, B[t][j][7] = (int)u.w;
        }
      }
    const int sh = 8 * (s & 3);
#pragma unroll
    for (int i = 0; i < RT; i++) sa[i] >>= sh;
#pragma unroll
    for (int j = 0; j < CT; j++) sb[j] = sb[j] >> sh & 255;
    constexpr int kB = FMT == 4 ? 4 : FMT == 6 ? 2 : 0;
#pragma unroll
    for (int t = 0; t < TERMS; t++) {
      if (t)
#pragma unroll
        for (int j = 0; j < CT; j++) sb[j] = (uint32_t)max((int)sb[j] - 5, 1);
#pragma unroll
      for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < CT; j++)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(i32x8{(int)A[i].x, (int)A[i].y, (int)A[i].z, (int)A[i].w, 0, 0, 0, 0},
                                                                       B[t][j], acc[i][j], 4, kB, 0, (int)sa[i], 0, (int)sb[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; i++)
#pragma unroll
    for (int j = 0; j < CT; j++) s_sum[wave][i * CT + j][lane] = acc[i][j];
  __syncthreads();
  // lane l of a tile: token l % 16, rows 4 (l / 16) ..
  for (int k = wave; k < RT * CT; k += kFewWaves) {
    f32x4 v = s_sum[0][k][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; w++) v = v + s_sum[w][k][lane];
    const uint32_t m = m0 + k / CT, t = (n0 + k % CT) * 16 + (lane & 15);
    if (m >= a.d.tiles || t >= a.r.tokens) continue;
    const uint32_t at = m * 16 + g * 4;
    if (a.bias) v = v + *(const f32x4 *)(a.bias + at);
    if (a.bf16) {
      uint16_t q[4];
#pragma unroll
      for (int x = 0; x < 4; x++) q[x] = __builtin_bit_cast(uint16_t, (__bf16)v[x]);
      *(uint2 *)((uint16_t *)a.out + (size_t)t * a.d.rows + at) = __builtin_bit_cast(uint2, q);
    } else {
      *(f32x4 *)((float *)a.out + (size_t)t * a.d.rows + at) = v;
    }
  }
}

template <int FMT, int TERMS, int RT, int CT>
hipError_t launch(const MxGemmArgs &a, hipStream_t s) {
  return launch_own(k_mx_few<FMT, TERMS, RT, CT>, dim3((a.d.tiles + RT - 1) / RT, (a.r.tiles + CT - 1) / CT), dim3(64 * kFewWaves), 0, s, a);
}

template <int FMT, int TERMS>
hipError_t by_tokens(const MxGemmArgs &a, hipStream_t s) {
  switch (a.r.tiles) {
    case 1: return launch<FMT, TERMS, 1, 1>(a, s);
    case 2: return launch<FMT, TERMS, 2, 2>(a, s);
    default: return launch<FMT, TERMS, 2, 4>(a, s);
  }
}

}  // namespace

hipError_t launch_mx_few(const MxGemmArgs &a, hipStream_t s) {
  if (a.d.tiles >= 1u << 22) return hipErrorInvalidValue;  // (a launch has less than 2^32 threads)
  switch (a.r.type) {
    case MOE_F32: return by_tokens<6, 6>(a, s);
    case MOE_BF16: return by_tokens<6, 4>(a, s);
    case MOE_MXFP8: return by_tokens<8, 1>(a, s);
    case MOE_MXFP4: return by_tokens<4, 1>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace moe
