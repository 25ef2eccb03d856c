// Products of a few rows with a resident MXFP4 matrix (mx_gemm.hpp's operands and arithmetic): bound by the weights, which a
// workgroup's 8 wavefronts stream through registers, each every eighth step of K, and by the latency of its loads.
// There is no barrier before the wavefronts' sums meet in LDS, where they are added in order. (One f32 row over 5760 x 2880: 4.7 us for
// 8.8 MB, of which the stream is 1.3 and the rest a launch's and a load's latency. K split over workgroups instead, with a launch that
// adds the parts, was slower.)
#include "act8.hpp"
#include "mx_gemm.hpp"
#include "serve.hpp"

namespace moe {
namespace {

constexpr int kFewWaves = 8;

// RT row tiles a workgroup, CT tiles of 16 tokens.
template <int FMT, int TERMS, int RT, int CT>
__global__ __launch_bounds__(64 * kFewWaves) void k_mx_few(MxGemmArgs a) {
  constexpr int kChunk = FMT == 4 || FMT == 16 ? 1024 : FMT == 6 ? 1536 : 2048;
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
      if constexpr (FMT != 16) sb[j] = a.scales[((size_t)n * nq + s / 4) * 64 + lane];
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
    for (int j = 0; j < CT; j++) sb[j] = FMT == 16 ? 0 : sb[j] >> sh & 255;
    constexpr int kB = FMT == 4 ? 4 : FMT == 6 ? 2 : 0;
#pragma unroll
    for (int t = 0; t < TERMS; t++) {
      if (t && FMT == 6)
#pragma unroll
        for (int j = 0; j < CT; j++) sb[j] = (uint32_t)max((int)sb[j] - 5, 1);
#pragma unroll
      for (int i = 0; i < RT; i++) {
        if constexpr (FMT == 16) {
          const bf16x8 w = mx_weights8(A[i][t], sa[i] & 255);
#pragma unroll
          for (int j = 0; j < CT; j++)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, as_bf16x8(make_uint4(B[t][j][0], B[t][j][1], B[t][j][2], B[t][j][3])), acc[i][j], 0, 0, 0);
          continue;
        }
#pragma unroll
        for (int j = 0; j < CT; j++)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(i32x8{(int)A[i].x, (int)A[i].y, (int)A[i].z, (int)A[i].w, 0, 0, 0, 0},
                                                                       B[t][j], acc[i][j], 4, kB, 0, (int)sa[i], 0, (int)sb[j]);
      }
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

// One or two f32 rows, whose terms fit the MFMA's 16 columns (column t TERMS + i: term i of token t): the terms are made by every
// workgroup for itself, while its weights are on their way. (Made by a launch of their own, one f32 row over 5760 x
// 2880 took 10.6 us, so 5.1.)
constexpr int kEarly = 3;  // steps of a wavefront whose weights are asked for first

__global__ __launch_bounds__(64 * kFewWaves) void k_mx_one(MxGemmArgs a, const float *x) {
  constexpr int TERMS = 6;
  extern __shared__ __align__(16) uint8_t s_mem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, col = lane & 15;
  const uint32_t m = blockIdx.x, nb = a.d.nb, ns = a.d.ns, nq = a.d.nq, T = a.r.tokens, cols = T * TERMS, blocks = 4 * ns;
  f32x4 *s_sum = (f32x4 *)s_mem;                   // [8 wavefronts][64]
  float *s_col = (float *)(s_mem + 8 * 64 * 16);   // [16 columns][16 rows]
  uint8_t *s_code = s_mem + 8 * 64 * 16 + 1024;    // [blocks][cols] 24 bytes
  uint32_t *s_scale = (uint32_t *)(s_code + (size_t)blocks * cols * 24);  // [blocks][cols]
  const uint8_t *w = a.w + (size_t)m * 256 * nb;
  const uint32_t *wsc = (const uint32_t *)(a.w + pack_weight_bytes(a.d)) + (size_t)m * nq * 64 + lane;
  auto weights = [&](uint32_t s) {  // (a last step may be short: its scales are 0)
    return __builtin_nontemporal_load((const u32x4 *)(w + min((s * 64 + lane) * 16, 256 * nb - 16)));
  };
  u32x4 A[kEarly];
  uint32_t sa[kEarly];
#pragma unroll
  for (int i = 0; i < kEarly; i++) {
    const uint32_t s = min((uint32_t)(wave + i * kFewWaves), ns - 1);
    A[i] = weights(s);
    sa[i] = wsc[s / 4 * 64];
  }
  // a pair of lanes a block of 32 values (pairs leave together)
  for (uint32_t k = tid; k < 2 * blocks * T; k += 64 * kFewWaves) {
    const uint32_t b = k / 2 % blocks, t = k / 2 / blocks, half = k & 1;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = 0.0f;
    if (b < nb) {
      float u[8];
      act8_load(x + (size_t)t * nb * 32 + b * 32 + half * 16, u);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = u[i];
      act8_load(x + (size_t)t * nb * 32 + b * 32 + half * 16 + 8, u);
#pragma unroll
      for (int i = 0; i < 8; i++) v[8 + i] = u[i];
    }
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      top = fmaxf(top, fabsf(v[i]));
      bad |= !isfinite(v[i]);
    }
    if (bad) top = INFINITY;
    top = fmaxf(top, __shfl_xor(top, 1));
    bad = !isfinite(top);
    int E = 0;
    if (top > 0.0f && !bad) frexpf(top, &E);
    f32x16v lo = {}, hi = {};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      lo[i] = bad ? 0.0f : v[2 * i];
      hi[i] = bad ? 0.0f : v[2 * i + 1];
    }
#pragma unroll
    for (int i = 0; i < TERMS; i++) {
      const int se = split_scale_exp<TERMS>(E, i);
      const float sc = __builtin_amdgcn_ldexpf(1.0f, se);
      u32x6v c;
      asm volatile("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3" : "=&v"(c) : "v"(lo), "v"(hi), "v"(sc));
      if (i + 1 < TERMS) {  // the residual feeds the next term
        f32x32v q;
        asm volatile("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2" : "=&v"(q) : "v"(c), "v"(sc));
#pragma unroll
        for (int n = 0; n < 8; n++) {
          lo[n] = lo[n] - q[2 * n];
          hi[n] = hi[n] - q[2 * n + 1];
        }
      }
      const uint32_t at = b * cols + t * TERMS + i;
      uint32_t *o = (uint32_t *)(s_code + at * 24 + half * 12);
      o[0] = c[0];
      o[1] = c[1];
      o[2] = c[2];
      if (!half) s_scale[at] = bad ? 255u : (uint32_t)(se + 127);
    }
  }
  __syncthreads();
  f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto step = [&](uint32_t s, const u32x4 &A, uint32_t sa) {
    const uint32_t at = (4 * s + g) * cols + min((uint32_t)col, cols - 1);  // (columns past the last: the last again)
    const uint2 *p = (const uint2 *)(s_code + at * 24);
    const uint2 p0 = p[0], p1 = p[1], p2 = p[2];
    const i32x8 B{(int)p0.x, (int)p0.y, (int)p1.x, (int)p1.y, (int)p2.x, (int)p2.y, 0, 0};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(i32x8{(int)A.x, (int)A.y, (int)A.z, (int)A.w, 0, 0, 0, 0}, B, acc, 4, 2, 0,
                                                           (int)(sa >> 8 * (s & 3)), 0, (int)s_scale[at]);
  };
#pragma unroll
  for (int i = 0; i < kEarly; i++)
    if (wave + i * kFewWaves < ns) step(wave + i * kFewWaves, A[i], sa[i]);
#pragma unroll 2
  for (uint32_t s = wave + kEarly * kFewWaves; s < ns; s += kFewWaves) step(s, weights(s), wsc[s / 4 * 64]);
  s_sum[wave * 64 + lane] = acc;
  __syncthreads();
  if (tid < 64) {  // the wavefronts' sums in order, then the terms'
    f32x4 v = s_sum[tid];
#pragma unroll
    for (int k = 1; k < kFewWaves; k++) v = v + s_sum[k * 64 + tid];
    *(f32x4 *)(s_col + col * 16 + g * 4) = v;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint32_t row = tid & 15, t = tid >> 4;
    if (t < T) {
      float v = s_col[(t * TERMS + TERMS - 1) * 16 + row];
#pragma unroll
      for (int i = TERMS - 2; i >= 0; i--) v = v + s_col[(t * TERMS + i) * 16 + row];
      if (a.bias) v = v + a.bias[m * 16 + row];
      const size_t at = (size_t)t * a.d.rows + m * 16 + row;
      if (a.bf16)
        ((__bf16 *)a.out)[at] = (__bf16)v;
      else
        ((float *)a.out)[at] = v;
    }
  }
}

// Up to 16 bf16 rows that fit 64 KB of LDS, where every workgroup puts them while its weights are on their way: 16 bytes a thread, those
// with a value that is not finite as NaN. One row over 201088 x 2880, whose weights are 308 MB, takes 49 us, 6.3 TB/s, over 5760 x 2880 4.5, eight
// rows 84 and 6. Two tiles of rows a workgroup share what it puts there, where there are tiles enough. (In terms: 70, 4.5, 133 and 9. Read
// by each wavefront from memory, 64 bytes a lane in 16 rows, one row took 67 and 5.1, eight 75 and 6.8.)
template <int RT>
__global__ __launch_bounds__(64 * kFewWaves) void k_mx_bf16(MxGemmArgs a, const uint16_t *x) {
  extern __shared__ __align__(16) uint8_t s_mem[];
  f32x4(*s_sum)[RT][64] = (f32x4(*)[RT][64])s_mem;  // [8 wavefronts]
  uint8_t *s_x = s_mem + kFewWaves * RT * 1024;     // [tokens] of 16 ns pieces of 16 bytes and one more
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, col = lane & 15;
  const uint32_t m0 = blockIdx.x * RT, nb = a.d.nb, ns = a.d.ns, nq = a.d.nq, T = a.r.tokens, stride = (16 * ns + 1) * 16;
  const uint32_t *wsc = (const uint32_t *)(a.w + pack_weight_bytes(a.d));
  u32x4 A[kEarly][RT];
  uint32_t sa[kEarly][RT];
  auto weights = [&](uint32_t s0) {
#pragma unroll
    for (int e = 0; e < kEarly; e++) {
      const uint32_t s = min(s0 + e * kFewWaves, ns - 1);
#pragma unroll
      for (int i = 0; i < RT; i++) {
        const uint32_t m = min(m0 + i, a.d.tiles - 1);
        A[e][i] = __builtin_nontemporal_load((const u32x4 *)(a.w + (size_t)m * 256 * nb + min((s * 64 + lane) * 16, 256 * nb - 16)));
        sa[e][i] = wsc[((size_t)m * nq + s / 4) * 64 + lane];
      }
    }
  };
  weights(wave);
  for (uint32_t t = 0; t < T; t++)
    for (uint32_t c = tid; c < 16 * ns; c += 64 * kFewWaves) {  // (a last step may be short)
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (c < 4 * nb) v = ((const uint4 *)x)[(size_t)t * 4 * nb + c];
      *(uint4 *)(s_x + t * stride + c * 16) = mx_not_finite(v) ? make_uint4(kNan2, kNan2, kNan2, kNan2) : v;
    }
  __syncthreads();
  f32x4 acc[RT][2];  // (one chain of MFMAs would be twice as long)
#pragma unroll
  for (int i = 0; i < RT; i++) acc[i][0] = acc[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const uint8_t *row = s_x + min((uint32_t)col, T - 1) * stride + g * 64;  // (columns past the last: the last again)
  for (uint32_t s0 = wave;;) {
#pragma unroll
    for (int e = 0; e < kEarly; e++) {
      const uint32_t s = s0 + e * kFewWaves;
      if (s >= ns) break;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const bf16x8 v = *(const bf16x8 *)(row + s * 256 + k * 16);
#pragma unroll
        for (int i = 0; i < RT; i++)
          acc[i][k & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_weights8(A[e][i][k], sa[e][i] >> 8 * (s & 3) & 255), v, acc[i][k & 1], 0, 0, 0);
      }
    }
    s0 += kEarly * kFewWaves;
    if (s0 >= ns) break;
    weights(s0);
  }
#pragma unroll
  for (int i = 0; i < RT; i++) s_sum[wave][i][lane] = acc[i][0] + acc[i][1];
  __syncthreads();
  if (wave >= RT) return;
  f32x4 v = s_sum[0][wave][lane];
#pragma unroll
  for (int w = 1; w < kFewWaves; w++) v = v + s_sum[w][wave][lane];
  const uint32_t m = m0 + wave, at = m * 16 + g * 4;
  if (m >= a.d.tiles || (uint32_t)col >= T) return;
  if (a.bias) v = v + *(const f32x4 *)(a.bias + at);
  if (a.bf16) {
    uint16_t q[4];
#pragma unroll
    for (int i = 0; i < 4; i++) q[i] = __builtin_bit_cast(uint16_t, (__bf16)v[i]);
    *(uint2 *)((uint16_t *)a.out + (size_t)col * a.d.rows + at) = __builtin_bit_cast(uint2, q);
  } else {
    *(f32x4 *)((float *)a.out + (size_t)col * a.d.rows + at) = v;
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

hipError_t launch_mx_one(const MxGemmArgs &a, const void *x, hipStream_t s) {
  if (!mx_one_takes(a.r.type, a.r.tokens, (size_t)a.d.nb * 32) || a.d.tiles >= 1u << 22) return hipErrorInvalidValue;
  if (a.r.type == MOE_BF16) {
    auto go = [&](auto k, unsigned rt) {
      return launch_own(k, dim3((a.d.tiles + rt - 1) / rt), dim3(64 * kFewWaves), mx_one_rows(a.d.nb, a.r.tokens) + kFewWaves * rt * 1024, s, a, (const uint16_t *)x);
    };
    return a.d.tiles < 1024 ? go(k_mx_bf16<1>, 1) : go(k_mx_bf16<2>, 2);
  }
  return launch_own(k_mx_one, dim3(a.d.tiles), dim3(64 * kFewWaves), mx_one_lds(a.d.nb, (size_t)a.r.tokens * 6), s, a, (const float *)x);
}

hipError_t launch_mx_few(const MxGemmArgs &a, hipStream_t s) {
  if (a.d.tiles >= 1u << 22) return hipErrorInvalidValue;  // (a launch has less than 2^32 threads)
  switch (a.r.type) {
    case MOE_F32: return by_tokens<6, 6>(a, s);
    case MOE_BF16: return by_tokens<16, 4>(a, s);
    case MOE_MXFP8: return by_tokens<8, 2>(a, s);
    case MOE_MXFP4: return by_tokens<4, 1>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace moe
