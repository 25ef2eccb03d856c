// Launches of the dense products, and the small kernels around them: f32 rows as bf16 planes, sums of
// partial results, column sums, the loss from the statistics of its tiles.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "act8.hpp"
#include "dense_launch.hpp"

namespace moe {

hipError_t launch_dense_pair(const DenseArgs &a0, const DenseArgs &b0, hipStream_t st) {
  DenseArgs a = a0, b = b0;
  const hipError_t e = dense_prepare_pair(a, b);
  if (e != hipSuccess) return e;
  double us = 0.0;
  return launch_dense_tt_pair(dense_pair_tile(a, b, us), a, b, st);
}

hipError_t launch_dense(const DenseShape &s, const DenseArgs &a0, hipStream_t st) {
  DenseArgs a = a0;
  const hipError_t e = dense_prepare(s, a);
  if (e != hipSuccess) return e;
  if (dense_few_rows(s, a)) return launch_dense_few(s, a, st);
  return s.at ? launch_dense_tn(s, a, st) : launch_dense_nt(s, a, st);
}

namespace {

// The job of this block of a launch of several: the first whose blocks end behind it. (The ends lie side by
// side, one scalar load.)
template <int N>
__device__ __forceinline__ int job_of(const unsigned (&end)[N]) {
  int j = 0;
#pragma unroll
  for (int i = 0; i < N - 1; i++) j += blockIdx.x >= end[i];
  return j;
}

// What a call does with its rows before its products, in one launch (each of its own cost 2 to 3 us): the
// planes of f32 rows, a checkpoint written or read, the column sums of up to kColRows rows, the scale of dloss.
// Bound by their bytes, of few rows by the launch.
// Rows of ignored tokens enter the loss's products as zeros: 0 times what they hold would make a NaN of dw.
__device__ __forceinline__ bool rows_ignored(const DenseRows &d, size_t i) {  // of value i
  if (!d.targets) return false;
  return d.targets[i >> 32 ? i / d.cols : (size_t)((uint32_t)i / (uint32_t)d.cols)] < 0;
}
__device__ __forceinline__ void rows_copy(const DenseRows &d, unsigned block) {
  for (size_t i = ((size_t)block * 256 + threadIdx.x) * 8; i < d.n; i += (size_t)d.blocks * 2048)
    *(uint4 *)((uint16_t *)d.out + i) = rows_ignored(d, i) ? uint4{0u, 0u, 0u, 0u} : *(const uint4 *)((const uint16_t *)d.x + i);
}
__device__ __forceinline__ void rows_planes(const DenseRows &d, unsigned block) {
  const float *x = (const float *)d.x;
  uint16_t *out = (uint16_t *)d.out;
  for (size_t i = ((size_t)block * 256 + threadIdx.x) * 4; i < d.n; i += (size_t)d.blocks * 1024) {  // (n is a multiple of 32)
    f32x4 v = *(const f32x4 *)(x + i);
    if (rows_ignored(d, i)) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    uint16_t p[4][kPlanes];
#pragma unroll
    for (int j = 0; j < 4; j++) dense_split(v[j], p[j]);
#pragma unroll
    for (int k = 0; k < kPlanes; k++) {
      uint16_t q[4] = {p[0][k], p[1][k], p[2][k], p[3][k]};
      dense_slots<false>(d.where, k, q, [&](size_t at, const auto &q) { *(uint2 *)(out + at * d.n + i) = __builtin_bit_cast(uint2, q); });
    }
  }
}

// by one block
__device__ __forceinline__ void dloss_scale(const DlossScale &d) {
  __shared__ float part[16];
  const int threads = blockDim.x;
  float m = 0.0f;
  for (size_t t = threadIdx.x; t < d.T; t += threads)
    if ((unsigned)d.targets[t] < (unsigned)d.vocab) m = fmaxf(m, fabsf(d.dloss[t]));
#pragma unroll
  for (int o = 1; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < threads / 64; i++) m = fmaxf(m, part[i]);
    *d.scale = m > 0.0f && isfinite(m) ? m : 1.0f;
  }
}
__global__ __launch_bounds__(1024) void k_dloss_scale(const DlossScale d) { dloss_scale(d); }

// The column sums of rows t0 to t1 (4096 x 2880 bf16: 7.7 us, 3.1 TB/s): a block of THREADS takes 64 columns, 8 threads of 8 columns a row.
template <int THREADS, class S>
__device__ __forceinline__ void column_sums(const S *x, size_t t0, size_t t1, size_t H, unsigned block, float *out) {
  __shared__ float s_sum[THREADS / 64][64];
  const int in = threadIdx.x % 8, row = threadIdx.x / 8;
  const size_t c = (size_t)block * 64 + in * 8;
  float s[8] = {};
  if (c < H) {  // (H is a multiple of 32)
#pragma unroll 4
    for (size_t t = t0 + row; t < t1; t += THREADS / 8) {
      float v[8];
      act8_load(x + t * H + c, v);
#pragma unroll
      for (int i = 0; i < 8; i++) s[i] += v[i];
    }
  }
  // over the 8 rows of a wavefront, then over the wavefronts in order
#pragma unroll
  for (int i = 0; i < 8; i++) {
    s[i] += __shfl_xor(s[i], 8);
    s[i] += __shfl_xor(s[i], 16);
    s[i] += __shfl_xor(s[i], 32);
    if (threadIdx.x % 64 < 8) s_sum[threadIdx.x / 64][in * 8 + i] = s[i];
  }
  __syncthreads();
  const size_t o = (size_t)block * 64 + threadIdx.x;
  if (threadIdx.x < 64 && o < H) {
    float v = 0.0f;
#pragma unroll
    for (int j = 0; j < THREADS / 64; j++) v += s_sum[j][threadIdx.x];
    out[o] = v;
  }
}
template <class S>
__global__ __launch_bounds__(1024) void k_colsum(const S *x, size_t T, size_t H, float *part) {
  const size_t t0 = (size_t)blockIdx.y * kColRows;
  column_sums<1024>(x, t0, min(T, t0 + kColRows), H, blockIdx.x, part + blockIdx.y * H);
}

// (planes alone, without the choice among jobs: 0.5 to 1 us less)
__global__ __launch_bounds__(256) void k_planes(const DenseRows d) { rows_planes(d, blockIdx.x); }
__global__ __launch_bounds__(256) void k_rows(const DenseRowJobs a) {
  const int j = job_of(a.end);
  const unsigned block = blockIdx.x - (j ? a.end[j - 1] : 0);
  const DenseRows &d = a.d[j];
  const size_t i0 = (size_t)block * 256 + threadIdx.x, step = (size_t)d.blocks * 256;  // of 8 values
  if (d.what == ROWS_PLANES) {
    rows_planes(d, block);
  } else if (d.what == ROWS_COPY) {
    rows_copy(d, block);
  } else if (d.what == ROWS_PACK8) {
    uint8_t *codes = (uint8_t *)d.out;
    for (size_t i = i0; i * 8 < d.n; i += step) act8_pack8((const float *)d.x, i, codes, codes + d.n);
  } else if (d.what == ROWS_UNPACK8) {
    const uint8_t *codes = (const uint8_t *)d.x;
    for (size_t i = i0; i * 8 < d.n; i += step) act8_unpack8(codes, codes + d.n, i, d.n / 32, (uint16_t *)d.out, d.copies);
  } else if (d.what == ROWS_SUM_BF16) {
    column_sums<256>((const uint16_t *)d.x, 0, d.n, d.cols, block, (float *)d.out);
  } else if (d.what == ROWS_SUM_F32) {
    column_sums<256>((const float *)d.x, 0, d.n, d.cols, block, (float *)d.out);
  } else {
    dloss_scale(a.scale);
  }
}

// Sums of parts, in order, of several results in one launch (each of its own cost 2 to 3 us, mostly the
// launch; a backward pass of 4096 rows of 2880 now 4.9 for its bias gradients). Many values: a thread each, 8 parts' loads in flight. Few of many parts (bias gradients): a
// block takes 32 values and 8 spans of the parts, whose sums join in order.
template <bool BF>
__device__ __forceinline__ void put(void *out, size_t i, float s) {
  if constexpr (BF)
    ((uint16_t *)out)[i] = dense_bf16(s);
  else
    ((float *)out)[i] = s;
}
__device__ __forceinline__ float sum_span(const float *part, size_t stride, int p0, int p1) {
  float s = 0.0f;
  int p = p0;
  for (; p + 8 <= p1; p += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = part[(size_t)(p + i) * stride];
#pragma unroll
    for (int i = 0; i < 8; i++) s += v[i];
  }
  for (; p < p1; p++) s += part[(size_t)p * stride];
  return s;
}
template <bool BF>
__device__ __forceinline__ void sum_many(const DenseSum &d, unsigned block) {
  for (size_t i = (size_t)block * 256 + threadIdx.x; i < d.n; i += (size_t)d.blocks * 256) {
    float s = sum_span(d.part + i, d.stride, 0, d.parts);
    if (d.bias) s += d.bias[i % d.n_bias];
    put<BF>(d.out, i, s);
  }
}
__global__ __launch_bounds__(256) void k_sums(const DenseSums a) {
  __shared__ float s_sum[8][32];
  const int j = job_of(a.end);
  const unsigned block = blockIdx.x - (j ? a.end[j - 1] : 0);
  const DenseSum &d = a.d[j];
  if (d.bf16) return sum_many<true>(d, block);
  if (!d.few) return sum_many<false>(d, block);
  const size_t i = (size_t)block * 32 + threadIdx.x % 32;
  const int span = threadIdx.x / 32, each = (d.parts + 7) / 8;
  if (i < d.n) s_sum[span][threadIdx.x % 32] = sum_span(d.part + i, d.stride, min(span * each, d.parts), min((span + 1) * each, d.parts));
  __syncthreads();
  if (span == 0 && i < d.n) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) s += s_sum[k][threadIdx.x];
    ((float *)d.out)[i] = s;
  }
}

// A block takes 16 rows of 128 inner columns, 2 rows a thread of 4 columns. Bound by its bytes (333 f32 rows of
// 1536, gate and up and dh in three parts each: 55 MB in 10 us, most of it from the caches).
template <bool ONE>
__global__ __launch_bounds__(256) void k_dgate(const DgateArgs a) {
  __shared__ float s_db[8][256];
  const int in = threadIdx.x % 32, row = threadIdx.x / 32, i = blockIdx.x * 128 + in * 4;
  float db[8] = {};
  if (i < a.I) {  // (I is a multiple of 8)
#pragma unroll
    for (int k = 0; k < kDgateRows / 8; k++) {
      const size_t t = (size_t)blockIdx.y * kDgateRows + k * 8 + row;
      if (t >= (size_t)a.T) break;
      float v[8] = {}, dh[4] = {}, d[8], hv[4];
      for (int p = 0; p < a.gu_parts; p++) {
        const f32x4 *x = (const f32x4 *)(a.gu + (p * (size_t)a.T + t) * 2 * a.I + 2 * i);
        const f32x4 lo = x[0], hi = x[1];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] += lo[r], v[4 + r] += hi[r];
      }
      for (int p = 0; p < a.dh_parts; p++) {
        const f32x4 x = *(const f32x4 *)(a.dh + (p * (size_t)a.T + t) * a.I + i);
#pragma unroll
        for (int r = 0; r < 4; r++) dh[r] += x[r];
      }
      if (a.bias)
#pragma unroll
        for (int r = 0; r < 8; r++) v[r] += a.bias[2 * i + r];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        DenseGate g;
        g.set<ONE>(v[2 * r], v[2 * r + 1], a.limit);
        hv[r] = g.h();
        d[2 * r] = g.dg(dh[r], v[2 * r], a.limit);
        d[2 * r + 1] = g.du(dh[r], v[2 * r + 1], a.limit);
      }
#pragma unroll
      for (int r = 0; r < 8; r++) db[r] += d[r];
      const size_t plane = (size_t)a.T * a.I;
      for (int p = 0; p < (ONE ? 1 : kPlanes); p++) {
        uint16_t q[8], e[4];
        dense_take<!ONE>(d, q);
        dense_take<!ONE>(hv, e);
        dense_slots<ONE>(a.dgu_where, p, q, [&](size_t at, const auto &q) { *(uint4 *)(a.dgu + at * 2 * plane + t * 2 * a.I + 2 * i) = __builtin_bit_cast(uint4, q); });
        dense_slots<ONE>(a.h_where, p, e, [&](size_t at, const auto &e) { *(uint2 *)(a.h + at * plane + t * a.I + i) = __builtin_bit_cast(uint2, e); });
      }
    }
  }
  if (!a.db_part) return;
#pragma unroll
  for (int r = 0; r < 8; r++) s_db[row][in * 8 + r] = db[r];
  __syncthreads();
  const int o = blockIdx.x * 256 + threadIdx.x;
  if (o < 2 * a.I) {
    float v = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) v += s_db[j][threadIdx.x];
    a.db_part[(size_t)blockIdx.y * 2 * a.I + o] = v;
  }
}

// One (maximum, sum of exponentials against it) of two; a sum whose maximum is minus infinity is 0 or NaN.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  const float s = (a.x == m ? a.y : a.x == -INFINITY ? a.y : a.y * dense_exp(a.x - m)) +
                  (b.x == m ? b.y : b.x == -INFINITY ? b.y : b.y * dense_exp(b.x - m));
  return make_float2(m, s);
}

// A block joins the parts of 2^lt tokens (16 of many tokens, so that its reads are whole lines; 1 of few,
// so that its 1024 threads share the parts), then their losses. Bound by the latency of its reads: 5 to 8 us of
// few tokens, 12 of 4096 (12.9 MB).
__global__ __launch_bounds__(1024) void k_loss(const float2 *stats, int parts, const float *picked, const int32_t *targets,
                                               size_t T, int vocab, int lt, float *loss, float *lse) {
  __shared__ float2 s_part[1024];
  const int in = threadIdx.x & ((1 << lt) - 1), rows = 1024 >> lt;
  const size_t t = ((size_t)blockIdx.x << lt) + in;
  float2 v = make_float2(-INFINITY, 0.0f);
  if (t < T) {
    int p = threadIdx.x >> lt;
    for (; p + 3 * rows < parts; p += 4 * rows) {  // 4 loads under way
      float2 q[4];
#pragma unroll
      for (int i = 0; i < 4; i++) q[i] = stats[(p + i * rows) * T + t];
#pragma unroll
      for (int i = 0; i < 4; i++) v = join(v, q[i]);
    }
    for (; p < parts; p += rows) v = join(v, stats[p * T + t]);
  }
  s_part[threadIdx.x] = v;
  for (int h = 512; h >= 1 << lt; h >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < h) s_part[threadIdx.x] = v = join(v, s_part[threadIdx.x + h]);
  }
  if ((threadIdx.x >> lt) == 0 && t < T) {
    const float l = (v.x == -INFINITY ? 0.0f : v.x) + logf(v.y);
    const int y = targets[t];
    lse[t] = l;
    loss[t] = y < 0 ? 0.0f : y >= vocab ? NAN : l - picked[t];
  }
}

}  // namespace

hipError_t launch_rows(DenseRowJobs a, hipStream_t s) {
  const size_t blocks = a.ends();
  if (a.count == 1 && a.d[0].what == ROWS_PLANES)
    return launch_own(k_planes, (unsigned)blocks, 256, 0, s, a.d[0]);
  return blocks ? launch_own(k_rows, (unsigned)blocks, 256, 0, s, a) : hipSuccess;
}

hipError_t launch_sums(DenseSums a, hipStream_t s) {
  const size_t blocks = a.ends();
  return blocks ? launch_own(k_sums, (unsigned)blocks, 256, 0, s, a) : hipSuccess;
}

hipError_t launch_dgate(const DgateArgs &a, hipStream_t s) {
  const dim3 grid((a.I + 127) / 128, dense_dgate_parts(a.T));
  if (a.T < 1 || a.I < 8 || a.I % 8 || grid.y > 65535) return hipErrorInvalidValue;
  return launch_own(a.planes == 1 ? k_dgate<true> : k_dgate<false>, grid, 256, 0, s, a);
}

hipError_t launch_dloss_scale(const DlossScale &d, hipStream_t s) {
  return launch_own(k_dloss_scale, 1, 1024, 0, s, d);
}

hipError_t launch_colsum(const void *x, bool bf16, size_t T, size_t H, float *part, hipStream_t s) {
  const dim3 grid((unsigned)((H + 63) / 64), (unsigned)dense_colsum_parts(T));
  if (!T || !H) return hipSuccess;
  return bf16 ? launch_own(k_colsum<uint16_t>, grid, 1024, 0, s, (const uint16_t *)x, T, H, part)
              : launch_own(k_colsum<float>, grid, 1024, 0, s, (const float *)x, T, H, part);
}

hipError_t launch_loss(const float2 *stats, int parts, const float *picked, const int32_t *targets, size_t T,
                       int vocab, float *loss, float *lse, hipStream_t s) {
  if (!T) return hipSuccess;
  const int lt = T >= 1024 ? 4 : T >= 64 ? 2 : 0;
  return launch_own(k_loss, (unsigned)((T + (1 << lt) - 1) >> lt), 1024, 0, s, stats, parts, picked, targets, T, vocab, lt, loss, lse);
}

}  // namespace moe
