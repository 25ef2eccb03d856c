// Launches of the dense products, and the small kernels around them: f32 rows as bf16 planes, sums of
// partial results, column sums, the loss from the statistics of its tiles.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "dense_launch.hpp"

namespace moe {

int dense_parts(const DenseShape &s, const DenseArgs &a) {
  const DenseTileDims d = dense_tile_dims(dense_tile(a));
  if (s.epi == DENSE_STATS) return (a.M + d.bm - 1) / d.bm * d.wm;
  if (s.epi == DENSE_DGATE) return (a.N + d.bn - 1) / d.bn * d.wn;
  return 0;
}

namespace {
// k values of each split, a multiple of the step
int split_k(const DenseArgs &a) {
  const long steps = ((long)a.K + kDenseStep - 1) / kDenseStep, n = a.splits < 1 ? 1 : a.splits;
  return (int)((steps + n - 1) / n * kDenseStep);
}
}  // namespace

int dense_split_count(const DenseArgs &a) {
  const long k = split_k(a);
  return (int)((a.K + k - 1) / k);
}

int dense_splits(const DenseShape &, const DenseArgs &a0, int n_cu) {
  const DenseTileDims d = dense_tile_dims(dense_tile(a0));
  const long tiles = (long)((a0.M + d.bm - 1) / d.bm) * ((a0.N + d.bn - 1) / d.bn);
  const long steps = ((long)a0.K + kDenseStep - 1) / kDenseStep;
  // as many splits as fill the device twice, each of at least 8 steps
  DenseArgs a = a0;
  a.splits = (int)std::max(1L, std::min({2L * n_cu / std::max(1L, tiles), steps / 8, 64L}));
  return dense_split_count(a);
}

hipError_t launch_dense(const DenseShape &s, const DenseArgs &a0, hipStream_t st) {
  DenseArgs a = a0;
  if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.n_pass < 1 || a.n_pass > kMaxPass || a.lda % 8 || a.ldb % 8)
    return hipErrorInvalidValue;
  // (stores of 4 rows)
  if (a.M % 4 && s.epi != DENSE_STATS && s.epi != DENSE_DLOGITS) return hipErrorInvalidValue;
  a.k_split = split_k(a0);
  a.splits = dense_split_count(a0);
  if (a.splits > 1 && (s.epi != DENSE_STORE || a.out_mode != 1)) return hipErrorInvalidValue;
  return s.at ? launch_dense_tn(s, a, st) : launch_dense_nt(s, a, st);
}

namespace {

// One value per thread and step; bound by its 4 bytes read and 6 written.
__global__ void k_planes(const float *x, size_t n, uint16_t *out, size_t plane) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    uint16_t p[kPlanes];
    dense_split(x[i], p);
#pragma unroll
    for (int j = 0; j < kPlanes; j++) out[j * plane + i] = p[j];
  }
}

template <bool BF>
__global__ void k_sum_parts(const float *part, size_t stride, int parts, size_t n, const float *bias, size_t n_bias,
                            void *out) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    float s = 0.0f;
    for (int p = 0; p < parts; p++) s += part[p * stride + i];
    if (bias) s += bias[i % n_bias];
    if constexpr (BF)
      ((uint16_t *)out)[i] = dense_bf16(s);
    else
      ((float *)out)[i] = s;
  }
}

constexpr int kColRows = 64;  // rows per part
template <bool BF>
__global__ void k_colsum(const void *x, size_t T, size_t H, float *part) {
  const size_t c = (size_t)blockIdx.x * 256 + threadIdx.x, t0 = (size_t)blockIdx.y * kColRows;
  if (c >= H) return;
  const size_t t1 = t0 + kColRows < T ? t0 + kColRows : T;
  float s = 0.0f;
  for (size_t t = t0; t < t1; t++) {
    if constexpr (BF)
      s += bf16_to_f32(((const uint16_t *)x)[t * H + c]);
    else
      s += ((const float *)x)[t * H + c];
  }
  part[blockIdx.y * H + c] = s;
}

// A wavefront per token: the parts' maxima and sums joined, then the loss. A part's sum is of
// exponentials against its own maximum (0 where that is minus infinity).
__global__ __launch_bounds__(256) void k_loss(const float2 *stats, int parts, const float *picked, const int32_t *targets,
                                              size_t T, int vocab, float *loss, float *lse) {
  const size_t t = (size_t)blockIdx.x * 4 + threadIdx.x / 64;
  const int lane = threadIdx.x % 64;
  if (t >= T) return;
  float mx = -INFINITY, sum = 0.0f;
  for (int p = lane; p < parts; p += 64) {
    const float2 s = stats[p * T + t];
    if (s.x > mx) {
      sum *= dense_exp(mx - s.x);
      mx = s.x;
    }
    sum += s.y * dense_exp((s.x == -INFINITY ? 0.0f : s.x) - (mx == -INFINITY ? 0.0f : mx));
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const float m2 = __shfl_xor(mx, o), s2 = __shfl_xor(sum, o), m = fmaxf(mx, m2), b = m == -INFINITY ? 0.0f : m;
    sum = (mx == -INFINITY ? sum : sum * dense_exp(mx - b)) + (m2 == -INFINITY ? s2 : s2 * dense_exp(m2 - b));
    mx = m;
  }
  if (lane == 0) {
    const float l = (mx == -INFINITY ? 0.0f : mx) + logf(sum);
    const int y = targets[t];
    lse[t] = l;
    loss[t] = y < 0 ? 0.0f : y >= vocab ? NAN : l - picked[t];
  }
}

unsigned blocks_for(size_t n) { return (unsigned)std::min<size_t>((n + 255) / 256, 65536); }

}  // namespace

hipError_t launch_planes(const float *x, size_t n, uint16_t *out, size_t plane, hipStream_t s) {
  if (!n) return hipSuccess;
  k_planes<<<blocks_for(n), 256, 0, s>>>(x, n, out, plane);
  return hipGetLastError();
}

hipError_t launch_sum_parts(const float *part, size_t stride, int parts, size_t n, const float *bias, size_t n_bias,
                            void *out, bool bf16, hipStream_t s) {
  if (!n) return hipSuccess;
  if (bf16)
    k_sum_parts<true><<<blocks_for(n), 256, 0, s>>>(part, stride, parts, n, bias, n_bias, out);
  else
    k_sum_parts<false><<<blocks_for(n), 256, 0, s>>>(part, stride, parts, n, bias, n_bias, out);
  return hipGetLastError();
}

int dense_colsum_parts(size_t T) { return (int)((T + kColRows - 1) / kColRows); }
hipError_t launch_colsum(const void *x, bool bf16, size_t T, size_t H, float *part, hipStream_t s) {
  const dim3 grid((unsigned)((H + 255) / 256), (unsigned)dense_colsum_parts(T));
  if (!T || !H) return hipSuccess;
  if (bf16)
    k_colsum<true><<<grid, 256, 0, s>>>(x, T, H, part);
  else
    k_colsum<false><<<grid, 256, 0, s>>>(x, T, H, part);
  return hipGetLastError();
}

hipError_t launch_loss(const float2 *stats, int parts, const float *picked, const int32_t *targets, size_t T,
                       int vocab, float *loss, float *lse, hipStream_t s) {
  if (!T) return hipSuccess;
  k_loss<<<(unsigned)((T + 3) / 4), 256, 0, s>>>(stats, parts, picked, targets, T, vocab, loss, lse);
  return hipGetLastError();
}

}  // namespace moe
