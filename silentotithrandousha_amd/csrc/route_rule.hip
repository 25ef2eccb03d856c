// The choice of experts from a token's logits by a rule (moe_routing), and its gradient. One wavefront a token;
// lane l holds experts l, l + 64, ...
//
// Scores are computed and compared in 64 bits: with a bias two experts' keys may lie closer than an f32 tells apart, and which
// of them a token takes would hang on the last bit of an exponential.
#include <algorithm>

#include "device.hpp"
#include "serve.hpp"

namespace moe {
namespace {

constexpr int kMaxRuleExperts = 1024, kMaxGroups = 64, kMaxRuleK = 32;

__device__ __forceinline__ double xor_double(double v, int m) { return __shfl_xor(v, m); }
__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmax(v, xor_double(v, m));
  return v;
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = v + xor_double(v, m);
  return v;
}
__device__ __forceinline__ double lane64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ double sigmoid64(double l) { return 1.0 / (1.0 + exp(-l)); }

// Scores of all experts from their logits (-inf: masked).
template <int Q>
__device__ __forceinline__ void scores64(const RouteRule &r, const float (&l)[Q], double (&s)[Q]) {
  if (r.score == MOE_SCORE_SIGMOID) {
#pragma unroll
    for (int q = 0; q < Q; q++) s[q] = l[q] == -INFINITY ? 0.0 : sigmoid64((double)l[q]);
    return;
  }
  float m = l[0];
#pragma unroll
  for (int q = 1; q < Q; q++) m = fmaxf(m, l[q]);
  m = wave_max(m);
  double sum = 0.0;
#pragma unroll
  for (int q = 0; q < Q; q++) {
    s[q] = l[q] == m ? 1.0 : exp((double)l[q] - (double)m);  // (infinite logits share; all masked: below)
    if (l[q] == -INFINITY) s[q] = 0.0;
    sum = sum + s[q];
  }
  sum = wave_sum64(sum);
#pragma unroll
  for (int q = 0; q < Q; q++) s[q] = sum > 0.0 ? s[q] / sum : 0.0;
}

template <int Q>
__device__ __forceinline__ void load_logits(const float *row, int E, int lane, float (&l)[Q]) {
#pragma unroll
  for (int q = 0; q < Q; q++) {
    const int e = 64 * q + lane;
    l[q] = e < E ? row[e] : -INFINITY;
    if (l[q] != l[q]) l[q] = -INFINITY;
  }
}

template <int Q>
__global__ __launch_bounds__(256) void k_route_rule(RouteRule r, const float *logits, uint32_t T, int E, int32_t *idx, float *w,
                                                    int32_t *counts, int whole) {
  extern __shared__ __align__(16) uint8_t s_mem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int *s_count = (int *)s_mem;  // [E] if counts
  double *s_key = (double *)(s_mem + (counts ? (size_t)64 * Q * 4 : 0)) + (size_t)wave * 64 * Q;  // [E] a wavefront, of a rule with groups
  if (counts) {
    for (int e = threadIdx.x; e < E; e += blockDim.x) s_count[e] = 0;
    __syncthreads();
  }
  for (uint32_t t = blockIdx.x * waves + wave; t < T; t += gridDim.x * waves) {
    float l[Q];
    double s[Q], key[Q];
    load_logits<Q>(logits + (size_t)t * E, E, lane, l);
    scores64<Q>(r, l, s);
#pragma unroll
    for (int q = 0; q < Q; q++) {
      const int e = 64 * q + lane;
      key[q] = l[q] == -INFINITY ? -INFINITY : r.bias && e < E ? s[q] + (double)r.bias[e] : s[q];
      if (key[q] != key[q]) key[q] = -INFINITY;  // (a NaN bias)
    }
    if (r.groups > 1) {
      const int per = E / r.groups;
#pragma unroll
      for (int q = 0; q < Q; q++) s_key[64 * q + lane] = key[q];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      double best = -INFINITY, next = -INFINITY;
      if (lane < r.groups)
        for (int i = 0; i < per; i++) {
          const double v = s_key[lane * per + i];
          next = v > best ? best : fmax(next, v);
          best = fmax(best, v);
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      double g = r.two && next > -INFINITY ? best + next : best;
      // groups taken: those with fewer than top_groups before them
      int before = 0;
      for (int i = 0; i < r.groups; i++) {
        const double o = lane64(g, i);
        before += o > g || (o == g && i < lane);
      }
      const uint64_t kept = __ballot(lane < r.groups && before < r.top_groups);
#pragma unroll
      for (int q = 0; q < Q; q++) {
        const int e = 64 * q + lane;
        if (e < E && !(kept >> (e / per) & 1)) l[q] = -INFINITY;
      }
    }
#pragma unroll
    for (int q = 0; q < Q; q++)
      key[q] = l[q] == -INFINITY ? -INFINITY : r.bias ? key[q] : (double)l[q];
    // (an infinite logit's key must not be a masked one's)
    double mine = 0.0, total = 0.0;  // of slot `lane`
    int slot = -1, chosen = 0;
    uint32_t live = 0;
#pragma unroll
    for (int q = 0; q < Q; q++) live |= (uint32_t)(key[q] > -INFINITY) << q;
    for (int j = 0; j < r.k; j++) {
      double top = -INFINITY;
#pragma unroll
      for (int q = 0; q < Q; q++)
        if (live >> q & 1) top = fmax(top, key[q]);
      top = wave_max64(top);
      if (top == -INFINITY) break;
      int e = -1;
      double sc = 0.0;
#pragma unroll
      for (int q = 0; q < Q; q++) {
        const uint64_t at = __ballot((live >> q & 1) && key[q] == top);
        if (e < 0 && at) {
          const int from = __builtin_ctzll(at);
          e = 64 * q + from;
          sc = lane64(s[q], from);
          if (lane == from) live &= ~(1u << q);
        }
      }
      total = total + sc;
      if (lane == j) {
        slot = e;
        mine = sc;
      }
      chosen++;
    }
    if (lane < r.k) {
      double v = mine;
      if (r.normalize) v = total > 0.0 ? mine / total : slot >= 0 ? 1.0 / chosen : 0.0;
      idx[(size_t)t * r.k + lane] = slot;
      w[(size_t)t * r.k + lane] = slot >= 0 ? (float)(v * (double)r.scale) : 0.0f;
      if (counts && slot >= 0) atomicAdd(s_count + slot, 1);
    }
  }
  if (counts) {
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
      if (whole)
        counts[e] = s_count[e];
      else if (s_count[e])
        atomicAdd(counts + e, s_count[e]);  // (whole numbers: any order gives the same)
    }
  }
}

// With w_j = scale s_j / S (S the chosen scores' sum, or 1):
//   d / d s_j = scale / S dw_j - (normalised) sum_i dw_i w_i / S,
//   sigmoid: d l_j = d s_j s_j (1 - s_j);  softmax: d l_e = s_e (d s_e - sum_j d s_j s_j).
// Of a normalised softmax the sum is 0 and only the chosen experts have a gradient.
template <int Q>
__global__ __launch_bounds__(256) void k_route_rule_backward(RouteRule r, const float *logits, const int32_t *idx, const float *dw, uint32_t T,
                                                             int E, float *dl) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (uint32_t t = blockIdx.x * 4 + wave; t < T; t += gridDim.x * 4) {
    float l[Q];
    double s[Q];
    load_logits<Q>(logits + (size_t)t * E, E, lane, l);
    scores64<Q>(r, l, s);
    int e = -1;
    double d = 0.0;
    if (lane < r.k) {
      e = idx[(size_t)t * r.k + lane];
      if (e < 0 || e >= E)
        e = -1;
      else
        d = (double)dw[(size_t)t * r.k + lane] * (double)r.scale;
    }
    // the scores of the chosen
    double sc = 0.0, rest = 0.0;  // and 1 - s of a sigmoid
    for (int j = 0; j < r.k; j++) {
      const int ej = __builtin_amdgcn_readlane(e, j);
      if (ej < 0) continue;
      double v = 0.0;
      float lg = 0.0f;
#pragma unroll
      for (int q = 0; q < Q; q++)
        if (q == ej >> 6) {
          v = lane64(s[q], ej & 63);
          lg = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l[q]), ej & 63));
        }
      if (lane == j) {
        sc = v;
        rest = lg == -INFINITY ? 0.0 : 1.0 / (1.0 + exp((double)lg));
      }
    }
    const double S = wave_sum64(sc);
    double ds = d;
    if (r.normalize) ds = S > 0.0 ? (d - wave_sum64(d * sc) / S) / S : 0.0;
    double g[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) g[q] = 0.0;
    if (r.score == MOE_SCORE_SIGMOID) ds = ds * sc * rest;
    for (int j = 0; j < r.k; j++) {
      const int ej = __builtin_amdgcn_readlane(e, j);
      const double v = lane64(ds, j);
      if (ej < 0) continue;
#pragma unroll
      for (int q = 0; q < Q; q++)
        if (64 * q + lane == ej) g[q] = g[q] + v;
    }
    if (r.score == MOE_SCORE_SOFTMAX) {
      const double mean = r.normalize ? 0.0 : wave_sum64(ds * sc);
#pragma unroll
      for (int q = 0; q < Q; q++) g[q] = s[q] * (g[q] - mean);
    }
#pragma unroll
    for (int q = 0; q < Q; q++)
      if (64 * q + lane < E) dl[(size_t)t * E + 64 * q + lane] = (float)g[q];
  }
}

}  // namespace

hipError_t launch_route_rule(const RouteRule &r, const float *logits, size_t T, int E, int32_t *idx, float *w, int32_t *counts, hipStream_t s) {
  if (E < 1 || E > kMaxRuleExperts || r.k < 1 || r.k > kMaxRuleK || r.groups > kMaxGroups) return hipErrorInvalidValue;
  const bool whole = T <= 64;  // one workgroup takes all: its counts are the result
  if (counts && !whole) {
    hipError_t e = launch_zero(counts, (size_t)E * 4, s);
    if (e != hipSuccess) return e;
  }
  const int Q = E <= 64 ? 1 : E <= 128 ? 2 : E <= 256 ? 4 : E <= 512 ? 8 : 16;
  const unsigned grid = whole ? 1 : (unsigned)std::min<size_t>((T + 3) / 4, 4096);
  const size_t lds = (counts ? (size_t)256 * Q : 0) + (r.groups > 1 ? (size_t)4 * 512 * Q : 0);
  auto go = [&](auto k) { return launch_own(k, grid, 256, lds, s, r, logits, (uint32_t)T, E, idx, w, counts, (int)whole); };
  return Q == 1 ? go(k_route_rule<1>) : Q == 2 ? go(k_route_rule<2>) : Q == 4 ? go(k_route_rule<4>) : Q == 8 ? go(k_route_rule<8>) : go(k_route_rule<16>);
}

hipError_t launch_route_rule_backward(const RouteRule &r, const float *logits, const int32_t *idx, const float *dw, size_t T, int E, float *dl,
                                      hipStream_t s) {
  if (E < 1 || E > kMaxRuleExperts || r.k < 1 || r.k > kMaxRuleK) return hipErrorInvalidValue;
  if (!T) return hipSuccess;
  const unsigned grid = (unsigned)std::min<size_t>((T + 3) / 4, 16384);
  auto go = [&](auto k) { return launch_own(k, grid, 256, 0, s, r, logits, idx, dw, (uint32_t)T, E, dl); };
  return E <= 64    ? go(k_route_rule_backward<1>)
         : E <= 128 ? go(k_route_rule_backward<2>)
         : E <= 256 ? go(k_route_rule_backward<4>)
         : E <= 512 ? go(k_route_rule_backward<8>)
                    : go(k_route_rule_backward<16>);
}

}  // namespace moe
