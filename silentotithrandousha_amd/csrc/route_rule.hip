// The choice of experts from a token's logits by a rule (moe_routing), and its gradient. One wavefront a token at a time; lane l
// holds experts Q l .. Q l + Q - 1.
//
// Which experts are chosen hangs on the order of their keys, score + bias, which may lie closer than an f32 tells apart; the
// scores are those of 64 bits. Computed for all experts they cost more than all else (16384 tokens of 256 experts: 85 us), so
// keys are first taken in f32, each within 2^-19 of the row's largest score (and 2^-24 of itself), and the choice stands if no two
// keys that it compares are closer than 2^-18 of that. Else (a token in some hundreds) it is made again with keys of 64 bits.
// Without a bias or groups the logits' order is the scores', exactly. Weights are of 64 bits until their rounding.
//
// 16384 tokens of 256 experts (8 of 4 of 8 groups, sigmoid, bias): 34 us, the gradient 13, where their bytes take 11. Bound by
// its instructions, 690 VALU and 440 SALU a token (VALU 71 % busy at 4 wavefronts a SIMD, for the 97 registers of the 64-bit choice):
// k times a largest key over the wavefront, its lane and its place, one after the other. 512 workgroups in place of 256: 40 us.
#include <algorithm>

#include "device.hpp"
#include "serve.hpp"

namespace moe {
namespace {

constexpr int kMaxRuleExperts = 1024, kMaxGroups = 64, kMaxRuleK = 32;

__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmax(v, __shfl_xor(v, m));
  return v;
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = v + __shfl_xor(v, m);
  return v;
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {  // (0 for lanes without a source)
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane64(double v, int lane);
// the sum over the lanes below 32, where the others hold 0
__device__ __forceinline__ double slots_sum64(double v) {
  v = v + dpp64<0x111>(v);  // row_shr 1, 2, 4, 8: a row's sum in its last lane
  v = v + dpp64<0x112>(v);
  v = v + dpp64<0x114>(v);
  v = v + dpp64<0x118>(v);
  return lane64(v, 15) + lane64(v, 31);
}
// 1 / v for v in [1, 2 kMaxRuleK] or so: v_rcp_f64 and two steps of Newton's.
__device__ __forceinline__ double inverse64(double v) {
  double y = __builtin_amdgcn_rcp(v);
  y = fma(fma(-v, y, 1.0), y, y);
  return fma(fma(-v, y, 1.0), y, y);
}
__device__ __forceinline__ double lane64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float lane32(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

// exp(x), x at most 0 or so: 2^n e^r, |r| <= ln 2 / 2, its Taylor series to the 12th power (within 2^-52); ln 2 in two parts.
__device__ __forceinline__ double exp64(double x) {
  x = fmax(x, -745.0);
  const double n = rint(x * 1.4426950408889634), r = fma(n, -1.9082149292705877e-10, fma(n, -0.693147180369123816490, x));
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}
__device__ __forceinline__ double sigmoid64(double l) {
  const double e = exp64(-fabs(l));
  return (l < 0.0 ? e : 1.0) * inverse64(1.0 + e);
}

// The logits of a lane's experts, -inf past the last one and for a NaN.
template <int Q>
__device__ __forceinline__ void load_logits(const float *row, int E, int lane, float (&l)[Q]) {
  struct __attribute__((packed, aligned(4))) some { float v[Q]; };
  const int e0 = lane * Q;
#pragma unroll
  for (int q = 0; q < Q; q++) l[q] = -INFINITY;
  if (e0 + Q <= E) {
    const some s = *(const some *)(row + e0);
#pragma unroll
    for (int q = 0; q < Q; q++) l[q] = s.v[q];
  } else {
#pragma unroll
    for (int q = 0; q < Q; q++)
      if (e0 + q < E) l[q] = row[e0 + q];
  }
}

// Scores of all experts (-inf: masked); m: the largest logit.
template <int Q>
__device__ __forceinline__ void scores64(int score, const float (&l)[Q], float m, double (&s)[Q]) {
  double sum = 0.0;
#pragma unroll
  for (int q = 0; q < Q; q++) {
    if (score == MOE_SCORE_SIGMOID)
      s[q] = l[q] == -INFINITY ? 0.0 : sigmoid64((double)l[q]);
    else  // (infinite logits share)
      s[q] = l[q] == -INFINITY ? 0.0 : l[q] == m ? 1.0 : exp64((double)l[q] - (double)m);
    sum = sum + s[q];
  }
  if (score == MOE_SCORE_SIGMOID) return;
  sum = wave_sum64(sum);
#pragma unroll
  for (int q = 0; q < Q; q++) s[q] = sum > 0.0 ? s[q] / sum : 0.0;
}

__device__ __forceinline__ float wave_largest(float v) { return wave_fmax_dpp(v); }

// The choice by keys of 64 bits (-inf: never): lane j < k gets slot j's expert, -1 for none. s_key: a wavefront's LDS.
template <int Q>
__device__ __forceinline__ void choose64(const RouteRule &r, int E, int lane, const double (&group_key)[Q], const double (&key)[Q], double *s_key,
                                         int &slot) {
  uint32_t live = 0;
#pragma unroll
  for (int q = 0; q < Q; q++) live |= (uint32_t)(key[q] > -INFINITY) << q;
  if (r.groups > 1) {
    const int per = E / r.groups;
#pragma unroll
    for (int q = 0; q < Q; q++) s_key[lane * Q + q] = group_key[q];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    double best = -INFINITY, next = -INFINITY;
    if (lane < r.groups)
      for (int i = 0; i < per; i++) {
        const double v = s_key[lane * per + i];
        next = fmax(next, fmin(best, v));
        best = fmax(best, v);
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const double g = lane < r.groups ? (r.two && next > -INFINITY ? best + next : best) : -INFINITY;
    // groups with fewer than top_groups before them
    int before = 0;
    for (int i = 0; i < r.groups; i++) {
      const double o = lane64(g, i);
      before += o > g || (o == g && i < lane);
    }
    const uint64_t kept = __ballot(lane < r.groups && before < r.top_groups);
#pragma unroll
    for (int q = 0; q < Q; q++) {
      const int e = lane * Q + q;
      if (e >= E || !(kept >> (e / per) & 1)) live &= ~(1u << q);
    }
  }
  slot = -1;
  for (int j = 0; j < r.k; j++) {
    double mine = -INFINITY;
    int at = 0;
#pragma unroll
    for (int q = 0; q < Q; q++)
      if ((live >> q & 1) && key[q] > mine) {
        mine = key[q];
        at = q;
      }
    const double top = wave_max64(mine);
    if (top == -INFINITY) return;
    const int from = __builtin_ctzll(__ballot(mine == top));
    const int e = from * Q + __builtin_amdgcn_readlane(at, from);
    if (lane == from) live &= ~(1u << at);
    if (lane == j) slot = e;
  }
}

// An f32's place in the order of f32s (-0 as 0); 0: never chosen.
__device__ __forceinline__ uint32_t order32(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return v > -INFINITY ? u ^ ((uint32_t)((int)u >> 31) | 0x80000000u) : 0u;
}
__device__ __forceinline__ float of_order32(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }
template <int CTRL>
__device__ __forceinline__ float dpp32(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, false));
}

// The same in f32, and only where it is sure: lane j < k gets slot j's expert. group_key, key: -inf for never.
template <int Q>
__device__ __forceinline__ bool choose32(const RouteRule &r, int E, int lane, const float (&group_key)[Q], const float (&key)[Q], float group_gap,
                                         float gap, int &slot) {
  uint32_t k[Q];
#pragma unroll
  for (int q = 0; q < Q; q++) k[q] = order32(key[q]);
  if (r.groups > 1) {
    const int per = E / r.groups, lanes = per / Q;
    if (lanes * Q != per || lanes > 16 || (lanes & (lanes - 1))) return false;  // (groups that share lanes)
    float best = -INFINITY, next = -INFINITY;
    auto take = [&](float b, float n) {  // the two largest of best >= next and b >= n
      next = fmaxf(fminf(best, b), fmaxf(next, n));
      best = fmaxf(best, b);
    };
#pragma unroll
    for (int q = 0; q < Q; q++) {
      next = fmaxf(next, fminf(best, group_key[q]));
      best = fmaxf(best, group_key[q]);
    }
    // (quad permutes and mirrors, as wave_max: every lane of a group ends with its result)
    if (lanes > 1) take(dpp32<0xB1>(best), dpp32<0xB1>(next));
    if (lanes > 2) take(dpp32<0x4E>(best), dpp32<0x4E>(next));
    if (lanes > 4) take(dpp32<0x141>(best), dpp32<0x141>(next));
    if (lanes > 8) take(dpp32<0x140>(best), dpp32<0x140>(next));
    const float g = r.two && next > -INFINITY ? best + next : best;
    const int mine = lane / lanes;
    int before = 0;
    bool close = false;
    for (int i = 0; i < r.groups; i++) {
      const float o = lane32(g, i * lanes);
      before += o > g || (o == g && i < mine);
      close |= i != mine && !(fabsf(o - g) > group_gap);
    }
    if (__any(close && mine < r.groups && g > -INFINITY)) return false;
    if (mine >= r.groups || before >= r.top_groups)
#pragma unroll
      for (int q = 0; q < Q; q++) k[q] = 0;
  }
  auto head = [&]() {
    uint32_t h = k[0];
#pragma unroll
    for (int q = 1; q < Q; q++) h = max(h, k[q]);
    return h;
  };
  slot = -1;
  uint32_t h = head(), tops = 0;  // lane j: the j-th key
  for (int j = 0; j < r.k; j++) {
    const uint32_t top = wave_max_u32(h);
    if (lane == j) tops = top;
    if (top == 0) break;
    const int from = __builtin_ctzll(__ballot(h == top));
    int at = 0;
#pragma unroll
    for (int q = Q - 1; q >= 0; q--)
      if ((uint32_t)__builtin_amdgcn_readlane((int)k[q], from) == top) at = q;
    if (lane == j) slot = from * Q + at;
#pragma unroll
    for (int q = 0; q < Q; q++)
      if (at == q) k[q] = lane == from ? 0u : k[q];
    h = head();
  }
  if (gap == 0.0f) return true;
  const uint32_t left = wave_max_u32(h);  // the first one left out
  if (lane >= r.k) tops = left;
  const uint32_t after = __shfl_down(tops, 1);
  // (keys of neighbouring slots; a slot without an expert is far from all)
  const bool close = lane < r.k && after != 0 && !(of_order32(tops) - of_order32(after) > gap);
  return !__any(close);
}

// Threads of a workgroup: each adds its counts to the result once, and additions to one line wait for each other, so
// workgroups are few and large (256 of 1024 threads 30.4 us, 1024 of 256 36.4, for 16384 tokens' 8 largest of 256 logits).
constexpr int rule_threads(int Q) { return Q <= 4 ? 1024 : Q == 8 ? 512 : 256; }

template <int Q>
__global__ __launch_bounds__(rule_threads(Q)) void k_route_rule(RouteRule r, const float *logits, uint32_t T, int E, int32_t *idx, float *w,
                                                    int32_t *counts, int whole) {
  extern __shared__ __align__(16) uint8_t s_mem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int *s_count = (int *)s_mem;  // [64 Q] if counts
  double *s_key = (double *)(s_mem + (counts ? (size_t)64 * Q * 4 : 0)) + (size_t)wave * 64 * Q;  // of a rule with groups
  float bias[Q];
  load_logits<Q>(r.bias ? r.bias : logits, r.bias ? E : 0, lane, bias);  // (-inf past the last expert)
  if (counts) {
    for (int e = threadIdx.x; e < E; e += rule_threads(Q)) s_count[e] = 0;
    __syncthreads();
  }
  float next[Q];
  constexpr int kWaves = rule_threads(Q) / 64;
  const uint32_t step = gridDim.x * kWaves;
  uint32_t t = blockIdx.x * kWaves + wave;
  if (t < T) load_logits<Q>(logits + (size_t)t * E, E, lane, next);
  for (; t < T; t += step) {
    float l[Q], m = -INFINITY;
#pragma unroll
    for (int q = 0; q < Q; q++) l[q] = next[q];
    if (t + step < T) load_logits<Q>(logits + (size_t)(t + step) * E, E, lane, next);
#pragma unroll
    for (int q = 0; q < Q; q++) {
      l[q] = fmaxf(l[q], -INFINITY);
      m = fmaxf(m, l[q]);
    }
    int slot;
    const bool by_logit = !r.bias && r.groups <= 1;
    if (by_logit || r.score == MOE_SCORE_SOFTMAX) m = wave_largest(m);
    bool sure;
    if (by_logit) {
      sure = choose32<Q>(r, E, lane, l, l, 0.0f, 0.0f, slot);
    } else {
      float s[Q], key[Q], top = 1.0f, most = 0.0f;  // top: the largest score
      if (r.score == MOE_SCORE_SIGMOID) {
#pragma unroll
        for (int q = 0; q < Q; q++) s[q] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[q] * -1.44269504f));
      } else {
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < Q; q++) {
          s[q] = l[q] == m ? 1.0f : __builtin_amdgcn_exp2f((l[q] - m) * 1.44269504f);
          sum = sum + (l[q] == -INFINITY ? 0.0f : s[q]);
        }
        top = __builtin_amdgcn_rcpf(wave_sum_xor(sum));
#pragma unroll
        for (int q = 0; q < Q; q++) s[q] = s[q] * top;
      }
#pragma unroll
      for (int q = 0; q < Q; q++) {
        if (r.bias) s[q] = s[q] + bias[q];
        s[q] = l[q] == -INFINITY ? -INFINITY : fmaxf(s[q], -INFINITY);  // (a NaN bias: never)
        key[q] = r.bias ? s[q] : l[q];
        if (r.bias) most = fmaxf(most, s[q] > -INFINITY ? fabsf(s[q]) : 0.0f);
      }
      if (r.bias) most = wave_largest(most);
      const float gap = 0x1p-18f * (top + most);
      sure = choose32<Q>(r, E, lane, s, key, 2.0f * gap, r.bias ? gap : 0.0f, slot);
    }
    if (!sure) {
      double s[Q], key[Q];
      scores64<Q>(r.score, l, m, s);
#pragma unroll
      for (int q = 0; q < Q; q++) {
        if (r.bias) s[q] = s[q] + (double)bias[q];
        if (l[q] == -INFINITY || s[q] != s[q]) s[q] = -INFINITY;
        key[q] = r.bias ? s[q] : s[q] == -INFINITY ? -INFINITY : (double)l[q];
      }
      choose64<Q>(r, E, lane, s, key, s_key, slot);
    }
    const float logit = slot >= 0 ? fmaxf(logits[(size_t)t * E + slot], -INFINITY) : -INFINITY;  // (in a cache)
    // the chosen scores, a lane a slot
    double sc = 0.0;
    if (r.score == MOE_SCORE_SIGMOID) {
      if (slot >= 0) sc = sigmoid64((double)logit);
    } else {
      if (slot >= 0) sc = logit == m ? 1.0 : exp64((double)logit - (double)m);
      if (!r.normalize) {
        double s[Q], sum = 0.0;
#pragma unroll
        for (int q = 0; q < Q; q++) {
          s[q] = l[q] == -INFINITY ? 0.0 : l[q] == m ? 1.0 : exp64((double)l[q] - (double)m);
          sum = sum + s[q];
        }
        sum = wave_sum64(sum);
        if (slot >= 0) sc = sc / sum;
      }
    }
    if (r.normalize) {
      const double total = slots_sum64(sc);
      sc = total > 0.0 ? sc / total : 1.0 / max(__popcll(__ballot(slot >= 0)), 1);
    }
    if (lane < r.k) {
      idx[(size_t)t * r.k + lane] = slot;
      w[(size_t)t * r.k + lane] = slot >= 0 ? (float)(sc * (double)r.scale) : 0.0f;
      if (counts && slot >= 0) atomicAdd(s_count + slot, 1);
    }
  }
  if (counts) {
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += rule_threads(Q)) {
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
// Of a normalised softmax that sum is 0, and S stands for its denominator, too: as for a sigmoid, the chosen experts' logits are
// all that is read, and the other gradients are 0.
template <int Q>
__global__ __launch_bounds__(256) void k_route_rule_backward(RouteRule r, const float *logits, const int32_t *idx, const float *dw, uint32_t T,
                                                             int E, float *dl) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool dense = r.score == MOE_SCORE_SOFTMAX && !r.normalize;
  const uint32_t step = gridDim.x * 4;
  for (uint32_t t = blockIdx.x * 4 + wave; t < T; t += step) {
    int e = -1;
    double d = 0.0;
    float lg = -INFINITY;
    if (lane < r.k) {
      e = idx[(size_t)t * r.k + lane];
      const float g = dw[(size_t)t * r.k + lane];
      if (e < 0 || e >= E) {
        e = -1;
      } else {
        lg = fmaxf(logits[(size_t)t * E + e], -INFINITY);
        d = (double)g * (double)r.scale;
      }
    }
    double sc = 0.0, rest = 1.0, sum = 1.0, g[Q];  // rest: 1 - s of a sigmoid
    float l[Q], m;
    if (r.score == MOE_SCORE_SIGMOID) {
      const double x = exp64(-fabs((double)lg)), y = inverse64(1.0 + x);
      sc = lg == -INFINITY ? 0.0 : lg < 0.0f ? x * y : y;
      rest = lg < 0.0f ? y : x * y;
    } else {
      m = lg;
      if (dense) {
        load_logits<Q>(logits + (size_t)t * E, E, lane, l);
#pragma unroll
        for (int q = 0; q < Q; q++) {
          l[q] = fmaxf(l[q], -INFINITY);
          m = fmaxf(m, l[q]);
        }
      }
      m = wave_largest(m);
      sc = lg == -INFINITY ? 0.0 : lg == m ? 1.0 : exp64((double)lg - (double)m);
      if (dense) {
        sum = 0.0;
#pragma unroll
        for (int q = 0; q < Q; q++) {
          g[q] = l[q] == -INFINITY ? 0.0 : l[q] == m ? 1.0 : exp64((double)l[q] - (double)m);
          sum = sum + g[q];
        }
        sum = wave_sum64(sum);
        sum = sum > 0.0 ? 1.0 / sum : 0.0;
        sc = sc * sum;
      }
    }
    double ds = d;
    if (r.normalize) {
      const double S = slots_sum64(sc), inv = S > 0.0 ? 1.0 / S : 0.0;
      ds = (d - slots_sum64(d * sc) * inv) * inv;
    }
    if (!dense) {
      ds = ds * sc * rest;
#pragma unroll
      for (int q = 0; q < Q; q++) g[q] = 0.0;
    } else {
      const double mean = slots_sum64(ds * sc);
#pragma unroll
      for (int q = 0; q < Q; q++) g[q] = g[q] * sum * -mean;
      ds = ds * sc;
    }
    for (int j = 0; j < r.k; j++) {
      const int ej = __builtin_amdgcn_readlane(e, j);
      const double v = lane64(ds, j);
      if (ej < 0) continue;
#pragma unroll
      for (int q = 0; q < Q; q++)
        if (q == ej % Q && lane == ej / Q) g[q] = g[q] + v;
    }
    struct __attribute__((packed, aligned(4))) some { float v[Q]; };
    float *out = dl + (size_t)t * E + lane * Q;
    if (lane * Q + Q <= E) {
      some o;
#pragma unroll
      for (int q = 0; q < Q; q++) o.v[q] = (float)g[q];
      *(some *)out = o;
    } else {
#pragma unroll
      for (int q = 0; q < Q; q++)
        if (lane * Q + q < E) out[q] = (float)g[q];
    }
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
  const int threads = rule_threads(Q), waves = threads / 64;
  const unsigned grid = whole && counts ? 1 : (unsigned)std::min<size_t>((T + waves - 1) / waves, 256);
  const size_t lds = (counts ? (size_t)256 * Q : 0) + (r.groups > 1 ? (size_t)waves * 512 * Q : 0);
  auto go = [&](auto k) { return launch_own(k, grid, threads, lds, s, r, logits, (uint32_t)T, E, idx, w, counts, (int)whole); };
  return Q == 1 ? go(k_route_rule<1>) : Q == 2 ? go(k_route_rule<2>) : Q == 4 ? go(k_route_rule<4>) : Q == 8 ? go(k_route_rule<8>) : go(k_route_rule<16>);
}

hipError_t launch_route_rule_backward(const RouteRule &r, const float *logits, const int32_t *idx, const float *dw, size_t T, int E, float *dl,
                                      hipStream_t s) {
  if (E < 1 || E > kMaxRuleExperts || r.k < 1 || r.k > kMaxRuleK) return hipErrorInvalidValue;
  if (!T) return hipSuccess;
  const unsigned grid = (unsigned)std::min<size_t>((T + 3) / 4, 4096);
  auto go = [&](auto k) { return launch_own(k, grid, 256, 0, s, r, logits, idx, dw, (uint32_t)T, E, dl); };
  return E <= 64    ? go(k_route_rule_backward<1>)
         : E <= 128 ? go(k_route_rule_backward<2>)
         : E <= 256 ? go(k_route_rule_backward<4>)
         : E <= 512 ? go(k_route_rule_backward<8>)
                    : go(k_route_rule_backward<16>);
}

}  // namespace moe
