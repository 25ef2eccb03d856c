// The choice of experts from a token's logits by a rule (moe_routing), and its gradient. One wavefront a token at a time; lane l
// holds experts Q l .. Q l + Q - 1.
//
// Which experts are chosen hangs on the order of their keys, score + bias, which may lie closer than an f32 tells apart; the
// scores are those of 64 bits. Computed for all experts they cost more than all else (16384 tokens of 256 experts: 85 us), so
// keys are first taken in f32, each within 2^-19 of the row's largest score (and 2^-24 of itself), and the choice stands if no two
// keys that it compares are closer than 2^-18 of that. Else (0.6 % of the tokens of the
// case below) it is made again with keys of 64 bits.
// Without a bias or groups the logits' order is the scores', exactly. Weights are of 64 bits until their rounding.
//
// 16384 tokens of 256 experts (8 of 4 of 8 groups, sigmoid, bias): 23 us, the gradient 8.4, where their bytes take 11. Bound by
// instructions at 4 wavefronts a SIMD (some 100 registers, the 64-bit choice's), and by the last wavefronts that make a 64-bit choice.
// One token a wavefront (k_route_rule: 690 VALU and 440 SALU instructions a token, k times a largest key over the wavefront, its lane and
// its place) took 33.
#include <algorithm>

#include "device.hpp"
#include "serve.hpp"

namespace moe {
namespace {

constexpr int kMaxRuleExperts = 1024, kMaxGroups = 64, kMaxRuleK = 32;

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
// the sum of a row of 16 lanes in its last lane: row_shr 1, 2, 4, 8
__device__ __forceinline__ double row_sum64(double v) {
  v = v + dpp64<0x111>(v);
  v = v + dpp64<0x112>(v);
  v = v + dpp64<0x114>(v);
  return v + dpp64<0x118>(v);
}
// the sum over the lanes below 32, where the others hold 0
__device__ __forceinline__ double slots_sum64(double v) {
  v = row_sum64(v);
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
// the largest of the wavefront: within rows by permutes, of which every lane gets its result, then of four lanes
template <int CTRL>
__device__ __forceinline__ double max_perm64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return fmax(v, __builtin_bit_cast(double, (uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double wave_max64(double v) {
  v = max_perm64<0x140>(max_perm64<0x141>(max_perm64<0x4E>(max_perm64<0xB1>(v))));
  return fmax(fmax(lane64(v, 0), lane64(v, 16)), fmax(lane64(v, 32), lane64(v, 48)));
}
__device__ __forceinline__ float lane32(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

// exp(x), x at most 0 or so: 2^n e^r, |r| <= ln 2 / 2, its Taylor series to the 12th power (within 2^-52); r by Cody and Waite's reduction,
// ln 2 as its first 32 bits, whose product with n is exact, and the rest.
__device__ __forceinline__ double exp64(double x) {
  x = fmax(x, -745.0);
  const double n = rint(x * 1.4426950408889634), r = fma(n, -0x1.a39ef35793c76p-33, fma(n, -0x1.62e42feep-1, x));
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

// Normalised weights stay the same if all scores are divided by one number. Where every chosen score lies below e^kFar, their 64-bit
// numbers lose bits and their sum's inverse leaves the range: there they are divided by the largest of them, which leaves
// e^(l - the largest chosen logit) of a softmax, and of a sigmoid, which is e^l to the last bit there. A softmax score below
// 2^-1075 (e^kGone) counts as 0.
constexpr double kFar = -600.0, kLeast = 0x1p-865 /* a little more than e^kFar */, kGone = -745.1332191019412;

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
    // (groups that share lanes: 64 bits for every token. 16384 of 160 experts in 8 groups 45 to 49 us, of 256 in 8 25 to 34)
    if (lanes * Q != per || lanes > 16 || (lanes & (lanes - 1))) return false;
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

// The choice by keys of 64 bits for logits l of a wavefront's lanes; m: the largest logit (of a softmax).
template <int Q>
__device__ __forceinline__ int choose_exact(const RouteRule &r, int E, int lane, const float (&l)[Q], const float (&bias)[Q], float m, double *s_key) {
  double s[Q], key[Q];
  scores64<Q>(r.score, l, m, s);
#pragma unroll
  for (int q = 0; q < Q; q++) {
    if (r.bias) s[q] = s[q] + (double)bias[q];
    if (l[q] == -INFINITY || s[q] != s[q]) s[q] = -INFINITY;
    key[q] = r.bias ? s[q] : s[q] == -INFINITY ? -INFINITY : (double)l[q];
  }
  int slot;
  choose64<Q>(r, E, lane, s, key, s_key, slot);
  return slot;
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
    if (!sure) slot = choose_exact<Q>(r, E, lane, l, bias, m, s_key);
    const float logit = slot >= 0 ? fmaxf(logits[(size_t)t * E + slot], -INFINITY) : -INFINITY;  // (in a cache)
    // the chosen scores, a lane a slot
    double sc = 0.0;
    if (r.score == MOE_SCORE_SIGMOID) {
      if (slot >= 0) sc = sigmoid64((double)logit);
      if (r.normalize && !__any((double)logit >= kFar)) {
        const double top = (double)wave_largest(logit);
        sc = slot >= 0 ? exp64((double)logit - top) : 0.0;
      }
    } else {
      if (slot >= 0) sc = logit == m ? 1.0 : exp64((double)logit - (double)m);
      if (r.normalize) {
        if (!__any(slot >= 0 && sc > kLeast)) {
          const double top = (double)wave_largest(logit);
          sc = slot >= 0 && top - (double)m >= kGone ? exp64((double)logit - top) : 0.0;
        }
      } else {
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

// A value of all 32 lanes of a half wavefront, from their own: rows of 16 by DPP, then each row with its half's other.
template <class F>
__device__ __forceinline__ uint32_t half_all(uint32_t v, F &&f) {
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
  v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
  const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return f(p[0], p[1]);
}
__device__ __forceinline__ uint32_t half_max_u32(uint32_t v) {
  return half_all(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ float half_max(float v) {
  return __uint_as_float(half_all(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
__device__ __forceinline__ float half_sum(float v) {
  return __uint_as_float(half_all(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
// the larger of two neighbours first
__device__ __forceinline__ void in_order(uint32_t &a, uint32_t &b) {
  const uint32_t top = max(a, b);
  b = min(a, b);
  a = top;
}

// Rules with a bias, two tokens a wavefront: lane 32 h + i holds experts Q i .. of the h-th. A key's lowest three bits give way to its
// place in the lane (its f32 is then 2^-21 of itself too low at most, which the margin counts), so that a lane's keys are sorted as they
// are, and the lane whose first is the half's largest writes its expert to LDS and moves its keys up.
template <int Q>
__global__ __launch_bounds__(1024) void k_route_pairs(RouteRule r, const float *logits, uint32_t T, int E, int32_t *idx, float *w, int32_t *counts) {
  constexpr int QF = Q / 2;  // experts a lane where a wavefront takes one token
  extern __shared__ __align__(16) uint8_t s_mem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hl = lane & 31, half = lane >> 5;
  uint2 *s_slot = (uint2 *)s_mem + wave * 64;                                           // [16 wavefronts][2][32] key, expert
  int *s_count = (int *)(s_mem + 16 * 64 * 8);                                          // [32 Q]
  double *s_key = (double *)(s_mem + 16 * 64 * 8 + 32 * Q * 4) + (size_t)wave * 64 * QF;  // of a rule with groups
  float bias[Q];
  load_logits<Q>(r.bias, E, hl, bias);
  if (counts)
    for (int e = threadIdx.x; e < E; e += 1024) s_count[e] = 0;
  __syncthreads();
  const int lanes = E / r.groups / Q;  // of a group (the launch sees to it that groups share none)
  const uint32_t step = gridDim.x * 32;
  float next[Q];
  uint32_t t0 = (blockIdx.x * 16 + wave) * 2;
  if (t0 < T) load_logits<Q>(logits + (size_t)min(t0 + half, T - 1) * E, E, hl, next);
  for (; t0 < T; t0 += step) {
    const uint32_t t = min(t0 + half, T - 1);
    float l[Q], s[Q], m = -INFINITY, top = 1.0f, most = 0.0f;  // top: the largest score
#pragma unroll
    for (int q = 0; q < Q; q++) l[q] = next[q];
    if (t0 + step < T) load_logits<Q>(logits + (size_t)min(t0 + step + half, T - 1) * E, E, hl, next);
#pragma unroll
    for (int q = 0; q < Q; q++) {
      l[q] = fmaxf(l[q], -INFINITY);
      m = fmaxf(m, l[q]);
    }
    if (r.score == MOE_SCORE_SIGMOID) {
#pragma unroll
      for (int q = 0; q < Q; q++) s[q] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[q] * -1.44269504f));
    } else {
      m = half_max(m);
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < Q; q++) {
        s[q] = l[q] == m ? 1.0f : __builtin_amdgcn_exp2f((l[q] - m) * 1.44269504f);
        sum = sum + (l[q] == -INFINITY ? 0.0f : s[q]);
      }
      top = __builtin_amdgcn_rcpf(half_sum(sum));
#pragma unroll
      for (int q = 0; q < Q; q++) s[q] = s[q] * top;
    }
    uint32_t k[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) {
      s[q] = s[q] + bias[q];
      s[q] = l[q] == -INFINITY ? -INFINITY : fmaxf(s[q], -INFINITY);  // (a NaN bias: never)
      most = fmaxf(most, s[q] > -INFINITY ? fabsf(s[q]) : 0.0f);
      const uint32_t o = order32(s[q]);
      k[q] = o ? (o & ~7u) | (7 - q) : 0u;
    }
    most = half_max(most);
    const float gap = 0x1.4p-18f * (top + most);
    bool unsure = !(most < INFINITY);
    if (r.groups > 1) {
      float best = -INFINITY, second = -INFINITY;
      auto take = [&](float b, float n) {  // the two largest of best >= second and b >= n
        second = fmaxf(fminf(best, b), fmaxf(second, n));
        best = fmaxf(best, b);
      };
#pragma unroll
      for (int q = 0; q < Q; q++) {
        second = fmaxf(second, fminf(best, s[q]));
        best = fmaxf(best, s[q]);
      }
      if (lanes > 1) take(dpp32<0xB1>(best), dpp32<0xB1>(second));
      if (lanes > 2) take(dpp32<0x4E>(best), dpp32<0x4E>(second));
      if (lanes > 4) take(dpp32<0x141>(best), dpp32<0x141>(second));
      if (lanes > 8) take(dpp32<0x140>(best), dpp32<0x140>(second));
      const float g = r.two && second > -INFINITY ? best + second : best;
      const int mine = hl / lanes;
      int before = 0;
      bool close = false;
      for (int i = 0; i < r.groups; i++) {
        const float o0 = lane32(g, i * lanes), o1 = lane32(g, 32 + i * lanes), o = half ? o1 : o0;
        before += o > g || (o == g && i < mine);
        close |= i != mine && !(fabsf(o - g) > 2.0f * gap);
      }
      unsure |= close && mine < r.groups && g > -INFINITY;
      if (mine >= r.groups || before >= r.top_groups)
#pragma unroll
        for (int q = 0; q < Q; q++) k[q] = 0;
    }
    // a lane's keys in falling order
    if constexpr (Q == 2) {
      in_order(k[0], k[1]);
    } else {
#pragma unroll
      for (int h = 0; h < Q; h += 4) {
        in_order(k[h], k[h + 1]), in_order(k[h + 2], k[h + 3]);
        in_order(k[h], k[h + 2]), in_order(k[h + 1], k[h + 3]);
        in_order(k[h + 1], k[h + 2]);
      }
      if constexpr (Q == 8) {  // two sorted fours: the upper's and the lower's, then each (odd-even merge)
#pragma unroll
        for (int i = 0; i < 4; i++) in_order(k[i], k[i + 4]);
        in_order(k[2], k[4]), in_order(k[3], k[5]);
        in_order(k[1], k[2]), in_order(k[3], k[4]), in_order(k[5], k[6]);
      }
    }
    s_slot[lane] = make_uint2(0u, 0xFFFFFFFFu);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint32_t twice[2] = {0, 0};  // not 0: two keys of a half were the same, and left together
    for (int j = 0; j < r.k; j++) {
      const uint32_t first = half_max_u32(k[0]);
      const bool mine = k[0] == first && first != 0;
      const uint64_t who = __ballot(mine);
      const uint32_t who0 = (uint32_t)who, who1 = (uint32_t)(who >> 32);
      twice[0] |= who0 & (who0 - 1);
      twice[1] |= who1 & (who1 - 1);
      if (mine) s_slot[half * 32 + j] = make_uint2(first, (uint32_t)(hl * Q + 7) - (first & 7));
      const uint32_t up = mine ? 0xFFFFFFFFu : 0u;  // (as a mask: of a choice between neighbours the compiler makes one among all)
#pragma unroll
      for (int q = 0; q < Q - 1; q++) k[q] = (k[q + 1] & up) | (k[q] & ~up);
      k[Q - 1] &= ~up;
    }
    const uint32_t left = half_max_u32(k[0]);  // the first one left out
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint2 chosen = s_slot[lane];
    int slot = hl < r.k ? (int)chosen.y : -1;
    const uint32_t after = hl + 1 < r.k ? s_slot[min(lane + 1, 63)].x : left;
    unsure |= (half ? twice[1] : twice[0]) != 0;
    // (a slot without an expert is far from all; keys as they are without their lowest bits)
    unsure |= hl < r.k && after != 0 && !(of_order32(chosen.x & ~7u) - of_order32(after & ~7u) > gap);
    const uint64_t again = __ballot(unsure);
#pragma unroll 1
    for (int h = 0; again && h < 2; h++) {
      if (!(uint32_t)(again >> 32 * h)) continue;
      const uint32_t at = min(t0 + h, T - 1);
      float lf[QF], bf[QF], mf = -INFINITY;
      load_logits<QF>(logits + (size_t)at * E, E, lane, lf);
      load_logits<QF>(r.bias, E, lane, bf);
#pragma unroll
      for (int q = 0; q < QF; q++) {
        lf[q] = fmaxf(lf[q], -INFINITY);
        mf = fmaxf(mf, lf[q]);
      }
      const int of = __shfl(choose_exact<QF>(r, E, lane, lf, bf, wave_largest(mf), s_key), hl);
      if (half == h) slot = hl < r.k ? of : -1;
    }
    // the chosen scores, a lane a slot
    const float logit = slot >= 0 ? fmaxf(logits[(size_t)t * E + slot], -INFINITY) : -INFINITY;  // (in a cache)
    double sc = 0.0;
    if (slot >= 0) sc = r.score == MOE_SCORE_SIGMOID ? sigmoid64((double)logit) : logit == m ? 1.0 : exp64((double)logit - (double)m);
    if (r.normalize) {
      const bool sigmoid = r.score == MOE_SCORE_SIGMOID;
      const uint64_t near = __ballot(slot >= 0 && (sigmoid ? (double)logit >= kFar : sc > kLeast));
      if (!(uint32_t)near || !(uint32_t)(near >> 32)) {
        const double top = (double)half_max(logit);
        if (!(uint32_t)(near >> 32 * half)) sc = slot >= 0 && (sigmoid || top - (double)m >= kGone) ? exp64((double)logit - top) : 0.0;
      }
      const double run = row_sum64(sc), s0 = lane64(run, 15) + lane64(run, 31), s1 = lane64(run, 47) + lane64(run, 63), total = half ? s1 : s0;
      const uint32_t n = __popc((uint32_t)(__ballot(slot >= 0) >> 32 * half));
      sc = total > 0.0 ? sc / total : 1.0 / max(n, 1u);
    }
    if (hl < r.k && t0 + half < T) {
      idx[(size_t)t * r.k + hl] = slot;
      w[(size_t)t * r.k + hl] = slot >= 0 ? (float)(sc * (double)r.scale) : 0.0f;
      if (counts && slot >= 0) atomicAdd(s_count + slot, 1);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  if (counts) {
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 1024)
      if (s_count[e]) atomicAdd(counts + e, s_count[e]);
  }
}

// With w_j = scale s_j / S (S the chosen scores' sum, or 1):
//   d / d s_j = scale / S dw_j - (normalised) sum_i dw_i w_i / S,
//   sigmoid: d l_j = d s_j s_j (1 - s_j);  softmax: d l_e = s_e (d s_e - sum_j d s_j s_j).
// Of a normalised softmax that sum is 0, and S stands for its denominator, too: as for a sigmoid, the chosen experts' logits are
// all that is read (under a bias the others' largest as well, 10.0 us for 8.8 of the case below: it tells whether the chosen scores count as 0),
// and the other gradients are 0: the chosen ones' go to their places through LDS (13 us for 16384 tokens of 256 experts
// if every lane looks for its own among all, with 64-bit sums, so 8.4). An expert that idx names twice gets their sum.
template <int Q, bool DENSE>  // DENSE: a softmax without normalisation, all of whose experts have a gradient
__global__ __launch_bounds__(256) void k_route_rule_backward(RouteRule r, const float *logits, const int32_t *idx, const float *dw, uint32_t T,
                                                             int E, float *dl) {
  __shared__ float s_out[4][64 * Q];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float *s_row = s_out[wave];
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
      if (r.normalize && !__any((double)lg >= kFar)) {
        const double top = (double)wave_largest(lg);
        sc = lg == -INFINITY ? 0.0 : exp64((double)lg - top);
      }
    } else {
      m = lg;
      if constexpr (DENSE) {
        load_logits<Q>(logits + (size_t)t * E, E, lane, l);
#pragma unroll
        for (int q = 0; q < Q; q++) {
          l[q] = fmaxf(l[q], -INFINITY);
          m = fmaxf(m, l[q]);
        }
      }
      m = wave_largest(m);
      sc = lg == -INFINITY ? 0.0 : lg == m ? 1.0 : exp64((double)lg - (double)m);
      if (!DENSE && r.bias) {  // (under a bias all chosen scores may be 0: their weights are uniform, whatever the logits)
        float all[Q], top = -INFINITY;
        load_logits<Q>(logits + (size_t)t * E, E, lane, all);
#pragma unroll
        for (int q = 0; q < Q; q++) top = fmaxf(top, all[q]);
        if ((double)m - (double)wave_largest(top) < kGone) sc = 0.0;
      }
      if constexpr (DENSE) {
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
    struct __attribute__((packed, aligned(4))) some { float v[Q]; };
    some o;
    bool twice = true;
    if constexpr (!DENSE) {
      ds = ds * sc * rest;
#pragma unroll
      for (int q = 0; q < Q; q++) s_row[lane * Q + q] = 0.0f;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (e >= 0) s_row[e] = __int_as_float(lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      twice = __any(e >= 0 && __float_as_int(s_row[max(e, 0)]) != lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (e >= 0) s_row[e] = (float)ds;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int q = 0; q < Q; q++) {
        o.v[q] = s_row[lane * Q + q];
        g[q] = 0.0;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else {
      const double mean = slots_sum64(ds * sc);
#pragma unroll
      for (int q = 0; q < Q; q++) g[q] = g[q] * sum * -mean;
      ds = ds * sc;
    }
    if (twice) {
      for (int j = 0; j < r.k; j++) {
        const int ej = __builtin_amdgcn_readlane(e, j);
        const double v = lane64(ds, j);
        if (ej < 0) continue;
#pragma unroll
        for (int q = 0; q < Q; q++)
          if (q == ej % Q && lane == ej / Q) g[q] = g[q] + v;
      }
#pragma unroll
      for (int q = 0; q < Q; q++) o.v[q] = (float)g[q];
    }
    float *out = dl + (size_t)t * E + lane * Q;
    if (lane * Q + Q <= E) {
      *(some *)out = o;
    } else {
#pragma unroll
      for (int q = 0; q < Q; q++)
        if (lane * Q + q < E) out[q] = o.v[q];
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
  const int QP = E <= 64 ? 2 : E <= 128 ? 4 : 8, lanes = E / r.groups / QP;
  const bool own_lanes = r.groups == 1 || (lanes * QP * r.groups == E && lanes <= 16 && !(lanes & (lanes - 1)));
  // (16384 tokens of 256, 128 and 64 experts 22.6, 20.1 and 14.7 us, one a wavefront 33.1, 27.8 and 20.9; 4096 of 64 10.5 and 11.4; 2000 of 256
  // 15.4 and 14.1, of 128 9.3 and 8.8)
  if (r.bias && E <= 256 && T >= 4096 && own_lanes && (r.score == MOE_SCORE_SIGMOID || r.normalize)) {
    const size_t lds = 16 * 64 * 8 + 128 * (size_t)QP + (r.groups > 1 ? (size_t)16 * 256 * QP : 0);
    const unsigned grid = (unsigned)std::min<size_t>((T + 31) / 32, 256);
    auto go = [&](auto k) { return launch_own(k, grid, 1024, lds, s, r, logits, (uint32_t)T, E, idx, w, counts); };
    return QP == 2 ? go(k_route_pairs<2>) : QP == 4 ? go(k_route_pairs<4>) : go(k_route_pairs<8>);
  }
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
  auto by_score = [&](auto dense, auto other) { return r.score == MOE_SCORE_SOFTMAX && !r.normalize ? go(dense) : go(other); };
  return E <= 64    ? by_score(k_route_rule_backward<1, true>, k_route_rule_backward<1, false>)
         : E <= 128 ? by_score(k_route_rule_backward<2, true>, k_route_rule_backward<2, false>)
         : E <= 256 ? by_score(k_route_rule_backward<4, true>, k_route_rule_backward<4, false>)
         : E <= 512 ? by_score(k_route_rule_backward<8, true>, k_route_rule_backward<8, false>)
                    : by_score(k_route_rule_backward<16, true>, k_route_rule_backward<16, false>);
}

}  // namespace moe
