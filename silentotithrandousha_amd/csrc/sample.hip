// A token from each row of logits: temperature, top-k, top-p, min-p, and a random number that says where in the
// vocabulary's running sum of probabilities the token lies.
//
// With m the row's largest logit, a token's mass is 2^s exp((l - m) / temperature) rounded to a whole number (s = 44, less for a
// vocabulary above 2^18): sums of masses are whole numbers of 64 bits, exact and the same in any order, so that workgroups can
// add them up as they come. The exponential takes 64-bit arithmetic (relative error below 2^-44).
//
// top-k, top-p and min-p each leave a first part of the row's falling order, so the tokens left are those above some
// logit, and of those equal to it the first few. To find it without sorting, logits are counted (and their masses summed)
// in 2047 bins of 1/64 of (m - l) / temperature; what lies beyond, 32 temperatures below m, has mass 0 and never matters. The
// border of top-k or top-p lies in one bin, whose tokens are gathered and searched digit by digit.
//
// Launches: largest logits of chunks; masses or bins; masses above the border's bin and the tokens in it; the draw, a
// workgroup a row. A workgroup takes a chunk of 8192 logits.
#include <algorithm>

#include "device.hpp"
#include "serve.hpp"

namespace moe {
namespace {

constexpr int kChunk = 8192, kThreads = 256, kEach = kChunk / kThreads;
constexpr int kBins = 2048, kTail = kBins - 1;  // bin kTail: mass 0, not counted
constexpr int kList = 4096;                     // tokens of a border's bins that are gathered

// Workspace of a launch over T rows.
struct Work {
  float *max;        // [T][chunks] largest logit of a chunk
  uint32_t *first;   // and its first place
  uint64_t *mass;    // [T][chunks]
  uint64_t *bin_mass;   // [T][kBins]
  uint32_t *bin_count;  // [T][kBins]
  uint2 *list;          // [T][kList] key, place
  uint32_t *listed;     // [T]
};
MOE_HD size_t work_layout(Work &w, char *p, size_t T, size_t chunks) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char *q = p + off;
    off += (bytes + 255) / 256 * 256;
    return q;
  };
  w.mass = (uint64_t *)take(T * chunks * 8);
  w.max = (float *)take(T * chunks * 4);
  w.first = (uint32_t *)take(T * chunks * 4);
  w.bin_mass = (uint64_t *)take(T * kBins * 8);
  w.bin_count = (uint32_t *)take(T * kBins * 4);
  w.list = (uint2 *)take(T * kList * 8);
  w.listed = (uint32_t *)take(T * 4);
  return off;
}

struct Args {
  moe_sampling rule;
  const float *logits;
  size_t ld;
  const float *u;
  uint32_t V, chunks;
  int shift;
  int32_t *tokens;
  float *logprob;
  Work w;
};

// f32 as a number whose order is the floats' (-0 as 0), and back.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }

// What a row's settings make of its logits.
struct Row {
  float m, bins;  // largest logit; bins a unit of (m - l) / 2
  double scale;   // log2 e / temperature
  double unit;    // 2^shift
  double p, min_p;
  uint32_t k;
  bool greedy, by_k, by_p;
  __device__ __forceinline__ void set(const Args &a, uint32_t t, float largest) {
    m = largest;
    const float temperature = a.rule.temperature ? a.rule.temperature[t] : 1.0f;
    greedy = !(temperature > 0.0f);
    bins = fminf(128.0f / temperature, 3e38f);
    scale = 1.4426950408889634 / (double)temperature;
    unit = (double)((uint64_t)1 << a.shift);
    const int kk = a.rule.top_k ? a.rule.top_k[t] : 0;
    by_k = kk > 0 && (uint32_t)kk < a.V;
    k = (uint32_t)kk;
    const float pp = a.rule.top_p ? a.rule.top_p[t] : 1.0f;
    by_p = pp < 1.0f;
    p = fmax((double)pp, 0.0);
    const float mp = a.rule.min_p ? a.rule.min_p[t] : 0.0f;
    min_p = mp > 0.0f ? (double)mp : 0.0;
  }
  __device__ __forceinline__ bool cut() const { return by_k || by_p; }
  // exp((l - m) / temperature) as 2^(n + f), n whole and f in [-1/2, 1/2]: the Taylor series of 2^f to the 12th power is
  // within 2^-52. l is not NaN.
  __device__ __forceinline__ double weight(float l) const {
    if (l == m) return 1.0;
    const double x = fmax(((double)l - (double)m) * scale, -1000.0);
    const double n = rint(x), f = (x - n) * 0.6931471805599453;
    double r = 1.0 / 479001600.0;
    r = fma(r, f, 1.0 / 39916800.0);
    r = fma(r, f, 1.0 / 3628800.0);
    r = fma(r, f, 1.0 / 362880.0);
    r = fma(r, f, 1.0 / 40320.0);
    r = fma(r, f, 1.0 / 5040.0);
    r = fma(r, f, 1.0 / 720.0);
    r = fma(r, f, 1.0 / 120.0);
    r = fma(r, f, 1.0 / 24.0);
    r = fma(r, f, 1.0 / 6.0);
    r = fma(r, f, 0.5);
    r = fma(r, f, 1.0);
    r = fma(r, f, 1.0);
    return r * __builtin_bit_cast(double, (uint64_t)(1023 + (int)n) << 52);
  }
  __device__ __forceinline__ uint64_t whole(double e) const {  // round(e 2^shift): the low bits of 2^52 + that
    return __builtin_bit_cast(uint64_t, fma(e, unit, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
  }
  __device__ __forceinline__ uint64_t mass(float l) const { return whole(weight(l)); }
  // what is left of it by min_p (a largest logit always stays)
  __device__ __forceinline__ uint64_t left(float l) const {
    const double e = weight(l);
    return l == m || e >= min_p ? whole(e) : 0;
  }
  __device__ __forceinline__ int bin(float l) const {
    return l == m ? 0 : (int)fminf((0.5f * m - 0.5f * l) * bins, (float)kTail);  // (halves: their difference is finite)
  }
};

// Four logits of a row from place i, -inf past its end and for a NaN.
__device__ __forceinline__ float4 load4(const float *row, uint32_t i, uint32_t V) {
  struct __attribute__((packed, aligned(4))) four { float v[4]; };
  float4 r = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  if (i + 4 <= V) {
    const four f = *(const four *)(row + i);
    r = make_float4(f.v[0], f.v[1], f.v[2], f.v[3]);
  } else {
    if (i < V) r.x = row[i];
    if (i + 1 < V) r.y = row[i + 1];
    if (i + 2 < V) r.z = row[i + 2];
  }
  r.x = fmaxf(r.x, -INFINITY);
  r.y = fmaxf(r.y, -INFINITY);
  r.z = fmaxf(r.z, -INFINITY);
  r.w = fmaxf(r.w, -INFINITY);
  return r;
}

// The larger logit, of equal ones the first place.
__device__ __forceinline__ void take_larger(float &m, uint32_t &at, float o, uint32_t oat) {
  if (o > m || (o == m && oat < at)) {
    m = o;
    at = oat;
  }
}
// over the workgroup's threads; every thread gets it
__device__ __forceinline__ void block_largest(float &m, uint32_t &at) {
  __shared__ float s_m[kThreads / 64];
  __shared__ uint32_t s_at[kThreads / 64];
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) take_larger(m, at, __shfl_xor(m, x), __shfl_xor(at, x));
  if ((threadIdx.x & 63) == 0) {
    s_m[threadIdx.x >> 6] = m;
    s_at[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  m = s_m[0];
  at = s_at[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; i++) take_larger(m, at, s_m[i], s_at[i]);
  __syncthreads();
}
__device__ __forceinline__ void row_largest(const Args &a, uint32_t t, float &m, uint32_t &at) {
  m = -INFINITY;
  at = 0xFFFFFFFFu;
  for (uint32_t c = threadIdx.x; c < a.chunks; c += kThreads)
    take_larger(m, at, a.w.max[(size_t)t * a.chunks + c], a.w.first[(size_t)t * a.chunks + c]);
  block_largest(m, at);
}

__device__ __forceinline__ uint64_t wave_add(uint64_t v) {
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) v += __shfl_xor((unsigned long long)v, x);
  return v;
}
__device__ __forceinline__ uint64_t block_add(uint64_t v) {
  __shared__ uint64_t s[kThreads / 64];
  v = wave_add(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t r = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; i++) r += s[i];
  return r;
}
// the sum of the threads before this one
__device__ __forceinline__ uint64_t block_before(uint64_t v) {
  __shared__ uint64_t s[kThreads / 64];
  uint64_t run = v;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = __shfl_up((unsigned long long)run, d);
    if (lane >= d) run += o;
  }
  __syncthreads();
  if (lane == 63) s[wave] = run;
  __syncthreads();
  uint64_t before = run - v;
  for (int i = 0; i < wave; i++) before += s[i];
  return before;
}

__global__ __launch_bounds__(kThreads) void k_sample_max(Args a) {
  const uint32_t c = blockIdx.x, t = blockIdx.y;
  const float *row = a.logits + t * a.ld;
  float4 v[kEach / 4];
#pragma unroll
  for (int j = 0; j < kEach / 4; j++) v[j] = load4(row, min(c * kChunk + j * 4 * kThreads + threadIdx.x * 4, a.V), a.V);
  float m = -INFINITY;
  uint32_t at = 0xFFFFFFFFu;
#pragma unroll
  for (int j = 0; j < kEach / 4; j++) {
    const uint32_t i = c * kChunk + j * 4 * kThreads + threadIdx.x * 4;
    // (places rise: an equal logit does not replace one)
    if (v[j].x > m) m = v[j].x, at = i;
    if (v[j].y > m) m = v[j].y, at = i + 1;
    if (v[j].z > m) m = v[j].z, at = i + 2;
    if (v[j].w > m) m = v[j].w, at = i + 3;
  }
  block_largest(m, at);
  if (threadIdx.x == 0) {
    a.w.max[(size_t)t * a.chunks + c] = m;
    a.w.first[(size_t)t * a.chunks + c] = at;
  }
  // the row's bins, a part by each of its workgroups
  for (uint32_t b = c * kThreads + threadIdx.x; b < kBins; b += a.chunks * kThreads) {
    a.w.bin_mass[(size_t)t * kBins + b] = 0;
    a.w.bin_count[(size_t)t * kBins + b] = 0;
  }
  if (c == 0 && threadIdx.x == 0) a.w.listed[t] = 0;
}

__global__ __launch_bounds__(kThreads) void k_sample_mass(Args a) {
  const uint32_t c = blockIdx.x, t = blockIdx.y;
  __shared__ unsigned long long s_mass[kBins];
  __shared__ uint32_t s_count[kBins];
  float m;
  uint32_t at;
  row_largest(a, t, m, at);
  Row r;
  r.set(a, t, m);
  if (r.greedy || m == -INFINITY) return;
  const float *row = a.logits + t * a.ld;
  const bool cut = r.cut();
  if (cut) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      s_mass[b] = 0;
      s_count[b] = 0;
    }
    __syncthreads();
  }
  uint64_t sum = 0;
  for (int j = 0; j < kEach / 4; j++) {
    const uint32_t i = c * kChunk + j * 4 * kThreads + threadIdx.x * 4;
    const float4 v = load4(row, min(i, a.V), a.V);
    const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int x = 0; x < 4; x++) {
      if (l[x] == -INFINITY) continue;
      if (!cut) {
        sum += r.left(l[x]);
        continue;
      }
      const int b = r.bin(l[x]);
      if (b == kTail) continue;
      atomicAdd(s_count + b, 1u);
      if (r.by_p) atomicAdd(s_mass + b, (unsigned long long)r.mass(l[x]));
    }
  }
  if (!cut) {
    sum = block_add(sum);
    if (threadIdx.x == 0) a.w.mass[(size_t)t * a.chunks + c] = sum;
    return;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kTail; b += kThreads)
    if (s_count[b]) {
      atomicAdd(a.w.bin_count + (size_t)t * kBins + b, s_count[b]);
      if (r.by_p) atomicAdd((unsigned long long *)a.w.bin_mass + (size_t)t * kBins + b, s_mass[b]);
    }
}

// A row's bins as a workgroup holds them: each thread 8 neighbours, their running sums. Bins end at the first whose
// running count (mass) reaches a target.
struct Bins {
  static constexpr int kPer = kBins / kThreads;
  uint32_t count[kPer];
  uint64_t mass[kPer];
  struct Found {
    int bin;                 // kTail: the target is not reached
    uint32_t count;          // before it
    uint64_t mass, through;  // before it, and with it
  };
  __device__ __forceinline__ void load(const Args &a, uint32_t t) {
    uint64_t m = 0, n = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const size_t b = (size_t)t * kBins + threadIdx.x * kPer + i;
      n += a.w.bin_count[b];
      m += a.w.bin_mass[b];
      count[i] = (uint32_t)n;
      mass[i] = m;
    }
    const uint32_t n0 = (uint32_t)block_before(n);
    const uint64_t m0 = block_before(m);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      count[i] += n0;
      mass[i] += m0;
    }
    before_count = n0;
    before_mass = m0;
  }
  uint32_t before_count;
  uint64_t before_mass;
  template <class F>
  __device__ __forceinline__ Found first(F &&reached) const {
    __shared__ Found s_f;
    __syncthreads();
    if (threadIdx.x == kThreads - 1) s_f = Found{kTail, count[kPer - 1], mass[kPer - 1], mass[kPer - 1]};
    __syncthreads();
    bool was = reached(before_count, before_mass);
    uint32_t n = before_count;
    uint64_t m = before_mass;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const bool is = reached(count[i], mass[i]);
      if (is && !was) s_f = Found{(int)threadIdx.x * kPer + i, n, m, mass[i]};
      was = is;
      n = count[i];
      m = mass[i];
    }
    __syncthreads();
    return s_f;
  }
};

// The bins in which a row's border may lie: that of top-k, and those of top-p for every sum that top-k may leave.
struct Border {
  Bins::Found k;    // of top-k (kTail: it leaves all that has mass)
  int p_low, p_high;
  int lowest;       // bins before it are left whole
  __device__ __forceinline__ void find(const Bins &b, const Row &r) {
    k = b.first([&](uint32_t n, uint64_t) { return r.by_k && n >= r.k; });
    p_low = p_high = kTail;
    lowest = k.bin;
    if (r.by_p) {
      const double low = r.p * (double)k.mass, high = r.p * (double)k.through;
      // (a bin ends the sum if it holds a token before which the sum is not below p: at least the first bin)
      p_low = min(b.first([&](uint32_t n, uint64_t m) { return n > 0 && (double)m >= low; }).bin, k.bin);
      p_high = min(b.first([&](uint32_t n, uint64_t m) { return n > 0 && (double)m >= high; }).bin, k.bin);
      lowest = min(p_low, k.bin);
    }
  }
  __device__ __forceinline__ bool holds(int bin) const { return (bin >= p_low && bin <= p_high) || bin == k.bin; }
};

__global__ __launch_bounds__(kThreads) void k_sample_border(Args a) {
  const uint32_t c = blockIdx.x, t = blockIdx.y;
  float m;
  uint32_t at;
  row_largest(a, t, m, at);
  Row r;
  r.set(a, t, m);
  if (r.greedy || m == -INFINITY || !r.cut()) return;
  Bins bins;
  bins.load(a, t);
  Border border;
  border.find(bins, r);
  const float *row = a.logits + t * a.ld;
  uint64_t sum = 0;
  for (int j = 0; j < kEach / 4; j++) {
    const uint32_t i = c * kChunk + j * 4 * kThreads + threadIdx.x * 4;
    const float4 v = load4(row, min(i, a.V), a.V);
    const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int x = 0; x < 4; x++) {
      if (l[x] == -INFINITY) continue;
      const int b = r.bin(l[x]);
      if (b == kTail) continue;
      if (b < border.lowest) sum += r.left(l[x]);
      if (border.holds(b)) {
        const uint32_t n = atomicAdd(a.w.listed + t, 1u);
        if (n < kList) a.w.list[(size_t)t * kList + n] = make_uint2(key_of(l[x]), i + x);
      }
    }
  }
  sum = block_add(sum);
  if (threadIdx.x == 0) a.w.mass[(size_t)t * a.chunks + c] = sum;
}

// The border among the tokens that `each` goes through (each(f): f(key, place) for this thread's share): the largest
// key at which the count or mass from above reaches a target, digit by digit.
struct Digits {
  uint32_t key;     // that key
  uint64_t before;  // what lies above it
  uint64_t here;    // and what has it
  uint32_t ties;    // tokens that have it
  template <class E, class W, class R>
  __device__ __forceinline__ void find(E &&each, W &&what, R &&reached) {
    __shared__ unsigned long long s_sum[256];
    __shared__ uint32_t s_ties[256];
    __shared__ uint32_t s_digit;
    __shared__ uint64_t s_before;
    key = 0;
    before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      s_sum[threadIdx.x] = 0;
      s_ties[threadIdx.x] = 0;
      __syncthreads();
      each([&](uint32_t k, uint32_t place) {
        if (shift < 24 && (k >> (shift + 8)) != (key >> (shift + 8))) return;
        atomicAdd(s_sum + (k >> shift & 255), (unsigned long long)what(k, place));
        atomicAdd(s_ties + (k >> shift & 255), 1u);
      });
      __syncthreads();
      if (threadIdx.x == 0) {  // (the last digit that holds a token, if none reaches the target)
        uint64_t sum = before, at = before;
        uint32_t digit = 0;
        for (int d = 255; d >= 0; d--) {
          if (!s_ties[d]) continue;
          digit = d;
          at = sum;
          sum += s_sum[d];
          if (reached(sum)) break;
        }
        s_digit = digit;
        s_before = at;
      }
      __syncthreads();
      key |= s_digit << shift;
      before = s_before;
      here = s_sum[s_digit];
      ties = s_ties[s_digit];
    }
    __syncthreads();
  }
};

__global__ __launch_bounds__(kThreads) void k_sample_draw(Args a) {
  const uint32_t t = blockIdx.x;
  float m;
  uint32_t at;
  row_largest(a, t, m, at);
  Row r;
  r.set(a, t, m);
  if (m == -INFINITY || r.greedy) {
    if (threadIdx.x == 0) {
      a.tokens[t] = m == -INFINITY ? -1 : (int32_t)at;
      if (a.logprob) a.logprob[t] = m == -INFINITY ? NAN : 0.0f;
    }
    return;
  }
  const float *row = a.logits + t * a.ld;
  uint64_t *mass = a.w.mass + (size_t)t * a.chunks;
  // tokens above `key` are left, and of those equal to it the ones up to `last`
  uint32_t key = 0, last = 0xFFFFFFFFu;
  if (r.cut()) {
    Bins bins;
    bins.load(a, t);
    Border border;
    border.find(bins, r);
    const uint32_t n = a.w.listed[t];
    const uint2 *list = a.w.list + (size_t)t * kList;
    // the tokens of the border's bins: the list, or the row again if they are too many
    auto each = [&](auto &&f) {
      if (n <= kList) {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) f(list[i].x, list[i].y);
      } else {
        for (uint32_t i = threadIdx.x; i < a.V; i += kThreads) {
          const float l = fmaxf(row[i], -INFINITY);
          if (l == -INFINITY) continue;
          const int b = r.bin(l);
          if (b != kTail && border.holds(b)) f(key_of(l), i);
        }
      }
    };
    auto in_bin = [&](int bin) {
      return [&, bin](auto &&f) {
        each([&](uint32_t k, uint32_t place) {
          if (r.bin(of_key(k)) == bin) f(k, place);
        });
      };
    };
    uint32_t keep = 0;  // of the tokens equal to `key`
    bool found = false;
    uint64_t Z = border.k.through;  // the masses that top-k leaves
    if (border.k.bin != kTail) {
      const uint32_t want = r.k - border.k.count;
      Digits d;
      d.find(in_bin(border.k.bin), [](uint32_t, uint32_t) { return 1ull; }, [&](uint64_t s) { return s >= want; });
      key = d.key;
      keep = want - (uint32_t)d.before;
      found = true;
      if (r.by_p) {
        uint64_t sum = 0;
        in_bin(border.k.bin)([&](uint32_t k, uint32_t) {
          if (k > key) sum += r.mass(of_key(k));
        });
        Z = border.k.mass + block_add(sum) + keep * r.mass(of_key(key));
      }
    }
    if (r.by_p) {
      const double P = r.p * (double)Z;
      const Bins::Found b = bins.first([&](uint32_t c, uint64_t s) { return c > 0 && (double)s >= P; });
      const int bin = min(b.bin, border.k.bin);
      if (bin != kTail) {
        Digits d;
        d.find(in_bin(bin), [&](uint32_t k, uint32_t) { return r.mass(of_key(k)); },
               [&](uint64_t s) { return (double)(b.mass + s) >= P; });
        // of equal tokens the i-th is left if the sum before it, before + i one, is below P
        const uint64_t one = d.here / max(d.ties, 1u);
        uint64_t few = d.ties;
        if (one) {
          const double rest = (P - (double)(b.mass + d.before)) / (double)one;
          few = rest > 0.0 ? (uint64_t)fmin(ceil(rest), (double)d.ties) : 0;
        }
        few = max(few, (uint64_t)1);
        if (!found || d.key > key || (d.key == key && few < keep)) {
          key = d.key;
          keep = (uint32_t)few;
        }
        found = true;
      }
    }
    if (found) {
      Digits d;  // the keep-th place of those equal to key
      d.find([&](auto &&f) { each([&](uint32_t k, uint32_t place) { if (k == key) f(~place, place); }); },
             [](uint32_t, uint32_t) { return 1ull; }, [&](uint64_t s) { return s >= keep; });
      last = ~d.key;
    }
    // their masses, beside those of the bins before
    each([&](uint32_t k, uint32_t place) {
      if (r.bin(of_key(k)) >= border.lowest && (k > key || (k == key && place <= last)))
        atomicAdd((unsigned long long *)mass + place / kChunk, (unsigned long long)r.left(of_key(k)));
    });
    __threadfence();
    __syncthreads();
  }
  // the chunk in which the running sum passes u
  __shared__ uint32_t s_chunk;
  __shared__ uint64_t s_rest;
  uint64_t total = 0;
  for (uint32_t c = threadIdx.x; c < a.chunks; c += kThreads) total += __hip_atomic_load(mass + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  total = block_add(total);
  const double u = fmin(fmax((double)a.u[t], 0.0), 1.0);
  uint64_t target = min((uint64_t)(u * (double)total), total - 1);
  uint64_t base = 0;
  for (uint32_t c0 = 0; c0 < a.chunks; c0 += kThreads) {
    const uint32_t c = c0 + threadIdx.x;
    const uint64_t v = c < a.chunks ? __hip_atomic_load(mass + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    const uint64_t before = base + block_before(v);
    if (before <= target && target < before + v) {
      s_chunk = c;
      s_rest = target - before;
    }
    base += block_add(v);
  }
  __syncthreads();
  // and the token in it, a thread 32 neighbours
  const uint32_t i0 = s_chunk * kChunk + threadIdx.x * kEach;
  const uint64_t rest = s_rest;
  uint64_t masses[kEach], sum = 0;
#pragma unroll
  for (int j = 0; j < kEach / 4; j++) {
    const float4 v = load4(row, min(i0 + 4 * j, a.V), a.V);
    const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int x = 0; x < 4; x++) {
      const uint32_t k = key_of(l[x]);
      uint64_t e = 0;
      if (l[x] != -INFINITY && (k > key || (k == key && i0 + 4 * j + x <= last))) e = r.left(l[x]);
      masses[4 * j + x] = e;
      sum += e;
    }
  }
  uint64_t before = block_before(sum);
  if (before <= rest && rest < before + sum) {
    uint32_t found = i0;
    bool done = false;
#pragma unroll
    for (int j = 0; j < kEach; j++) {
      if (!done && rest < before + masses[j]) {
        found = i0 + j;
        done = true;
      }
      before += masses[j];
    }
    a.tokens[t] = (int32_t)found;
    if (a.logprob) {
      const float l = row[found];
      const double z = l == m ? 0.0 : ((double)l - (double)m) * r.scale * 0.6931471805599453;
      a.logprob[t] = (float)(z - log((double)total / r.unit));
    }
  }
}

}  // namespace

static uint32_t sample_chunks(size_t V) { return (uint32_t)((V + kChunk - 1) / kChunk); }

size_t sample_workspace(size_t T, size_t V) {
  Work w;
  return work_layout(w, nullptr, T, sample_chunks(V));
}

hipError_t launch_sample(const SampleArgs &s, hipStream_t st) {
  if (!s.T || s.T > 65535 || !s.V || s.V > 1u << 28 || s.ld < s.V) return hipErrorInvalidValue;
  Args a{s.rule, s.logits, s.ld, s.u, s.V, sample_chunks(s.V), 44, s.tokens, s.logprob, {}};
  while (a.shift > 62 - 32 && ((uint64_t)s.V << a.shift) > (uint64_t)1 << 62) a.shift--;
  work_layout(a.w, (char *)s.work, s.T, a.chunks);
  const dim3 grid(a.chunks, s.T);
  hipError_t e = launch_own(k_sample_max, grid, kThreads, 0, st, a);
  if (e == hipSuccess) e = launch_own(k_sample_mass, grid, kThreads, 0, st, a);
  if (e == hipSuccess && (s.rule.top_k || s.rule.top_p)) e = launch_own(k_sample_border, grid, kThreads, 0, st, a);
  if (e == hipSuccess) e = launch_own(k_sample_draw, dim3(s.T), kThreads, 0, st, a);
  return e;
}

}  // namespace moe
