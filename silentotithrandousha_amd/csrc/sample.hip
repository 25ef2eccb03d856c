// A token from each row of logits: temperature, top-k, top-p, min-p, and a random number that says where in the
// vocabulary's running sum of probabilities the token lies.
//
// With m the row's largest logit, a token's mass is 2^s exp((l - m) / temperature) rounded to a whole number (s = 44, less for a
// vocabulary above 2^18): sums of masses are whole numbers of 64 bits, exact and the same in any order, so that workgroups can
// add them up as they come. The exponential takes 64-bit arithmetic where it has to: a mass is off by less than one.
//
// top-k, top-p and min-p each leave a first part of the row's falling order, so the tokens left are those above some
// logit, and of those equal to it the first few. To find it without sorting, logits are counted (and their masses summed)
// in 2047 bins of 1/64 of (m - l) / temperature; what lies beyond, 32 temperatures below m, has mass 0 and never matters. The
// border of top-k or top-p lies in one bin, whose tokens are gathered and searched digit by digit.
//
// Launches: largest logits of chunks; masses or bins; the border's tokens (and masses above them); the draw, a workgroup a
// row. A workgroup takes one or more chunks of 2048 logits. A row with a top-k of up to kFewK counts bins, no masses, and gathers all
// that top-k leaves; other rows sum masses by bin, and gather the bins that hold a border. Of a top-k well below the row's pieces
// of 256 logits even the bins are those of the pieces' largest alone: no piece below the k-th of them holds one of the k, and
// the second launch gathers from the few that may. What is gathered is sorted in LDS. Should it be more than kList tokens, the draw
// goes through the row itself, a workgroup a row: 201088 logits of deviation 1 under a temperature of 4 and a top-p of 0.6 take 0.98 ms (64 such
// rows 1.8), all equal 2.6 ms.
//
// 256 rows of 201088 logits, of which half have a top-k of 20 to 400, half a top-p: 34, 50, 20 and 18 us. The first is bound by its 206
// MB (6.1 TB/s), the second by the 64-bit arithmetic and LDS atomics of the rows without a small top-k, the third by reads through the
// last-level cache, the draw by the latency of some 40 steps that wait for each other (11 us for a single row).
#include <algorithm>

#include "device.hpp"
#include "serve.hpp"

namespace moe {
namespace {

constexpr int kThreads = 512, kChunk = 4 * kThreads;  // a thread has four logits of a chunk
constexpr int kMaxSpan = 4;                            // chunks of a workgroup that looks for the largest logit
static_assert(kThreads == 512 && kMaxSpan * kChunk == kSampleSpan, "sample_rows");
constexpr int kBins = 2048, kTail = kBins - 1;  // bin kTail: mass 0, not counted
constexpr int kList = 4096;                     // tokens that are gathered of a row
constexpr uint32_t kParts = 1024;                // chunks whose masses the draw holds in LDS
constexpr uint32_t kFewK = 2048;                // top-k up to which all that it leaves is
constexpr int kPiece = 256;                      // neighbouring logits whose largest is kept, a wavefront's of a chunk
constexpr int kPieces = 8 * kThreads;            // of a row, at most

struct RowState;

// Workspace of a launch over T rows.
struct Work {
  uint2 *largest;       // [T][groups] largest logit of kMaxSpan chunks and its first place
  float *peak;          // [T][8 chunks] largest logit of a piece
  uint64_t *mass;       // [T][chunks]
  uint64_t *bin_mass;   // [T][kBins]
  uint32_t *bin_count;  // [T][kBins]
  uint2 *list;          // [T][kList] key, place
  RowState *row;        // [T]
};

struct Args {
  moe_sampling rule;
  const float *logits;
  size_t ld;
  const float *u;
  uint32_t V, chunks, groups;
  int shift, span;  // span: chunks that a workgroup takes
  bool peaks;       // Work::peak is filled
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

// 2^(i / 32), each its nearest 64-bit number: as many as LDS has pairs of banks, so that lanes reading different ones do not wait
// for each other.
constexpr int kPowersOf2 = 32;
__device__ const double kPowers[kPowersOf2] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0,
};
// into LDS, by the workgroup's first lanes
__device__ __forceinline__ void load_powers(double *s_powers) {
  if (threadIdx.x < kPowersOf2) s_powers[threadIdx.x] = kPowers[threadIdx.x];
}

// What a row's settings make of its logits.
struct Row {
  float m, bins;        // largest logit; bins a unit of (m - l) / 2
  double scale;         // 32 log2 e / temperature
  double least;         // min_p 2^shift
  double p;
  const double *table;  // kPowers in LDS
  uint32_t k;
  int shift;
  bool greedy, by_k, by_p, few, direct;
  __device__ __forceinline__ void set(const Args &a, uint32_t t, float largest, const double *powers) {
    table = powers;
    m = largest;
    const float temperature = a.rule.temperature ? a.rule.temperature[t] : 1.0f;
    greedy = !(temperature > 0.0f);
    bins = fminf(128.0f / temperature, 3e38f);
    scale = 32 * 1.4426950408889634 / (double)temperature;
    shift = a.shift;
    const int kk = a.rule.top_k ? a.rule.top_k[t] : 0;
    by_k = kk > 0 && (uint32_t)kk < a.V;
    k = (uint32_t)kk;
    const float pp = a.rule.top_p ? a.rule.top_p[t] : 1.0f;
    by_p = pp < 1.0f;
    few = by_k && k <= kFewK;
    direct = takes_direct(a, kk);
    p = fmax((double)pp, 0.0);
    const float mp = a.rule.min_p ? a.rule.min_p[t] : 0.0f;
    least = mp > 0.0f ? (double)mp * (double)((uint64_t)1 << shift) : 0.0;
  }
  // A row whose top-k is up to half of its pieces is gathered without counting its logits: pieces whose largest is below the k-th largest of those
  // hold none of the k. (Above that, most pieces hold one, and the list of tokens above that border grows.)
  static __device__ __forceinline__ bool takes_direct(const Args &a, int k) {
    return a.peaks && k > 0 && (uint32_t)k <= kFewK && (uint32_t)k * 2 <= a.chunks * (kChunk / kPiece) && (uint32_t)k < a.V;
  }
  __device__ __forceinline__ bool cut() const { return by_k || by_p; }
  // Masses of four logits, and which of them min_p leaves (a largest logit always).
  // exp((l - m) / temperature) = 2^(k / 32) 2^(t / 32), k whole and t in [-1/2, 1/2]: 2^(k % 32 / 32) from the table, the
  // second factor its Taylor series to the fifth power, within 2^-48. (Of 12 powers without a table, 161 MB of logits
  // took 70 us.)
  __device__ __forceinline__ void masses(const float (&l)[4], uint64_t (&e)[4], bool (&stays)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      // (from 40 temperatures below the largest logit the mass is 0; a -inf lies there, under an infinite temperature too, where
      // the product is NaN)
      const double x = fmax(((double)l[i] - (double)m) * scale, -40.0 * 32 * 1.4426950408889634);
      const double r = x + 6755399441055744.0;  // 1.5 2^52: the low word is x rounded
      const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, r);
      const double t = x - (r - 6755399441055744.0);
      double p = 3.973709984549416e-11;
      p = fma(p, t, 9.172562701824643e-09);
      p = fma(p, t, 1.693850972437182e-06);
      p = fma(p, t, 0.0002345961982022468);
      p = fma(p, t, 0.02166084939249829);
      const uint64_t power = __builtin_bit_cast(uint64_t, table[k & 31]) + ((uint64_t)(uint32_t)((k >> 5) + shift) << 52);
      const double f = __builtin_bit_cast(double, power), w = fma(f, p * t, f);
      // rounded: the low bits of 2^52 + w
      e[i] = __builtin_bit_cast(uint64_t, w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
      stays[i] = least == 0.0 || l[i] == m || w >= least;
    }
    if (m == INFINITY)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        stays[i] = l[i] == m;
        e[i] = stays[i] ? (uint64_t)1 << shift : 0;
      }
  }
  __device__ __forceinline__ void left(const float (&l)[4], uint64_t (&e)[4]) const {
    bool stays[4];
    masses(l, e, stays);
#pragma unroll
    for (int i = 0; i < 4; i++) e[i] = stays[i] ? e[i] : 0;
  }
  __device__ __forceinline__ uint64_t mass(float l) const {
    uint64_t e[4];
    bool stays[4];
    masses({l, l, l, l}, e, stays);
    return e[0];
  }
  __device__ __forceinline__ uint64_t left(float l) const {
    uint64_t e[4];
    left({l, l, l, l}, e);
    return e[0];
  }
  __device__ __forceinline__ int bin(float l) const {
    return l == m ? 0 : (int)fminf((0.5f * m - 0.5f * l) * bins, (float)kTail);  // (halves: their difference is finite)
  }
};

// This thread's four logits of chunk c, as they are and -inf past the row's end; chunks past the last read the last. (What is
// done with them waits for them: it has to come after the next loads.)
__device__ __forceinline__ uint32_t place_of(uint32_t c) { return c * kChunk + threadIdx.x * 4; }
__device__ __forceinline__ float4 load_chunk(const Args &a, const float *row, uint32_t c) {
  struct __attribute__((packed, aligned(4))) four { float v[4]; };
  const uint32_t i = place_of(min(c, a.chunks - 1));
  if (c + 1 < a.chunks) {
    const four f = *(const four *)(row + i);
    return make_float4(f.v[0], f.v[1], f.v[2], f.v[3]);
  }
  float4 r = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  if (i < a.V) r.x = row[i];
  if (i + 1 < a.V) r.y = row[i + 1];
  if (i + 2 < a.V) r.z = row[i + 2];
  if (i + 3 < a.V) r.w = row[i + 3];
  return r;
}
// a NaN counts as -inf
__device__ __forceinline__ void logits_of(const float4 &v, float (&l)[4]) {
  l[0] = fmaxf(v.x, -INFINITY);
  l[1] = fmaxf(v.y, -INFINITY);
  l[2] = fmaxf(v.z, -INFINITY);
  l[3] = fmaxf(v.w, -INFINITY);
}

// The larger logit, of equal ones the first place.
__device__ __forceinline__ void take_larger(float &m, uint32_t &at, float o, uint32_t oat) {
  if (o > m || (o == m && oat < at)) {
    m = o;
    at = oat;
  }
}
// The row's largest logit from those of its groups of chunks, in every wavefront for itself.
__device__ __forceinline__ void row_largest(const Args &a, uint32_t t, float &m, uint32_t &at) {
  m = -INFINITY;
  at = 0xFFFFFFFFu;
  for (uint32_t g = threadIdx.x & 63; g < a.groups; g += 64) {
    const uint2 q = a.w.largest[(size_t)t * a.groups + g];
    take_larger(m, at, __uint_as_float(q.x), q.y);
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) take_larger(m, at, __shfl_xor(m, x), __shfl_xor(at, x));
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, true);
  return (uint64_t)hi << 32 | lo;
}
// the sum of the lanes up to this one
__device__ __forceinline__ uint64_t wave_run(uint64_t v) {
  v += dpp64<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += dpp64<0x112, 0xF>(v);
  v += dpp64<0x114, 0xF>(v);
  v += dpp64<0x118, 0xF>(v);
  v += dpp64<0x142, 0xA>(v);  // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
  v += dpp64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ uint64_t wave_add(uint64_t v) { return lane_of(wave_run(v), 63); }
// adds a wavefront's masses to its chunk's
__device__ __forceinline__ void add_mass(const Args &a, uint32_t t, uint32_t c, uint64_t sum) {
  const uint64_t some = __ballot(sum != 0);
  if (!some) return;
  const bool few = __popcll(some) <= 4;  // (their own additions are sooner done than a sum over lanes)
  if (!few) sum = wave_add(sum);
  if (few ? sum != 0 : (threadIdx.x & 63) == 0) atomicAdd((unsigned long long *)a.w.mass + (size_t)t * a.chunks + c, (unsigned long long)sum);
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
  const uint64_t run = wave_run(v);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 63) s[wave] = run;
  __syncthreads();
  uint64_t before = run - v;
  for (int i = 0; i < wave; i++) before += s[i];
  return before;
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
  __device__ __forceinline__ void load(const Args &a, uint32_t t, const Row &r) {
    uint64_t m = 0, n = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const size_t b = (size_t)t * kBins + threadIdx.x * kPer + i;
      if (r.by_k) n += __hip_atomic_load(a.w.bin_count + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (r.by_p && !r.few) m += __hip_atomic_load(a.w.bin_mass + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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

// The bins in which a row's border may lie, whose tokens are gathered.
struct Border {
  Bins::Found k;    // of top-k (kTail: it leaves all that has mass)
  int low, high;    // of top-p, for every sum that top-k may leave; of few: all that top-k may leave
  uint64_t before;  // the mass before bin `low`
  bool first;       // no token lies before it
  __device__ __forceinline__ void find(const Bins &b, const Row &r) {
    k = b.first([&](uint32_t n, uint64_t) { return r.by_k && n >= r.k; });
    before = 0;
    first = true;
    low = 0;
    high = min(k.bin, kTail - 1);
    if (r.few) return;
    low = high = kTail;
    if (r.by_p) {
      const double least = r.p * (double)k.mass, most = r.p * (double)k.through;
      // (top-p ends in the first bin through which the sum reaches p; every row leaves one token)
      const Bins::Found f = b.first([&](uint32_t, uint64_t m) { return m > 0 && (double)m >= least; });
      low = min(f.bin, k.bin);
      before = f.mass;
      first = f.mass == 0;
      high = min(b.first([&](uint32_t, uint64_t m) { return m > 0 && (double)m >= most; }).bin, k.bin);
    }
  }
  __device__ __forceinline__ int lowest() const { return min(low, k.bin); }  // bins before it are left whole
  __device__ __forceinline__ bool holds(int bin) const { return (bin >= low && bin <= high) || bin == k.bin; }
};

// What the launches leave each other of a row (a cache line apart from the next row's: every wavefront adds to it).
struct __attribute__((aligned(256))) RowState {
  uint2 largest;    // the row's largest logit and its first place
  uint32_t listed;  // tokens in its list
  uint32_t done;    // workgroups that have added their bins
  Border border;
};

// Clears a row's bins, sums and state, a part by each of the row's workgroups.
__device__ __forceinline__ void begin_row(const Args &a, uint32_t t) {
  for (uint32_t b = blockIdx.x * kThreads + threadIdx.x; b < kBins; b += gridDim.x * kThreads) {
    a.w.bin_mass[(size_t)t * kBins + b] = 0;
    a.w.bin_count[(size_t)t * kBins + b] = 0;
  }
  for (uint32_t c = blockIdx.x * kThreads + threadIdx.x; c < a.chunks; c += gridDim.x * kThreads) a.w.mass[(size_t)t * a.chunks + c] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.w.row[t].listed = a.w.row[t].done = 0;
}

__global__ __launch_bounds__(kThreads) void k_sample_max(Args a) {
  __shared__ float s_m[kThreads / 64];
  __shared__ uint32_t s_at[kThreads / 64];
  const uint32_t t = blockIdx.y, c0 = blockIdx.x * kMaxSpan;
  const float *row = a.logits + t * a.ld;
  float4 v[kMaxSpan];
#pragma unroll
  for (int j = 0; j < kMaxSpan; j++) v[j] = load_chunk(a, row, c0 + j);
  begin_row(a, t);
  float m = -INFINITY;
  uint32_t at = 0xFFFFFFFFu;
  if (a.peaks) {
#pragma unroll
    for (int j = 0; j < kMaxSpan; j++) {
      const float peak = wave_fmax_dpp(fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(fmaxf(v[j].z, v[j].w), -INFINITY)));
      if ((threadIdx.x & 63) == 0 && c0 + j < a.chunks)
        a.w.peak[((size_t)t * a.chunks + c0 + j) * (kChunk / kPiece) + (threadIdx.x >> 6)] = peak;
    }
  }
#pragma unroll
  for (int j = 0; j < kMaxSpan; j++) {
    const uint32_t i = place_of(c0 + j);
    // (places rise: an equal logit does not replace one)
    if (v[j].x > m) m = v[j].x, at = i;
    if (v[j].y > m) m = v[j].y, at = i + 1;
    if (v[j].z > m) m = v[j].z, at = i + 2;
    if (v[j].w > m) m = v[j].w, at = i + 3;
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) take_larger(m, at, __shfl_xor(m, x), __shfl_xor(at, x));
  if ((threadIdx.x & 63) == 0) {
    s_m[threadIdx.x >> 6] = m;
    s_at[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < kThreads / 64; i++) take_larger(m, at, s_m[i], s_at[i]);
    a.w.largest[(size_t)t * a.groups + blockIdx.x] = make_uint2(__float_as_uint(m), at);
  }
}

// f(chunk, its four logits) for the workgroup's chunks, two loads ahead.
template <class F>
__device__ __forceinline__ void each_chunk(const Args &a, const float *row, const float4 &first, F &&f) {
  const uint32_t c0 = blockIdx.x * a.span, c1 = min(c0 + a.span, a.chunks);
  float4 v = first, next = load_chunk(a, row, c0 + 1);
#pragma unroll 1
  for (uint32_t c = c0; c < c1; c++) {
    const float4 after = load_chunk(a, row, c + 2);
    float l[4];
    logits_of(v, l);
    f(c, l);
    v = next;
    next = after;
  }
}

// Gives the lanes of N masks places behind `n` of a list, with one atomic a wavefront: to(i, place) in the lanes of mask i.
template <int N, class F>
__device__ __forceinline__ void append(const uint64_t (&takes)[N], uint32_t *n, F &&to) {
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < N; i++) all += __popcll(takes[i]);
  if (!all) return;
  uint32_t at = 0;
  if ((threadIdx.x & 63) == 0) at = atomicAdd(n, all);
  at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (takes[i] >> (threadIdx.x & 63) & 1) to(i, at + __popcll(takes[i] & ((1ull << (threadIdx.x & 63)) - 1)));
    at += __popcll(takes[i]);
  }
}

// Into the row's list, of this workgroup's chunks: all tokens whose bin is up to that in which the k-th largest of the row's
// pieces lies, read from the pieces that hold one.
__device__ __forceinline__ void gather_few(const Args &a, uint32_t t, const Row &r, const float *row, uint32_t *s_count) {
  __shared__ uint32_t s_some;
  __shared__ uint16_t s_piece[kPieces];
  constexpr int kMine = kPieces / kThreads, kOfChunk = kChunk / kPiece;
  const uint32_t pieces = a.chunks * kOfChunk, lane = threadIdx.x & 63;
  int bin[kMine];
#pragma unroll
  for (int i = 0; i < kMine; i++) {
    const uint32_t p = i * kThreads + threadIdx.x;
    bin[i] = p < pieces ? r.bin(a.w.peak[(size_t)t * pieces + p]) : kTail;
  }
  for (int b = threadIdx.x; b < kBins; b += kThreads) s_count[b] = 0;
  if (threadIdx.x == 0) s_some = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMine; i++)
    if (bin[i] < kTail) atomicAdd(s_count + bin[i], 1u);
  __syncthreads();
  Bins bins;
  uint32_t sum = 0;
#pragma unroll
  for (int i = 0; i < Bins::kPer; i++) {
    bins.count[i] = sum += s_count[threadIdx.x * Bins::kPer + i];
    bins.mass[i] = 0;
  }
  bins.before_count = (uint32_t)block_before(sum);
  bins.before_mass = 0;
#pragma unroll
  for (int i = 0; i < Bins::kPer; i++) bins.count[i] += bins.before_count;
  const int most = min(bins.first([&](uint32_t c, uint64_t) { return c >= r.k; }).bin, kTail - 1);
  const uint32_t first = blockIdx.x * a.span * kOfChunk, last = first + a.span * kOfChunk;
  {
    uint64_t takes[kMine];
#pragma unroll
    for (int i = 0; i < kMine; i++) {
      const uint32_t p = i * kThreads + threadIdx.x;
      takes[i] = __ballot(bin[i] <= most && p >= first && p < last);
    }
    append(takes, &s_some, [&](int i, uint32_t at) { s_piece[at] = (uint16_t)(i * kThreads + threadIdx.x); });
  }
  __syncthreads();
  // a wavefront a piece, several under way
  constexpr int kAhead = 8, kWaves = kThreads / 64;
  const uint32_t some = s_some;
  for (uint32_t p0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); p0 < some; p0 += kAhead * kWaves) {
    struct __attribute__((packed, aligned(4))) four { float v[4]; };
    four f[kAhead];
    uint32_t place[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const uint32_t p = p0 + j * kWaves;
      place[j] = s_piece[min(p, some - 1)] * kPiece + lane * 4;
      f[j] = four{{-INFINITY, -INFINITY, -INFINITY, -INFINITY}};
      if (p >= some) continue;
      if (place[j] + 4 <= a.V) {
        f[j] = *(const four *)(row + place[j]);
      } else {
#pragma unroll
        for (int x = 0; x < 4; x++)
          if (place[j] + x < a.V) f[j].v[x] = row[place[j] + x];
      }
    }
    uint64_t takes[4 * kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      float l[4];
      logits_of(make_float4(f[j].v[0], f[j].v[1], f[j].v[2], f[j].v[3]), l);
#pragma unroll
      for (int x = 0; x < 4; x++) {
        f[j].v[x] = l[x];
        takes[4 * j + x] = __ballot(r.bin(l[x]) <= most);
      }
    }
    append(takes, &a.w.row[t].listed, [&](int i, uint32_t at) {
      if (at < kList) a.w.list[(size_t)t * kList + at] = make_uint2(key_of(f[i / 4].v[i % 4]), place[i / 4] + i % 4);
    });
  }
}

__global__ __launch_bounds__(kThreads) void k_sample_mass(Args a) {
  const uint32_t t = blockIdx.y;
  __shared__ unsigned long long s_mass[kBins];
  __shared__ uint32_t s_count[kBins];
  __shared__ uint32_t s_done;
  const float *row = a.logits + t * a.ld;
  __shared__ double s_powers[kPowersOf2];
  load_powers(s_powers);
  const float4 v = load_chunk(a, row, blockIdx.x * a.span);
  float m;
  uint32_t at;
  row_largest(a, t, m, at);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.w.row[t].largest = make_uint2(__float_as_uint(m), at);
  Row r;
  r.set(a, t, m, s_powers);
  if (r.greedy || m == -INFINITY) return;
  if (r.direct) {
    gather_few(a, t, r, row, s_count);
    return;
  }
  if (!r.cut()) {
    __syncthreads();
    each_chunk(a, row, v, [&](uint32_t c, const float (&l)[4]) {
      uint64_t e[4];
      r.left(l, e);
      add_mass(a, t, c, (e[0] + e[1]) + (e[2] + e[3]));
    });
    return;
  }
  const bool masses = r.by_p && !r.few;
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    s_mass[b] = 0;
    s_count[b] = 0;
  }
  __syncthreads();
  each_chunk(a, row, v, [&](uint32_t, const float (&l)[4]) {
    uint64_t e[4];
    bool stays[4];
    if (masses) r.masses(l, e, stays);
#pragma unroll
    for (int x = 0; x < 4; x++) {
      const int b = r.bin(l[x]);
      if (b == kTail) continue;
      if (r.by_k) atomicAdd(s_count + b, 1u);
      if (masses) atomicAdd(s_mass + b, (unsigned long long)e[x]);
    }
  });
  __syncthreads();
  for (int b = threadIdx.x; b < kTail; b += kThreads) {
    if (s_count[b]) atomicAdd(a.w.bin_count + (size_t)t * kBins + b, s_count[b]);
    if (s_mass[b]) atomicAdd((unsigned long long *)a.w.bin_mass + (size_t)t * kBins + b, s_mass[b]);
  }
  // the row's last workgroup finds where its border lies
  wait_mem();
  __syncthreads();
  if (threadIdx.x == 0) s_done = atomicAdd(&a.w.row[t].done, 1u);
  __syncthreads();
  if (s_done + 1 != gridDim.x) return;
  Bins bins;
  bins.load(a, t, r);
  Border border;
  border.find(bins, r);
  if (threadIdx.x == 0) a.w.row[t].border = border;
}

__device__ __forceinline__ bool row_of(const Args &a, uint32_t t, const double *powers, Row &r, uint32_t &at) {
  const uint2 q = a.w.row[t].largest;
  at = q.y;
  r.set(a, t, __uint_as_float(q.x), powers);
  return r.m != -INFINITY;
}

__global__ __launch_bounds__(kThreads) void k_sample_border(Args a) {
  __shared__ double s_powers[kPowersOf2];
  __shared__ uint2 s_held[kList];
  __shared__ uint32_t s_n, s_at;
  const uint32_t t = blockIdx.y;
  if (a.peaks && Row::takes_direct(a, a.rule.top_k[t])) return;
  load_powers(s_powers);
  if (threadIdx.x == 0) s_n = 0;
  const float *row = a.logits + t * a.ld;
  const float4 v = load_chunk(a, row, blockIdx.x * a.span);
  Row r;
  uint32_t at;
  const Border border = a.w.row[t].border;
  if (!row_of(a, t, s_powers, r, at) || r.greedy || !r.cut()) return;
  __syncthreads();
  const int lowest = border.lowest(), most = border.k.bin == kTail ? max(border.high, lowest - 1) : border.k.bin;
  // The border's tokens are noted in LDS and get their places in the row's list behind the loop: an atomic that waits
  // for its result held the stream of logits up (206 MB took 68 us).
  each_chunk(a, row, v, [&](uint32_t c, const float (&l)[4]) {
    int b[4];
    bool near = false, whole = false;
#pragma unroll
    for (int x = 0; x < 4; x++) {
      b[x] = r.bin(l[x]);
      near |= b[x] <= most;
      whole |= b[x] < lowest;
    }
    if (!__any(near)) return;  // (few logits are)
    if (__any(whole)) {
      uint64_t e[4], sum = 0;
      r.left(l, e);
#pragma unroll
      for (int x = 0; x < 4; x++) sum += b[x] < lowest ? e[x] : 0;
      add_mass(a, t, c, sum);
    }
    uint32_t n = 0;
#pragma unroll
    for (int x = 0; x < 4; x++) n += b[x] < kTail && border.holds(b[x]);
    if (!n) return;
    uint32_t place = atomicAdd(&s_n, n);
#pragma unroll
    for (int x = 0; x < 4; x++)
      if (b[x] < kTail && border.holds(b[x])) {
        if (place < kList) s_held[place] = make_uint2(key_of(l[x]), place_of(c) + x);
        place++;
      }
  });
  __syncthreads();
  if (s_n == 0) return;
  if (threadIdx.x == 0) s_at = atomicAdd(&a.w.row[t].listed, s_n);
  __syncthreads();
  for (uint32_t i = threadIdx.x, end = min(s_n, kList - min(s_at, (uint32_t)kList)); i < end; i += kThreads)
    a.w.list[(size_t)t * kList + s_at + i] = s_held[i];
}

// The largest key at which a sum over the tokens from above reaches a target, digit by digit; `each` goes through this
// thread's share of the tokens (f(key, place)).
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
      if (threadIdx.x < 256) {
        s_sum[threadIdx.x] = 0;
        s_ties[threadIdx.x] = 0;
      }
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

// Sorts 2^log n values (n >= 64) in LDS, the largest first: pairs within a wavefront's 64 values pass through
// registers.
__device__ __forceinline__ void sort_down(uint64_t *v, uint32_t n) {
  auto meet = [](uint64_t x, uint32_t i, uint32_t size, uint32_t far) {
    const uint64_t o = __shfl_xor((unsigned long long)x, (int)far);
    const bool larger = ((i & far) == 0) == ((i & size) == 0);  // this place takes the larger of the two
    return larger == (x > o) ? x : o;
  };
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {  // (n is a multiple of 64: whole wavefronts)
    uint64_t x = v[i];
#pragma unroll
    for (uint32_t size = 2; size <= 64; size <<= 1)
#pragma unroll
      for (uint32_t far = size >> 1; far; far >>= 1) x = meet(x, i, size, far);
    v[i] = x;
  }
  __syncthreads();
  for (uint32_t size = 128; size <= n; size <<= 1)
    for (uint32_t far = size >> 1; far; ) {
      if (far >= 64) {
        for (uint32_t i = threadIdx.x; i < n / 2; i += kThreads) {
          const uint32_t lo = (i / far) * 2 * far + i % far, hi = lo + far;
          const uint64_t x = v[lo], y = v[hi];
          if ((x < y) == ((lo & size) == 0)) {
            v[lo] = y;
            v[hi] = x;
          }
        }
        __syncthreads();
        far >>= 1;
      } else {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
          uint64_t x = v[i];
#pragma unroll
          for (uint32_t f = 32; f; f >>= 1) x = meet(x, i, size, f);
          v[i] = x;
        }
        __syncthreads();
        far = 0;
      }
    }
}

__global__ __launch_bounds__(kThreads) void k_sample_draw(Args a) {
  __shared__ uint64_t s_list[kList];
  const uint32_t t = blockIdx.x;
  // (what the row's list may hold, before it is known how much that is)
  const uint2 early = a.w.list[(size_t)t * kList + threadIdx.x];
  const uint32_t n = a.w.row[t].listed;
  Border border = a.w.row[t].border;
  Row r;
  uint32_t at;
  __shared__ double s_powers[kPowersOf2];
  load_powers(s_powers);
  const bool live = row_of(a, t, s_powers, r, at);
  if (r.direct) border.low = 0, border.high = kTail, border.before = 0, border.first = true;  // (k is of other rows)
  if (!live || r.greedy) {
    if (threadIdx.x == 0) {
      a.tokens[t] = live ? (int32_t)at : -1;
      if (a.logprob) a.logprob[t] = live ? 0.0f : NAN;
    }
    return;
  }
  const float *row = a.logits + t * a.ld;
  // masses of the chunks, of ordinary vocabularies in LDS
  __shared__ uint64_t s_mass[kParts];
  uint64_t *mass = a.w.mass + (size_t)t * a.chunks;
  if (a.chunks <= kParts) {
    for (uint32_t c = threadIdx.x; c < a.chunks; c += kThreads) s_mass[c] = mass[c];
    mass = s_mass;
  }
  __syncthreads();
  // tokens above `key` are left, and of those equal to it the ones up to `last`
  uint32_t key = 0, last = 0xFFFFFFFFu;
  if (r.cut()) {
    if (__builtin_expect(n <= kList, 1)) {
      uint32_t padded = 64;
      while (padded < n) padded <<= 1;
      for (uint32_t i = threadIdx.x; i < padded; i += kThreads) {
        uint64_t e = 0;  // (behind every token)
        if (i < n) {
          const uint2 q = i < kThreads ? early : a.w.list[(size_t)t * kList + i];
          e = (uint64_t)q.x << 32 | (uint32_t)~q.y;
        }
        s_list[i] = e;
      }
      __syncthreads();
      sort_down(s_list, padded);
      // A thread's neighbours of the list, in order: up to two times four.
      constexpr int kMost = kList / kThreads;
      static_assert(kMost == 8, "two groups of four");
      const uint32_t each = (padded + kThreads - 1) / kThreads, i0 = threadIdx.x * each;
      uint32_t keys[kMost];
      uint64_t e[kMost], above = 0, of_k = 0;
      bool stays[kMost];
      int bin[kMost];
      uint32_t rank = 0;  // of the first token of the border of top-k in the list
#pragma unroll
      for (int g = 0; g < kMost; g += 4) {
        float l[4];
        uint64_t e4[4] = {0, 0, 0, 0};
        bool stays4[4] = {false, false, false, false};
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const uint32_t i = i0 + g + x;
          keys[g + x] = g + x < (int)each && i < n ? (uint32_t)(s_list[i] >> 32) : 0;
          l[x] = keys[g + x] ? of_key(keys[g + x]) : -INFINITY;
          bin[g + x] = r.bin(l[x]);
          rank += bin[g + x] < border.k.bin;
        }
        if (g < (int)each) r.masses(l, e4, stays4);
#pragma unroll
        for (int x = 0; x < 4; x++) {
          e[g + x] = e4[x];
          stays[g + x] = stays4[x];
        }
      }
      // top-k: a token's place in the row's order
      const uint32_t of_few = r.few ? 0u : border.k.count - (uint32_t)block_add(rank);  // (tokens before the list, for those of its border)
      uint64_t Z = r.few ? 0 : border.k.mass;
#pragma unroll
      for (int x = 0; x < kMost; x++) {
        const bool in_k = r.few ? i0 + x < r.k : bin[x] == border.k.bin && of_few + i0 + x < r.k;
        if (in_k) of_k += e[x];
        above += e[x];
      }
      if (r.by_p) Z += block_add(of_k);
      const double P = r.p * (double)Z;
      uint64_t run = border.before + block_before(above);
      bool keep[kMost];
      uint32_t kept = 0;
#pragma unroll
      for (int x = 0; x < kMost; x++) {
        const uint32_t i = i0 + x;
        keep[x] = keys[x] != 0;
        if (r.by_k && (r.few || bin[x] == border.k.bin)) keep[x] &= of_few + i < r.k;
        if (r.by_p) keep[x] &= (bin[x] <= border.high && (double)run < P) || (i == 0 && border.first);
        run += e[x];
        kept += keep[x];
        if (keep[x] && stays[x])
          atomicAdd((unsigned long long *)mass + ~(uint32_t)s_list[i] / kChunk, (unsigned long long)e[x]);
      }
      kept = (uint32_t)block_add(kept);  // they are the list's first
      if (kept) {
        key = (uint32_t)(s_list[kept - 1] >> 32);
        last = ~(uint32_t)s_list[kept - 1];
      }
    } else {
      auto each = [&](auto &&f) {
        for (uint32_t i = threadIdx.x; i < a.V; i += kThreads) {
          const float l = fmaxf(row[i], -INFINITY);
          if (l != -INFINITY) f(key_of(l), i);
        }
      };
      auto sum = [&](auto &&what) {
        uint64_t s = 0;
        each([&](uint32_t k, uint32_t place) { s += what(k, place); });
        return block_add(s);
      };
      const uint64_t tokens = sum([](uint32_t, uint32_t) { return 1ull; });
      uint64_t keep = 0xFFFFFFFFull;  // of the tokens equal to `key`
      uint64_t Z = 0;
      if (r.by_k && r.k < tokens) {
        Digits d;
        d.find(each, [](uint32_t, uint32_t) { return 1ull; }, [&](uint64_t s) { return s >= r.k; });
        key = d.key;
        keep = r.k - d.before;
        if (r.by_p) Z = sum([&](uint32_t k, uint32_t) { return k > key ? r.mass(of_key(k)) : 0ull; }) + keep * r.mass(of_key(key));
      } else if (r.by_p) {
        Z = sum([&](uint32_t k, uint32_t) { return r.mass(of_key(k)); });
      }
      if (r.by_p) {
        const double P = r.p * (double)Z;
        Digits d;
        d.find(each, [&](uint32_t k, uint32_t) { return r.mass(of_key(k)); }, [&](uint64_t s) { return s > 0 && (double)s >= P; });
        // of equal tokens the i-th is left if the sum before it, before + i one, is below P
        const uint64_t one = d.here / max(d.ties, 1u);
        uint64_t some = d.ties;
        if (one) {
          const double rest = (P - (double)d.before) / (double)one;
          some = rest > 0.0 ? (uint64_t)fmin(ceil(rest), (double)d.ties) : 0;
        }
        some = max(some, (uint64_t)1);
        if (d.key > key || (d.key == key && some < keep)) {
          key = d.key;
          keep = some;
        }
      }
      if (key) {
        Digits d;  // the keep-th place of those equal to key
        d.find([&](auto &&f) { each([&](uint32_t k, uint32_t place) { if (k == key) f(~place, place); }); },
               [](uint32_t, uint32_t) { return 1ull; }, [&](uint64_t s) { return s >= keep; });
        last = ~d.key;
      }
      for (uint32_t c = threadIdx.x; c < a.chunks; c += kThreads) __hip_atomic_store(mass + c, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      wait_mem();
      __syncthreads();
      each([&](uint32_t k, uint32_t place) {
        if (k > key || (k == key && place <= last)) {
          const uint64_t e = r.left(of_key(k));
          if (e) atomicAdd((unsigned long long *)mass + place / kChunk, (unsigned long long)e);
        }
      });
    }
    wait_mem();  // (the sums of chunks are atomics, read as such: no cache has to be written back)
    __syncthreads();
  }
  // the chunk in which the running sum passes u
  __shared__ uint32_t s_chunk;
  __shared__ uint64_t s_rest, s_total;
  if (threadIdx.x < 64) {
    auto of_chunk = [&](uint32_t c) { return c < a.chunks ? __hip_atomic_load(mass + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0; };
    uint64_t total = 0;
    for (uint32_t c = threadIdx.x; c < a.chunks; c += 64) total += of_chunk(c);
    total = wave_add(total);
    const double u = fmin(fmax((double)a.u[t], 0.0), 1.0);
    const uint64_t target = min((uint64_t)(u * (double)total), total - 1);
    uint64_t base = 0;
    for (uint32_t c0 = 0; c0 < a.chunks; c0 += 64) {
      const uint64_t v = of_chunk(c0 + threadIdx.x);
      const uint64_t run = wave_run(v);
      const uint64_t before = base + run - v;
      if (before <= target && target < before + v) {
        s_chunk = c0 + threadIdx.x;
        s_rest = target - before;
        s_total = total;
      }
      base += lane_of(run, 63);
    }
  }
  __syncthreads();
  const uint64_t total = s_total;
  // and the token in it, a thread 4 neighbours
  const uint32_t i0 = place_of(s_chunk);
  const uint64_t rest = s_rest;
  const float4 v = load_chunk(a, row, s_chunk);
  float l[4];
  logits_of(v, l);
  uint64_t e[4];
  r.left(l, e);
#pragma unroll
  for (int x = 0; x < 4; x++) {
    const uint32_t k = key_of(l[x]);
    if (k < key || (k == key && i0 + x > last)) e[x] = 0;
  }
  const uint64_t sum = (e[0] + e[1]) + (e[2] + e[3]);
  uint64_t before = block_before(sum);
  if (before <= rest && rest < before + sum) {
    uint32_t x = 0;
    while (x < 3 && rest >= before + e[x]) before += e[x++];
    a.tokens[t] = (int32_t)(i0 + x);
    if (a.logprob) {
      const double z = l[x] == r.m ? 0.0 : ((double)l[x] - (double)r.m) * r.scale * (0.6931471805599453 / 32);
      a.logprob[t] = (float)(z - log(ldexp((double)total, -r.shift)));
    }
  }
}

size_t work_layout(Work &w, char *p, size_t T, size_t chunks, size_t groups) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char *q = p + off;
    off += (bytes + 255) / 256 * 256;
    return q;
  };
  w.row = (RowState *)take(T * sizeof(RowState));
  w.mass = (uint64_t *)take(T * chunks * 8);
  w.largest = (uint2 *)take(T * groups * 8);
  w.peak = (float *)take(T * chunks * (kChunk / kPiece) * 4);
  w.bin_mass = (uint64_t *)take(T * kBins * 8);
  w.bin_count = (uint32_t *)take(T * kBins * 4);
  w.list = (uint2 *)take(T * kList * 8);
  return off;
}

}  // namespace

static uint32_t sample_chunks(size_t V) { return (uint32_t)((V + kChunk - 1) / kChunk); }
static uint32_t sample_groups(uint32_t chunks) { return (chunks + kMaxSpan - 1) / kMaxSpan; }

size_t sample_workspace(size_t T, size_t V) {
  Work w;
  return work_layout(w, nullptr, T, sample_chunks(V), sample_groups(sample_chunks(V)));
}

hipError_t launch_sample(const SampleArgs &s, hipStream_t st) {
  if (!s.T || s.T > sample_rows(s.V) || !s.V || s.V > 1u << 28 || s.ld < s.V) return hipErrorInvalidValue;
  Args a{};
  a.rule = s.rule;
  a.logits = s.logits;
  a.ld = s.ld;
  a.u = s.u;
  a.V = s.V;
  a.chunks = sample_chunks(s.V);
  a.groups = sample_groups(a.chunks);
  // (All launches of 257 rows of 201088 with a top-k of 50: 128 us if their logits are counted and read again for the border's tokens,
  // 75 by pieces; with one of 390, 136 and 106; 8 rows 28 and 25. A single row takes 28 and 30.)
  a.peaks = s.rule.top_k && a.chunks * (kChunk / kPiece) <= kPieces && (size_t)s.T * a.chunks >= 768;
  a.shift = sample_shift(s.V);
  a.tokens = s.tokens;
  a.logprob = s.logprob;
  work_layout(a.w, (char *)s.work, s.T, a.chunks, a.groups);
  // Workgroups add their bins to the row's once, which costs as much as some chunks: 3 a CU, and up to 6 while a workgroup keeps
  // 8 chunks (256 rows of 201088 mixed: 3 a CU 59 and 32 us, 6 a CU 50 and 20; 254 rows of 32003: 13 and 12, or 20 and 15).
  const size_t all = (size_t)s.T * a.chunks;
  a.span = (int)std::max((all + 1535) / 1536, std::min<size_t>((all + 767) / 768, 8));
  const dim3 grid((a.chunks + a.span - 1) / a.span, s.T);
  hipError_t e = launch_own(k_sample_max, dim3(a.groups, s.T), kThreads, 0, st, a);
  if (e == hipSuccess) e = launch_own(k_sample_mass, grid, kThreads, 0, st, a);
  if (e == hipSuccess && (s.rule.top_k || s.rule.top_p)) e = launch_own(k_sample_border, grid, kThreads, 0, st, a);
  if (e == hipSuccess) e = launch_own(k_sample_draw, dim3(s.T), kThreads, 0, st, a);
  return e;
}

}  // namespace moe
