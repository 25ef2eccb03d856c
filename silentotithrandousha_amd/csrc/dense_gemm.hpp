// bf16 matrix product of the dense operators on v_mfma_f32_16x16x32_bf16, f32 accumulation:
// D[m][n] = sum A[m][k] B[n][k], each operand K-contiguous or transposed in memory, with the
// operators' epilogues applied to the accumulators.
//
// A workgroup of WM x WN wavefronts computes a BM x BN tile in K-steps of 64 values, two halves of 32.
// Both operands of a step arrive by LDS-DMA in one of NS LDS slots (2 for the large tiles, more for the
// small ones, which wait for memory). Fragments are read one half ahead of the MFMAs, the first half of
// the next step included: the step's one barrier stands between its halves, where this step's reads are
// done (its slot takes the step NS ahead) and the next step's loads have landed.
// f32 rows are three bf16 planes: a step then holds a tile of A and PL = 3 tiles of B, and A's fragments meet
// each of them, the lowest plane first. As three passes over K, each loading A again, the 64 x 64 tile's wave
// read 4 fragments for 4 MFMAs instead of 8 for 12 (loss of 333 rows over 50257 x 2048: 242 -> 200 us).
// A K-contiguous operand lies in LDS as rows of 128 bytes (a line each, so that no line is asked for
// twice) whose 16-byte chunks are permuted by the row (chunk ^ row % 8), so that 8 lanes reading one chunk
// of 8 rows touch different banks. A transposed one lies as its 64 rows of k, and the fragments are read
// by the transposing LDS load, whose 16 lanes take 4 rows x 32 bytes: the 32-byte pieces are permuted by
// the row.
//
// Large products are bound by the MFMAs' power and the LDS reads beside them: the logits of 4096 bf16 rows
// (201088 x 2880) take 3.41 to 3.57 ms, 1.33 to 1.39 PFLOP/s, where the card's largest library product reached
// 1.46; of 333 f32 rows (50257 x 2048, three planes) 200 to 230 us, 0.89 to 1.03 PFLOP/s. Those of few rows by
// the weights: one f32 row, 1.16 GB in 184 us, 6.3 TB/s. In between by the tiles that 256 CUs do not share evenly.
#pragma once
#include "dense_index.hpp"
#include "dense_plan.hpp"
#include "stream.hpp"

namespace moe {

__device__ __forceinline__ uint16_t dense_bf16(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);  // round to nearest even
}

// v as `planes` bf16 values that sum to it; a non-finite v in the first alone.
__device__ __forceinline__ void dense_split(float v, uint16_t (&p)[kPlanes]) {
  p[0] = dense_bf16(v);
  const float h = bf16_to_f32(p[0]);
  const float r = isfinite(h) ? v - h : 0.0f;
  p[1] = dense_bf16(r);
  p[2] = dense_bf16(r - bf16_to_f32(p[1]));
}

// exp(t) as 2^(t log2 e), the product in two parts so that a large |t| costs no bits. The second part is far
// below 1 wherever the result is neither 0 nor infinite; past that it is bounded, as 2^a alone is the result there
// (above 2.36e38 the first part overflows and the second is infinite, for an infinite t it is NaN).
__device__ __forceinline__ float dense_exp(float t) {
  const float a = t * 1.4426950408889634f;
  const float b = fminf(fmaxf(fmaf(t, 1.4426950408889634f, -a) + t * 1.925963e-8f, -1.0f), 1.0f);
  return __builtin_amdgcn_exp2f(a) * fmaf(b, 0.6931471805599453f, 1.0f);
}

// The same within 2^-24 (1 + |t|), for sums whose terms of large |t| vanish and for results that bf16 rounds.
__device__ __forceinline__ float dense_exp_near(float t) { return __builtin_amdgcn_exp2f(t * 1.4426950408889634f); }

// The gated activation of one pair: G = min(g, limit), U = clamp(u, +-limit), s = sigmoid(1.702 G);
// h = (U + 1) G s. A NaN stays one.
struct DenseGate {
  float G, U, s;
  template <bool NEAR>
  __device__ __forceinline__ void set(float g, float u, float limit) {
    G = g > limit ? limit : g;
    U = rclamp(u, -limit, limit);
    const float t = -1.702f * G;
    s = __builtin_amdgcn_rcpf(1.0f + (NEAR ? dense_exp_near(t) : dense_exp(t)));
  }
  __device__ __forceinline__ float h() const { return (U + 1.0f) * (G * s); }
  // d loss / d(g, u) from dh = d loss / d h: nothing passes a clamp
  __device__ __forceinline__ float dg(float dh, float g, float limit) const {
    return g > limit ? 0.0f : dh * (U + 1.0f) * (s + 1.702f * ((G * s) * (1.0f - s)));  // (G s is 0 where G (1 - s) overflows, 1 - s where 1.702 G s does)
  }
  __device__ __forceinline__ float du(float dh, float u, float limit) const { return fabsf(u) > limit ? 0.0f : dh * (G * s); }
};

// One operand's tile (dense_index.hpp) as a wavefront loads and reads it.
template <int R, int W, bool TR>
struct DenseTile : DenseIndex<R, W, TR> {
  using At = DenseIndex<R, W, TR>;
  uint32_t off[At::kLoads];  // byte offset of this lane's 16 bytes from the tile's base

  __device__ __forceinline__ void init(int wave, int lane, int rows, uint32_t ld, int skip_every = 0) {
#pragma unroll
    for (int i = 0; i < At::kLoads; i++) off[i] = At::offset(i, wave, lane, rows, ld, skip_every);
  }
  // the wavefront's load i of the step whose first k is at `base`
  __device__ __forceinline__ void load(int i, const uint16_t *base, uint32_t lds, int wave) const {
    str_dma16(off[i], base, lds + At::dma(i, wave) * 1024);
  }
  __device__ __forceinline__ void clamp(int wave, int lane, uint32_t ld, int left) {
#pragma unroll
    for (int i = 0; i < At::kLoads; i++) off[i] -= At::behind(i, wave, lane, ld, left);
  }
  // zeroes the k values of the step past `left` (the last step of a K that is no multiple of 64)
  __device__ __forceinline__ static void zero_tail(uint8_t *lds, int left, int tid, int threads) {
    for (int c = tid; c < R * 8; c += threads)
      if (At::k_of(c) >= left) *(uint4 *)(lds + c * 16) = uint4{0u, 0u, 0u, 0u};
  }
  // MFMA operand of 16 rows from row0 (tile-relative), half h of the step at lds
  static __device__ __forceinline__ bf16x8 frag(const uint8_t *lds, int row0, int h, int lane) {
    if constexpr (!TR) {
      return *(const bf16x8 *)At::frag_at(lds, row0, h, lane, 0);
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      auto at = [&](int part) { return (__attribute__((address_space(3))) s16x4 *)At::frag_at(lds, row0, h, lane, part); };
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(0));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(1));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// v itself, but what is computed from it stays where it is: hoisted out of the main loop (from its rare
// branches) or shared by the columns of the epilogue it took registers and was spilled.
__device__ __forceinline__ int apart(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Stores 16 rows of 16-bit results of a wavefront: lane l holds the V values q[i] of row l % 16 from column
// (4 i + l / 16) V on. They pass through LDS (`stage`, the wavefront's own, dense_stage_bytes) so that
// a row leaves in 16-byte pieces side by side: stored from the accumulators' layout, in pieces of
// 8 bytes over 16 rows, the gradient of the LM head ran at 2.3 TB/s. ONCE: results that no later launch of
// the call reads go past the caches (that gradient for 16 rows of x 320 -> 260 us).
constexpr int dense_stage_bytes(int tm, int v) { return 16 * (tm * v * 8 + 16); }
template <int TM, int V, bool ONCE = false>
__device__ __forceinline__ void dense_rows(uint8_t *stage, int lane, const uint16_t (&q)[TM][V], uint16_t *out, size_t ld, int rows, int cols) {
  constexpr int kRow = TM * V * 8, kPieces = kRow / 16;  // bytes and 16-byte pieces of a row
  typedef uint16_t vec __attribute__((ext_vector_type(V)));
  lane = apart(lane);
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < TM; i++) *(vec *)(stage + (lane & 15) * (kRow + 16) + (4 * i + (lane >> 4)) * V * 2) = __builtin_bit_cast(vec, q[i]);
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int c = 0; c < 16 * kPieces; c += 64) {
    const int at = c + lane, row = at / kPieces, piece = at % kPieces;
    if (row < min(rows, 16) && piece * 8 < cols) {
      const u32x4 v = *(const u32x4 *)(stage + row * (kRow + 16) + piece * 16);
      u32x4 *o = (u32x4 *)(out + row * ld + piece * 8);
      if constexpr (ONCE)
        __builtin_nontemporal_store(v, o);
      else
        *o = v;
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// The same for the f32 results of columns j of the accumulators.
template <bool ONCE, int TM, int TN>
__device__ __forceinline__ void dense_rows_f32(uint8_t *stage, int lane, const f32x4 (&acc)[TM][TN], int j, float *out, size_t ld, int rows, int cols) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  uint16_t q[TM][8];
#pragma unroll
  for (int i = 0; i < TM; i++) {
    const u16x8 v = __builtin_bit_cast(u16x8, acc[i][j]);
#pragma unroll
    for (int r = 0; r < 8; r++) q[i][r] = v[r];
  }
  dense_rows<TM, 8, ONCE>(stage, lane, q, (uint16_t *)out, 2 * ld, rows, 2 * cols);
}

// f(slot, values) for the slots of plane p, the last of them with the values q as they are, the others with 0 for
// those that are not finite (which are in plane 0). ONE: rows of one plane, slot 0.
__device__ __forceinline__ void dense_finite(uint16_t &q) {
  if ((q & 0x7F80) == 0x7F80) q = 0;
}
template <class Q, int N>
__device__ __forceinline__ void dense_finite(Q (&q)[N]) {
#pragma unroll
  for (int i = 0; i < N; i++) dense_finite(q[i]);
}
template <bool ONE, class Q, class F>
__device__ __forceinline__ void dense_slots(uint32_t where, int p, Q &q, F &&f) {
  if constexpr (ONE) {
    f((size_t)0, q);
  } else {
    uint32_t m = (where >> 8 * p) & 255;
    const int last = dense_last_slot(where, p);
    f((size_t)last, q);
    m ^= 1u << last;
    if (!m) return;
    if (p == 0) dense_finite(q);
    for (; m; m &= m - 1) f((size_t)__builtin_ctz(m), q);
  }
}

// Takes the bf16 of each value, and leaves what it did not hold (if another is to follow).
template <bool MORE, int N>
__device__ __forceinline__ void dense_take(float (&v)[N], uint16_t (&q)[N]) {
#pragma unroll
  for (int r = 0; r < N; r++) {
    q[r] = dense_bf16(v[r]);
    if constexpr (MORE) {
      const float h = bf16_to_f32(q[r]);
      v[r] = isfinite(h) ? v[r] - h : 0.0f;
    }
  }
}

template <int BM, int BN, int WM, int WN, int NS, int PL, bool AT, bool BT, int EPI>
__device__ __forceinline__ void dense_tile_product(const DenseArgs &a, int block) {
  constexpr int W = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  using TA = DenseTile<BM, W, AT>;
  using TB = DenseTile<BN, W, BT>;
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int kSlot = TA::kBytes + PL * TB::kBytes, kLoads = TA::kLoads + PL * TB::kLoads;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int rows_b = a.N * a.stack;
  const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (rows_b + BN - 1) / BN;
  int tile_m, tile_n;
  dense_tile_of(block, tiles_m, tiles_n, tile_m, tile_n);
  const int m0 = tile_m * BM, n0 = tile_n * BN;
  const int split = blockIdx.y;
  const int k_lo = split * a.k_split, k_hi = min(a.K, k_lo + a.k_split);
  const int steps = (k_hi - k_lo + kDenseStep - 1) / kDenseStep;

  const uint32_t lds0 = str_lds(lds), lda = (uint32_t)a.lda * 2, ldb = (uint32_t)a.ldb * 2;
  TA la;
  TB lb;
  la.init(wave, lane, a.M - m0, lda);
  lb.init(wave, lane, rows_b - n0, ldb, PL == 1 && BN <= 64 && !BT && a.stack_step > 1 ? a.N : 0);
  // the step to load: its operands' addresses, k values left from there
  int left = k_hi - k_lo;
  const uint16_t *pa = a.A + (AT ? (size_t)k_lo * a.lda + m0 : (size_t)m0 * a.lda + k_lo), *pb[PL];
#pragma unroll
  for (int p = 0; p < PL; p++)
    pb[p] = a.B + ((a.pb >> 4 * p) & 15) * a.b_slot + (BT ? (size_t)k_lo * a.ldb + n0 : (size_t)n0 * a.ldb + k_lo);
  auto tail = [&]() __attribute__((always_inline)) {
    if (left > 0 && left < kDenseStep) {
      const int l = apart(lane);
      la.clamp(wave, l, lda, left);
      lb.clamp(wave, l, ldb, left);
    }
  };
  tail();
  auto loaded = [&]() __attribute__((always_inline)) {
    left -= kDenseStep;
    pa += AT ? a.lda * kDenseStep : kDenseStep;
#pragma unroll
    for (int p = 0; p < PL; p++) pb[p] += BT ? a.ldb * kDenseStep : kDenseStep;
    tail();
  };
  auto load_one = [&](int i, uint32_t slot) __attribute__((always_inline)) {
    if (i < TA::kLoads) {
      la.load(i, pa, slot, wave);
    } else {
      const int p = (i - TA::kLoads) / TB::kLoads;
      lb.load((i - TA::kLoads) % TB::kLoads, pb[p], slot + TA::kBytes + p * TB::kBytes, wave);
    }
  };
  auto load = [&](uint32_t slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) load_one(i, slot);
    loaded();
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // what the loss's epilogues need of a lane's columns: before the steps where the registers hold it (the
  // wait for it after 45 steps of a 32 x 16 tile was a sixth of the launch)
  constexpr bool kLoss = EPI == DENSE_STATS || EPI == DENSE_DLOGITS, kEarly = kLoss && TN <= 2;
  struct Column {
    int target;
    float lse, scale;
  } columns[kLoss ? TN : 1];
  auto column = [&](int j) __attribute__((always_inline)) {
    const int n = min(n0 + (wn * TN + j) * 16 + (lane & 15), a.N - 1);  // (columns past N are not stored)
    Column c{a.targets[n], 0.0f, 0.0f};
    if constexpr (EPI == DENSE_DLOGITS) {
      c.lse = a.lse[n];
      c.scale = a.dloss[n] / *a.scale;
    }
    return c;
  };
  if constexpr (kEarly) {
#pragma unroll
    for (int j = 0; j < TN; j++) columns[j] = column(j);
  }
  // two sets of A fragments where the registers hold them, else one, whose rows take the next half as soon
  // as their products are done
  constexpr bool kTwoA = 4 * (TM * TN + 2 * (TM + TN)) <= 224;
  constexpr bool kPinned = !AT || kTwoA;  // (the transposing loads' addresses take registers: 288 x 256 spilled)
  bf16x8 fa0[TM], fa1[kTwoA ? TM : 1], fb0[TN], fb1[TN];
  auto read_b = [&](const uint8_t *sl, int half, int p, int j) __attribute__((always_inline)) { return TB::frag(sl + TA::kBytes + p * TB::kBytes, (wn * TN + j) * 16, half, lane); };
  auto read_a = [&](const uint8_t *sl, int half, int i) __attribute__((always_inline)) { return TA::frag(sl, (wm * TM + i) * 16, half, lane); };
  // The products of a half with one of B's planes (fa, fb), row by row, and between the rows the reads for
  // the products after them (half `half` and plane `p` of sl, into nb and, if READ is 2, na) and the LDS-DMAs
  // of the step NS ahead (into slot `to`, if DMA): issued in one go they held the MFMAs up, as the LDS serves 8
  // wavefronts' 12 reads in 768 cycles (256 x 256: 958 against 1130 TFLOP/s). The reads come in the first three
  // quarters of the rows.
  auto multiply = [&](auto DMA, auto READ, auto &fa, const bf16x8(&fb)[TN], auto &na, bf16x8(&nb)[TN], const uint8_t *sl, int half, int p, uint32_t to) __attribute__((always_inline)) {
    constexpr int kRead = decltype(READ)::value, kReads = kTwoA && kRead == 2 ? TN + TM : TN, kOver = (3 * TM + 3) / 4, kEach = (kReads + kOver - 1) / kOver;
    constexpr int kDma = kPinned ? (kLoads + TM - 1) / TM : kLoads;
    if constexpr (kPinned) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < TM; i++) {
      if constexpr (decltype(DMA)::value && !kPinned) {
#pragma unroll
        for (int l = i * kDma; l < (i + 1) * kDma && l < kLoads; l++) load_one(l, to);
      }
      if constexpr (kRead != 0) {
#pragma unroll
        for (int r = i * kEach; r < (i + 1) * kEach && r < kReads; r++) {
          if (r < TN)
            nb[r] = read_b(sl, half, p, r);
          else
            na[r - TN] = read_a(sl, half, r - TN);
        }
      }
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
      if constexpr (!kTwoA && kRead == 2) fa[i] = read_a(sl, half, i);
      if constexpr (decltype(DMA)::value && kPinned) {
#pragma unroll
        for (int l = i * kDma; l < (i + 1) * kDma && l < kLoads; l++) load_one(l, to);
      }
      if constexpr (kPinned) __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  constexpr std::integral_constant<int, 0> none{};
  constexpr std::integral_constant<int, 1> only_b{};
  constexpr std::integral_constant<int, 2> both{};
  // this wavefront's loads have landed, up to those of the `NS - 2` steps after it if MORE are on their way,
  // and its reads are done, and every other's
  auto meet = [&](auto MORE) __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(vm_lgkm_wait(decltype(MORE)::value ? (NS - 2) * kLoads : 0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  int here = k_hi - k_lo;  // k values left from the next step to be read
  auto zero = [&](uint8_t *sl) __attribute__((always_inline)) {
    if (here < kDenseStep) {
      const int t = apart(tid);
      TA::zero_tail(sl, here, t, 64 * W);
#pragma unroll
      for (int p = 0; p < PL; p++) TB::zero_tail(sl + TA::kBytes + p * TB::kBytes, here, t, 64 * W);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    here -= kDenseStep;
  };
  auto landed = [&](auto MORE, uint8_t *sl) __attribute__((always_inline)) {
    meet(MORE);
    zero(sl);
  };
  for (int t = 0; t < NS && t < steps; t++) load(lds0 + t * kSlot);
  if (NS <= steps)  // step 0 is there
    __builtin_amdgcn_s_waitcnt(vm_wait((NS - 1) * kLoads));
  else
    __builtin_amdgcn_s_waitcnt(vm_wait(0));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  zero(lds);
#pragma unroll
  for (int j = 0; j < TN; j++) fb0[j] = read_b(lds, 0, 0, j);
#pragma unroll
  for (int i = 0; i < TM; i++) fa0[i] = read_a(lds, 0, i);
  uint32_t cur = 0;
  auto &fa_odd = [&]() -> auto & {
    if constexpr (kTwoA) return fa1; else return fa0;
  }();
  auto after = [&](uint32_t slot) __attribute__((always_inline)) {
    const uint32_t n = slot + kSlot;
    return n == NS * kSlot ? 0u : n;
  };
  // A step: the products of its two halves with each of B's planes. Its last ones run while the next step's
  // first fragments are read (if MORE) and its slot takes the step NS ahead (if DMA).
  auto step = [&](auto MORE, auto DMA) __attribute__((always_inline)) {
    const uint32_t next = after(cur);
    uint8_t *sl = lds + cur;
    if constexpr (PL == 1) {
      multiply(no, both, fa0, fb0, fa_odd, fb1, sl, 1, 0, 0);
    } else {
      multiply(no, only_b, fa0, fb0, fa_odd, fb1, sl, 0, 1, 0);
      multiply(no, only_b, fa0, fb1, fa_odd, fb0, sl, 0, 2, 0);
      multiply(no, both, fa0, fb0, fa_odd, fb1, sl, 1, 0, 0);
      multiply(no, only_b, fa_odd, fb1, fa0, fb0, sl, 1, 1, 0);
      multiply(no, only_b, fa_odd, fb0, fa0, fb1, sl, 1, 2, 0);
    }
    if constexpr (decltype(MORE)::value) {
      landed(DMA, lds + next);
      multiply(DMA, both, fa_odd, fb1, fa0, fb0, lds + next, 0, 0, lds0 + cur);
      if constexpr (decltype(DMA)::value) loaded();
    } else {
      multiply(no, none, fa_odd, fb1, fa0, fb0, sl, 0, 0, 0);
    }
    cur = next;
  };
  int s = 0;
  for (; s + NS < steps; s++) step(yes, yes);
  for (; s + 1 < steps; s++) step(yes, no);
  step(no, no);

  if constexpr (PL == 1 && BM * BN * 4 <= NS * kSlot && BN <= 64) {
    // B's planes were stacked as rows of one pass (so that A, which few rows wait for, streams once): a
    // column's result is the sum of its planes' columns, the first plane's last
    if (a.stack > 1) {
      __syncthreads();
      float *o = (float *)lds;
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int i = 0; i < TM; i++)
          *(f32x4 *)(o + ((wn * TN + j) * 16 + (lane & 15)) * BM + (wm * TM + i) * 16 + (lane >> 4) * 4) = acc[i][j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const int n = (wn * TN + j) * 16 + (lane & 15);
#pragma unroll
        for (int i = 0; i < TM; i++) {
          f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          if (n < a.N)
            for (int p = 0; p < a.stack; p++) v += *(const f32x4 *)(o + (p * a.N + n) * BM + (wm * TM + i) * 16 + (lane >> 4) * 4);
          acc[i][j] = v;
        }
      }
    }
  }

  // lane: column n = lane % 16 of each tile, rows m = lane / 16 * 4 + 0..3
  const int mw = m0 + wm * TM * 16 + (lane >> 4) * 4, nw = n0 + wn * TN * 16 + (lane & 15);
  // the wavefront's first row and column, and its part of the LDS for 16-bit results
  const int m_first = m0 + wm * TM * 16, n_first = n0 + wn * TN * 16;
  constexpr int kStage = dense_stage_bytes(TM, EPI == DENSE_GATE ? 2 : EPI == DENSE_DLOGITS ? 4 : 8);
  static_assert(W * kStage <= NS * kSlot, "the results of 16 columns fit the LDS of the steps");
  uint8_t *stage = lds + wave * kStage;
  if constexpr (EPI != DENSE_STATS && EPI != DENSE_DGATE) __syncthreads();
  // results in planes come of rows in planes, which only the small tiles take beside single ones
  auto by_planes = [&](auto &&f) __attribute__((always_inline)) {
    if constexpr (PL > 1)
      f(no);
    else if constexpr (BN > 64)
      f(yes);
    else if (a.planes == 1)
      f(yes);
    else
      f(no);
  };
  if constexpr (EPI == DENSE_STORE || EPI == DENSE_GATE) {
    const float scale = EPI == DENSE_STORE && a.scale ? *a.scale : 1.0f;
#pragma unroll
    for (int i = 0; i < TM; i++) {
      f32x4 b = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (a.bias && mw + i * 16 < a.M) b = *(const f32x4 *)(a.bias + mw + i * 16);
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] = (acc[i][j] + b) * scale;
    }
  }
  if constexpr (EPI == DENSE_STORE) {
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int n = nw + j * 16;
      if (a.out_mode == 0) {
        uint16_t q[TM][4];
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
          for (int r = 0; r < 4; r++) q[i][r] = dense_bf16(acc[i][j][r]);
        dense_rows<TM, 4, BT>(stage, lane, q, (uint16_t *)a.out + (size_t)(n_first + j * 16) * a.ldo + m_first, a.ldo, a.N - n_first - j * 16, a.M - m_first);
        continue;
      }
      if (a.out_mode == 2) {
#pragma unroll
        for (int i = 0; i < TM; i++) {
          const int m = mw + i * 16;
          if (n >= a.N || m >= a.M) continue;
          f32x4 *o = (f32x4 *)((float *)a.out + (size_t)n * a.ldo + m);
          *o = acc[i][j] + *o;
        }
        continue;
      }
      dense_rows_f32<BT>(stage, lane, acc, j, (float *)a.out + split * a.split_stride + (size_t)(n_first + j * 16) * a.ldo + m_first, a.ldo,
                     a.N - n_first - j * 16, a.M - m_first);
    }
  } else if constexpr (EPI == DENSE_GATE) {
    auto gate = [&](auto ONE) __attribute__((always_inline)) {  // ONE plane, or kPlanes
      constexpr bool one = decltype(ONE)::value;
#pragma unroll
      for (int j = 0; j < TN; j++) {
        float h[TM][2];
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
          for (int r = 0; r < 2; r++) {
            DenseGate g;
            g.set<one>(acc[i][j][2 * r], acc[i][j][2 * r + 1], a.limit);
            h[i][r] = g.h();
          }
        for (int p = 0; p < (one ? 1 : kPlanes); p++) {
          uint16_t q[TM][2];
#pragma unroll
          for (int i = 0; i < TM; i++) dense_take<!one>(h[i], q[i]);
          dense_slots<one>(a.h_where, p, q, [&](size_t at, const auto &q) {
            dense_rows<TM, 2>(stage, lane, q, a.h + at * a.h_slot + (size_t)(n_first + j * 16) * a.ldh + m_first / 2, a.ldh,
                              a.N - n_first - j * 16, (a.M - m_first) / 2);
          });
        }
      }
    };
    by_planes(gate);
  } else if constexpr (EPI == DENSE_DGATE) {
    // (stored from the accumulators' layout, 64 and 32 bytes of a row at a time: staged as the other results
    // it kept too much in registers and was no faster, 107 and 116 us of 4096 x 2880 against 108)
    auto dgate = [&](auto ONE) __attribute__((always_inline)) {
      constexpr bool one = decltype(ONE)::value;
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const int m = mw + i * 16;
        float db[8] = {};
#pragma unroll
        for (int j = 0; j < TN; j++) {
          const int n = nw + j * 16;
          if (n >= a.N || m >= a.M) continue;
          const f32x4 *row = (const f32x4 *)(a.gu + (size_t)n * a.M * 2 + 2 * m);
          const f32x4 g01 = row[0], g23 = row[1];
          float d[8], hv[4];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float gate = r < 2 ? g01[2 * r] : g23[2 * r - 4], up = r < 2 ? g01[2 * r + 1] : g23[2 * r - 3];
            DenseGate g;
            g.set<one>(gate, up, a.limit);
            const float dh = acc[i][j][r];
            hv[r] = g.h();
            d[2 * r] = g.dg(dh, gate, a.limit);
            d[2 * r + 1] = g.du(dh, up, a.limit);
          }
#pragma unroll
          for (int r = 0; r < 8; r++) db[r] += d[r];
          for (int p = 0; p < (one ? 1 : kPlanes); p++) {
            uint16_t q[8], e[4];
            dense_take<!one>(d, q);
            dense_take<!one>(hv, e);
            dense_slots<one>(a.dgu_where, p, q, [&](size_t at, const auto &q) { *(uint4 *)(a.dgu + at * a.dgu_slot + (size_t)n * a.M * 2 + 2 * m) = __builtin_bit_cast(uint4, q); });
            dense_slots<one>(a.h_where, p, e, [&](size_t at, const auto &e) { *(uint2 *)(a.h + at * a.h_slot + (size_t)n * a.ldh + m) = __builtin_bit_cast(uint2, e); });
          }
        }
        if (a.db_part) {  // over the wavefront's columns: 16 lanes, then a part per wavefront column
#pragma unroll
          for (int r = 0; r < 8; r++) {
            db[r] += __shfl_xor(db[r], 1);
            db[r] += __shfl_xor(db[r], 2);
            db[r] += __shfl_xor(db[r], 4);
            db[r] += __shfl_xor(db[r], 8);
          }
          if ((lane & 15) == 0 && m < a.M) {
            f32x4 *o = (f32x4 *)(a.db_part + (size_t)(tile_n * WN + wn) * a.M * 2 + 2 * m);
            o[0] = f32x4{db[0], db[1], db[2], db[3]};
            o[1] = f32x4{db[4], db[5], db[6], db[7]};
          }
        }
      }
    };
    by_planes(dgate);
  } else if constexpr (EPI == DENSE_STATS) {
    const bool whole = m_first + TM * 16 <= a.M;  // else the rows past the vocabulary count as minus infinity
    if (!whole) {
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (mw + i * 16 + r >= a.M) {
#pragma unroll
            for (int j = 0; j < TN; j++) acc[i][j][r] = -INFINITY;
          }
    }
#pragma unroll
    for (int j = 0; j < TN; j++) {
      if constexpr (!kEarly) columns[j] = column(j);
      const int n = nw + j * 16, t = n < a.N ? columns[j].target : -1;
      const int want = t >= a.v0 ? t - a.v0 - mw : -1;  // the target's row from the lane's first
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < TM; i++) {
#pragma unroll
        for (int r = 0; r < 4; r++) mx = fmaxf(mx, acc[i][j][r]);
        if (want >> 4 == i && (want & 15) < 4 && t - a.v0 < a.M)
          a.picked[n] = (want & 2) ? ((want & 1) ? acc[i][j][3] : acc[i][j][2]) : ((want & 1) ? acc[i][j][1] : acc[i][j][0]);
      }
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      // no value above minus infinity: every exponential is 0 against a base of 0
      float base = mx == -INFINITY ? 0.0f : mx;
      if (__any(fabsf(base) > 2e38f)) {  // its product with log2 e may overflow: the difference first
#pragma unroll
        for (int i = 0; i < TM; i++) acc[i][j] -= f32x4{base, base, base, base};
        base = 0.0f;
      }
      base *= 1.4426950408889634f;
      float sum = 0.0f;  // (a NaN among the logits makes it one)
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], 1.4426950408889634f, -base));
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lane < 16 && n < a.N) a.stats[(size_t)(tile_m * WM + wm) * a.N + n] = make_float2(mx, sum);
    }
  } else {
    auto dlogits = [&](auto ONE) __attribute__((always_inline)) {
      constexpr bool one = decltype(ONE)::value;
#pragma unroll
      for (int j = 0; j < TN; j++) {
        if constexpr (!kEarly) columns[j] = column(j);
        const int t = columns[j].target;
        const int want = t >= a.v0 ? t - a.v0 - mw : -1;
        const float lse = t >= a.vocab ? NAN : columns[j].lse, scale = columns[j].scale;
        float d[TM][4];
#pragma unroll
        for (int i = 0; i < TM; i++) {
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float x = acc[i][j][r] - lse;
            d[i][r] = scale * (one ? dense_exp_near(x) : dense_exp(x));
          }
          if (want >> 4 == i && (want & 15) < 4) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const float x = acc[i][j][r] - lse;
              if ((want & 3) == r) d[i][r] = scale * ((one ? dense_exp_near(x) : dense_exp(x)) - 1.0f);
            }
          }
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (t < 0 || mw + i * 16 + r >= a.M) d[i][r] = 0.0f;  // ignored token, padding column
        }
        for (int p = 0; p < (one ? 1 : kPlanes); p++) {
          uint16_t q[TM][4];
#pragma unroll
          for (int i = 0; i < TM; i++) dense_take<!one>(d[i], q[i]);
          dense_slots<one>(a.dl_where, p, q, [&](size_t at, const auto &q) {
            dense_rows<TM, 4>(stage, lane, q, a.dl + at * a.dl_slot + (size_t)(n_first + j * 16) * a.ld_dl + m_first, a.ld_dl,
                              a.N - n_first - j * 16, (int)a.ld_dl - m_first);
          });
        }
      }
    };
    by_planes(dlogits);
  }
}

template <int BM, int BN, int WM, int WN, int NS, int PL, bool AT, bool BT, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void k_dense(const DenseArgs a) {
  dense_tile_product<BM, BN, WM, WN, NS, PL, AT, BT, EPI>(a, blockIdx.x);
}

// Two products in one launch: the tiles of one fill the CUs that the other's last round leaves idle (the
// weight gradients of 4096 rows, 5760 and 2880 x 2880: 230 and 180 tiles for 256 CUs took 156 + 91 us, 420
// together 222; of 257 f32 rows, 1024 x 2056, 28 + 20 and 31).
struct DensePair {
  DenseArgs a[2];
  int first;  // tiles of a[0]
};
template <int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void k_dense_pair(const DensePair p) {
  const int second = (int)blockIdx.x >= p.first;
  dense_tile_product<BM, BN, WM, WN, NS, 1, true, true, DENSE_STORE>(p.a[second], blockIdx.x - (second ? p.first : 0));
}
template <int BM, int BN, int WM, int WN, int NS>
hipError_t launch_dense_pair_as(const DenseArgs &a, const DenseArgs &b, hipStream_t st) {
  static DynLdsOnce once;
  const size_t bytes = NS * (BM + BN) * 128;
  auto kernel = k_dense_pair<BM, BN, WM, WN, NS>;
  hipError_t e = ensure_dyn_lds(once, (const void *)kernel, bytes);
  if (e != hipSuccess) return e;
  auto tiles = [](const DenseArgs &a) { return (size_t)((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN); };
  if ((tiles(a) + tiles(b)) * 64 * WM * WN >> 32) return hipErrorInvalidValue;  // (a launch counts threads in 32 bits)
  return launch_own(kernel, (unsigned)(tiles(a) + tiles(b)), 64 * WM * WN, bytes, st, DensePair{{a, b}, (int)tiles(a)});
}

template <int BM, int BN, int WM, int WN, int NS, int PL, bool AT, bool BT, int EPI>
hipError_t launch_dense_as(const DenseArgs &a, hipStream_t st) {
  static DynLdsOnce once;
  const size_t bytes = NS * (BM + PL * BN) * 128;
  auto kernel = k_dense<BM, BN, WM, WN, NS, PL, AT, BT, EPI>;
  hipError_t e = ensure_dyn_lds(once, (const void *)kernel, bytes);
  if (e != hipSuccess) return e;
  const size_t tiles = (size_t)((a.M + BM - 1) / BM) * ((a.N * a.stack + BN - 1) / BN);
  if (a.b_planes != PL || (a.stack > 1 && (PL > 1 || a.N * a.stack > BN || BN > 64))) return hipErrorInvalidValue;
  if ((EPI == DENSE_GATE || EPI == DENSE_DGATE || EPI == DENSE_DLOGITS) && (PL > 1 ? a.planes == 1 : BN > 64 && a.planes > 1)) return hipErrorInvalidValue;
  if (tiles * 64 * WM * WN >> 32 || a.splits > 65535) return hipErrorInvalidValue;  // (a launch counts threads in 32 bits)
  return launch_own(kernel, dim3((unsigned)tiles, a.splits), 64 * WM * WN, bytes, st, a);
}

}  // namespace moe
