// Product of rows with a resident MXFP4 matrix: D[r][t] = sum W[r][k] x[t][k], A = the weights as stored (tile16, layout.hpp), B = the rows
// as MxRows (serve.hpp).
//
// On v_mfma_scale_f32_16x16x128_f8f6f4: MXFP4 rows as they are, MXFP8 rows as their larger and their smaller codes, f32 rows as 6
// E2M3 terms whose sum they are to 2^-29 of their block's largest (three bf16 planes would hold them whole and take twice as long).
// On v_mfma_f32_16x16x32_bf16: bf16 rows as they are, the weights decoded in registers, four conversions for 8 values that meet all of a
// wavefront's row tiles. (As 4 E2M3 terms, whose products take as long, what is below 2^-11 of a block's largest lost bits, and the terms
// cost half as many bytes again: 4096 rows over 2880 x 2880 73 us, so 64.)
//
// A workgroup of WM x WN wavefronts computes MT x NT16 tiles of 16 x 16. A package is one term of a step of 128 values: the
// rows' chunks, with the first term the weights' chunks, and with every fourth step both sides' scale words. Packages arrive by LDS-DMA in rings
// of DEPTH slots; every wavefront issues the same number of loads a package, so that one counted wait and one barrier hand a
// package over. That barrier stands in the middle of the package before it, whose operands are in registers by then: the next
// one's are read, and the loads that take its slots issued, between the MFMAs of its second half. (With the reads in front of all
// of a package's MFMAs both wavefronts of a SIMD waited for them together: 4096 bf16 rows in terms 68 us, so 66.)
// The weights' operands stay in registers over the terms of a step. What bounds the 192 x 256 tile: its MFMAs, issued at some 60 % of their
// rate (4096 x 2880 x 2880 in bf16 60 us, 1.14 PFLOP/s; MXFP4 rows over 5760 x 2880 44 us, 3.0 PFLOP/s, of which some 10 us a
// tile are its first loads and its results, which no other workgroup of the CU covers).
#pragma once
#include <algorithm>
#include <cmath>

#include "serve.hpp"
#include "stream.hpp"

namespace moe {

// a row's weights of 8 values in bf16 (E2M1 times a power of two, exactly; of 2^128 and above infinite as in f32); a scale byte of 255
// is NaN
__device__ __forceinline__ bf16x8 mx_weights8(uint32_t codes, uint32_t scale_byte) {
  return decode8(codes, __uint_as_float(scale_byte == 255 ? 0x7FC00000u : scale_byte << 23));
}
// whether one of 8 bf16 values is infinite or NaN: its exponent's carry
__device__ __forceinline__ bool mx_not_finite(const uint4 &v) {
  auto carry = [](uint32_t w) { return (w & 0x7F807F80u) + 0x00800080u; };
  return ((carry(v.x) | carry(v.y) | carry(v.z) | carry(v.w)) & 0x80008000u) != 0;
}
constexpr uint32_t kNan2 = 0x7FC07FC0u;  // two bf16

// FMT: the rows' format (4 E2M1, 6 E2M3, 8 E4M3, 16 bf16: TERMS are the four quarters of a block).
template <int FMT, int TERMS, int MT_, int NT_, int WM_, int WN_, int DEPTH_>
struct MxShape {
  static constexpr int kFmt = FMT, kTerms = TERMS, MT = MT_, NT = NT_, WM = WM_, WN = WN_, kDepth = DEPTH_;
  static constexpr int kWaves = WM * WN, TM = MT / WM, TN = NT / WN;
  static constexpr int kChunk = FMT == 4 || FMT == 16 ? 1024 : FMT == 6 ? 1536 : 2048;
  // 1 KB pieces of a package, and those a wavefront loads (the last ones again where they do not divide)
  static constexpr int kPiecesA = MT, kPiecesB = (NT * kChunk + 1023) / 1024, kPiecesSA = (MT + 3) / 4, kPiecesSB = FMT == 16 ? 0 : (NT + 3) / 4;
  static constexpr int per(int n) { return (n + kWaves - 1) / kWaves; }
  static constexpr int kLoadA = per(kPiecesA), kLoadB = per(kPiecesB), kLoadS = per(kPiecesSA + kPiecesSB);
  static constexpr int kRound = 4 * TERMS;  // packages whose scales come in one word
  static constexpr int loads(int u) { return kLoadB + (u % TERMS == 0 ? kLoadA : 0) + (u % kRound == 0 ? kLoadS : 0); }
  // rings: packages i + 1 .. i + DEPTH are in LDS while i is multiplied; a step's weights leave it with its first package
  static constexpr int kSlotsB = kDepth, kSlotsA = (kDepth + TERMS - 1) / TERMS, kSlotsS = (kDepth + kRound - 1) / kRound;
  static constexpr int kBytesA = kPiecesA * 1024, kBytesB = kPiecesB * 1024, kBytesS = (kPiecesSA + kPiecesSB) * 1024;
  static constexpr int kOffB = kSlotsA * kBytesA, kOffS = kOffB + kSlotsB * kBytesB, kRings = kOffS + kSlotsS * kBytesS;
  // loads that may be outstanding when the package after the round's u-th is awaited: those of the packages behind it
  static constexpr int behind(int u) {
    int n = 0;
    for (int j = 2; j < kDepth; j++) n += loads(u + j);
    return n;
  }
  static constexpr int most() {
    int n = 0;
    for (int u = 0; u < kRound; u++) n = behind(u) + loads(u + kDepth) > n ? behind(u) + loads(u + kDepth) : n;
    return n;
  }
  static constexpr int kStage = 16 * (TM * 64 + 16);  // bytes a wavefront's results pass through
  static constexpr int kLds = kRings > kWaves * kStage ? kRings : kWaves * kStage;
  static_assert(kLds <= 160 * 1024 && most() <= 63 && MT % WM == 0 && NT % WN == 0, "rings");
};

// A wavefront's tiles to out [tokens][rows]. Lane l of a tile holds token l % 16, rows 4 (l / 16) ..; they pass through LDS so
// that a token's rows leave in 16-byte pieces side by side (stored as they lie, in pieces of 8 bytes over 16 tokens, 4096 x
// 5760 results in bf16 took some 25 us more).
template <class S, class O>
__device__ __forceinline__ void mx_store(const MxGemmArgs &a, const f32x4 (&acc)[S::TM][S::TN], uint8_t *stage, int lane, uint32_t row0,
                                         uint32_t t0, const float *bias, O *out) {
  constexpr int kRow = S::TM * 16 * sizeof(O), kPieces = kRow / 16;
  const uint32_t R = a.d.rows;
  f32x4 b[S::TM];
#pragma unroll
  for (int i = 0; i < S::TM; i++) {
    b[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (bias && row0 + i * 16 < R) b[i] = *(const f32x4 *)(bias + row0 + i * 16 + (lane >> 4) * 4);
  }
#pragma unroll
  for (int j = 0; j < S::TN; j++) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < S::TM; i++) {
      const f32x4 v = acc[i][j] + b[i];
      uint8_t *to = stage + (lane & 15) * (kRow + 16) + (i * 16 + (lane >> 4) * 4) * sizeof(O);
      if constexpr (sizeof(O) == 2) {
        uint16_t q[4];
#pragma unroll
        for (int x = 0; x < 4; x++) q[x] = __builtin_bit_cast(uint16_t, (__bf16)v[x]);
        *(uint2 *)to = __builtin_bit_cast(uint2, q);
      } else {
        *(f32x4 *)to = v;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int c = 0; c < 16 * kPieces; c += 64) {
      const int at = c + lane, tok = at / kPieces, piece = at % kPieces;
      const uint32_t t = t0 + j * 16 + tok, row = row0 + piece * (16 / sizeof(O));
      if (tok < 16 && t < a.r.tokens && row < R)
        *(uint4 *)(out + (size_t)t * R + row) = *(const uint4 *)(stage + tok * (kRow + 16) + piece * 16);
    }
  }
}

template <class S>
__global__ __launch_bounds__(64 * S::kWaves) void k_mx_gemm(MxGemmArgs a) {
  extern __shared__ __align__(1024) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN;
  // Workgroups go to the 8 XCDs in turn, each of which takes tiles that lie together, in strips of a.strip tiles of rows: what
  // its CUs read at a time then comes through its L2 once.
  const uint32_t nm = (a.d.tiles + S::MT - 1) / S::MT, nn = (a.r.tiles + S::NT - 1) / S::NT, all = nm * nn;
  const uint32_t at = blockIdx.x % 8 * ((all + 7) / 8) + blockIdx.x / 8;
  if (blockIdx.x / 8 >= (all + 7) / 8 || at >= all) return;
  const uint32_t strip = at / (nm * a.strip) * a.strip, in = at - strip * nm, wide = min((uint32_t)a.strip, nn - strip);
  // (uniform, and said to be: the loads' bases are scalar)
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(in / wide) * S::MT, n0 = __builtin_amdgcn_readfirstlane(strip + in % wide) * S::NT;
  const uint32_t nb = a.d.nb, ns = a.d.ns, nq = a.d.nq;
  const uint32_t lds0 = str_lds(lds);

  // this lane's offsets from the workgroup's first tile (tiles past the matrix read its last one)
  const uint8_t *wa = a.w + (size_t)m0 * 256 * nb;
  const uint8_t *wsc = a.w + pack_weight_bytes(a.d) + (size_t)m0 * nq * 256;
  const size_t row_tile = (size_t)ns * S::kTerms * S::kChunk;
  const uint8_t *xb = a.codes + n0 * row_tile;
  const uint8_t *xsc = (const uint8_t *)a.scales + (size_t)n0 * nq * 256;
  const uint32_t m_last = a.d.tiles - 1 - m0, n_last = a.r.tiles - 1 - n0;
  uint32_t off_a[S::kLoadA], off_b[S::kLoadB], off_s[S::kLoadS];
#pragma unroll
  for (int i = 0; i < S::kLoadA; i++) off_a[i] = min((uint32_t)min(i * S::kWaves + wave, S::kPiecesA - 1), m_last) * 256 * nb;
#pragma unroll
  for (int i = 0; i < S::kLoadB; i++) {
    const int c = min(min(i * S::kWaves + wave, S::kPiecesB - 1) * 64 + lane, S::NT * S::kChunk / 16 - 1);
    off_b[i] = min((uint32_t)(c / (S::kChunk / 16)), n_last) * (uint32_t)row_tile + c % (S::kChunk / 16) * 16;
  }
#pragma unroll
  for (int i = 0; i < S::kLoadS; i++) {
    const int p = min(i * S::kWaves + wave, S::kPiecesSA + S::kPiecesSB - 1);
    const bool of_a = p < S::kPiecesSA;
    const uint32_t t = (of_a ? p : p - S::kPiecesSA) * 4 + (lane >> 4);
    off_s[i] = min(t, of_a ? m_last : n_last) * nq * 256 + (lane & 15) * 16;
  }

  // load `piece` of the package of step s and term u % TERMS into slots; steps past the last one load the last again
  auto issue = [&](int piece, uint32_t s, int u, uint32_t slot_a, uint32_t slot_b, uint32_t slot_s) {
    s = min(s, ns - 1);
    if (piece < S::kLoadB) {
      str_dma16(off_b[piece], xb + ((size_t)s * S::kTerms + u % S::kTerms) * S::kChunk,
                lds0 + S::kOffB + slot_b * S::kBytesB + min(piece * S::kWaves + wave, S::kPiecesB - 1) * 1024);
    } else if (piece < S::kLoadB + S::kLoadA) {
      const int i = piece - S::kLoadB;
      const uint32_t in_tile = min((uint32_t)lane * 16, 256 * nb - 16 - s * 1024);  // (a last step may be short)
      str_dma16(off_a[i] + in_tile, wa + (size_t)s * 1024, lds0 + slot_a * S::kBytesA + min(i * S::kWaves + wave, S::kPiecesA - 1) * 1024);
    } else {
      const int i = piece - S::kLoadB - S::kLoadA, p = min(i * S::kWaves + wave, S::kPiecesSA + S::kPiecesSB - 1);
      str_dma16(off_s[i], (p < S::kPiecesSA ? wsc : xsc) + (size_t)(s / 4) * 256, lds0 + S::kOffS + slot_s * S::kBytesS + p * 1024);
    }
  };
  auto wait = [&](auto outstanding) {  // for the loads before the last `outstanding` ones, of every wavefront
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(vm_lgkm_wait(decltype(outstanding)::value));
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };
  // the operands of a package, of a step, and the scale words of a round
  auto read_b = [&](uint32_t slot, i32x8 (&B)[S::TN]) {
    const uint8_t *pb = lds + S::kOffB + slot * S::kBytesB + wn * S::TN * S::kChunk + lane * 16;
#pragma unroll
    for (int j = 0; j < S::TN; j++) {
      const uint8_t *p = pb + j * S::kChunk;
      const uint4 v = *(const uint4 *)p;
      B[j] = i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
      if constexpr (S::kFmt == 6) {
        const uint2 u = *(const uint2 *)(p - lane * 8 + 1024);
        B[j][4] = (int)u.x, B[j][5] = (int)u.y;
      } else if constexpr (S::kFmt == 8) {
        const uint4 u = *(const uint4 *)(p + 1024);
        B[j][4] = (int)u.x, B[j][5] = (int)u.y, B[j][6] = (int)u.z, B[j][7] = (int)u.w;
      }
    }
  };
  auto read_a = [&](uint32_t slot, i32x8 (&A)[S::TM]) {
    const uint8_t *pa = lds + slot * S::kBytesA + wm * S::TM * 1024 + lane * 16;
#pragma unroll
    for (int i = 0; i < S::TM; i++) {
      const uint4 v = *(const uint4 *)(pa + i * 1024);
      A[i] = i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
    }
  };
  auto read_s = [&](uint32_t slot, uint32_t (&sa)[S::TM], uint32_t (&sb)[S::TN]) {
    const uint8_t *ps = lds + S::kOffS + slot * S::kBytesS + lane * 4;
#pragma unroll
    for (int i = 0; i < S::TM; i++) sa[i] = *(const uint32_t *)(ps + (wm * S::TM + i) * 256);
#pragma unroll
    for (int j = 0; j < S::TN; j++) sb[j] = S::kPiecesSB ? *(const uint32_t *)(ps + S::kPiecesSA * 1024 + (wn * S::TN + j) * 256) : 0;
  };

  f32x4 acc[S::TM][S::TN];
#pragma unroll
  for (int i = 0; i < S::TM; i++)
#pragma unroll
    for (int j = 0; j < S::TN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
  for (int d = 0; d < S::kDepth; d++)
#pragma unroll
    for (int i = 0; i < S::loads(d); i++) issue(i, d / S::kTerms, d, d / S::kTerms, d, d / S::kRound);
  // (package 0: those of the packages 1 .. DEPTH - 1 may be outstanding)
  wait(std::integral_constant<int, S::behind(S::kRound - 1) + S::loads(S::kDepth - 1)>{});
  i32x8 A[2][S::TM], B[2][S::TN];  // of the step and package at hand, and of the next
  uint32_t sa[S::TM], sb[S::TN], sw[S::TN];
  read_s(0, sa, sb);
  read_a(0, A[0]);
  read_b(0, B[0]);
  // slots of the next package, step and round; and of the step and round to be loaded next
  uint32_t slot_b = 1 % S::kSlotsB, slot_a = 1 % S::kSlotsA, slot_s = 1 % S::kSlotsS, next_a = 0, next_s = 0;
  for (uint32_t s0 = 0; s0 < ns; s0 += 4) {
    str_static_for<0, S::kRound>([&](auto u_) {
      constexpr int u = decltype(u_)::value, step = u / S::kTerms, term = u % S::kTerms;
      const uint32_t s = s0 + step;
      if (step && s >= ns) return;  // (steps are no multiple of 4)
      // the rows' scales: of E2M3 terms 2^-5 each (a NaN's 255 is the first one's alone: the codes are 0)
      if constexpr (S::kFmt == 6) {
#pragma unroll
        for (int j = 0; j < S::TN; j++) sw[j] = term == 0 ? sb[j] >> 8 * step & 255 : (uint32_t)max((int)sw[j] - 5, 1);
      }
      constexpr int kB = S::kFmt == 4 ? 4 : S::kFmt == 6 ? 2 : 0, kAll = S::TM * S::TN, kHalf = kAll / 2;
      bf16x8 w[S::kFmt == 16 ? S::TM : 1];
      auto mfma = [&](int p) {
        const int i = p % S::TM, j = p / S::TM;
        if constexpr (S::kFmt == 16) {
          if (j == 0) w[i] = mx_weights8((uint32_t)A[step & 1][i][term], sa[i] >> 8 * step & 255);
          const i32x8 &b = B[u & 1][j];
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i], as_bf16x8(make_uint4(b[0], b[1], b[2], b[3])), acc[i][j], 0, 0, 0);
        } else if constexpr (S::kFmt == 6)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A[step & 1][i], B[u & 1][j], acc[i][j], 4, kB, step, (int)sa[i], 0, (int)sw[j]);
        else
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A[step & 1][i], B[u & 1][j], acc[i][j], 4, kB, step, (int)sa[i], step, (int)sb[j]);
      };
#pragma unroll
      for (int p = 0; p < kHalf; p++) mfma(p);
      __builtin_amdgcn_sched_barrier(0);
      wait(std::integral_constant<int, S::behind(u)>{});
      if constexpr (term == S::kTerms - 1) {
        read_a(slot_a, A[step & 1 ^ 1]);
        slot_a = slot_a + 1 == S::kSlotsA ? 0 : slot_a + 1;
      }
      read_b(slot_b, B[u & 1 ^ 1]);
      uint32_t sa2[S::TM], sb2[S::TN];
      if constexpr (u == S::kRound - 1) {
        read_s(slot_s, sa2, sb2);
        slot_s = slot_s + 1 == S::kSlotsS ? 0 : slot_s + 1;
      }
      __builtin_amdgcn_sched_barrier(0);
      constexpr int ahead = u + S::kDepth;
      const uint32_t into_b = slot_b == 0 ? S::kSlotsB - 1 : slot_b - 1;
#pragma unroll
      for (int p = kHalf; p < kAll || p - kHalf < S::loads(ahead); p++) {
        if (p < kAll) mfma(p);
        if (p - kHalf < S::loads(ahead)) {
          issue(p - kHalf, s0 + ahead / S::kTerms, ahead, next_a, into_b, next_s);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (ahead % S::kTerms == 0) next_a = next_a + 1 == S::kSlotsA ? 0 : next_a + 1;
      if (ahead % S::kRound == 0) next_s = next_s + 1 == S::kSlotsS ? 0 : next_s + 1;
      slot_b = slot_b + 1 == S::kSlotsB ? 0 : slot_b + 1;
      if constexpr (u == S::kRound - 1) {
#pragma unroll
        for (int i = 0; i < S::TM; i++) sa[i] = sa2[i];
#pragma unroll
        for (int j = 0; j < S::TN; j++) sb[j] = sb2[j];
      }
    });
  }

  // (no load may land once the workgroup's LDS holds something else, its own results or another's)
  __builtin_amdgcn_s_waitcnt(vm_wait(0));
  __syncthreads();
  uint8_t *stage = lds + wave * S::kStage;
  const uint32_t row0 = (m0 + wm * S::TM) * 16, t0 = (n0 + wn * S::TN) * 16;
  if (a.bf16)
    mx_store<S, uint16_t>(a, acc, stage, lane, row0, t0, a.bias, (uint16_t *)a.out);
  else
    mx_store<S, float>(a, acc, stage, lane, row0, t0, a.bias, (float *)a.out);
}

template <class S>
hipError_t launch_mx_shape(const MxGemmArgs &a, hipStream_t s) {
  static DynLdsOnce once;
  hipError_t e = ensure_dyn_lds(once, (const void *)k_mx_gemm<S>, S::kLds);
  if (e != hipSuccess) return e;
  const size_t nm = (a.d.tiles + S::MT - 1) / S::MT, nn = (a.r.tiles + S::NT - 1) / S::NT, all = nm * nn;
  if (all > (size_t)1 << 22) return hipErrorInvalidValue;  // (a launch has less than 2^32 threads)
  MxGemmArgs b = a;
  // an XCD's 32 CUs on about as many rows as tokens
  b.strip = std::max(1, (int)std::lround(std::sqrt(32.0 * S::MT / S::NT)));
  return launch_own(k_mx_gemm<S>, dim3((unsigned)((all + 7) / 8 * 8)), dim3(64 * S::kWaves), S::kLds, s, b);
}

}  // namespace moe
