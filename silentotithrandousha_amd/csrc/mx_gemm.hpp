// Product of rows with a resident MXFP4 matrix on v_mfma_scale_f32_16x16x128_f8f6f4: D[r][t] = sum W[r][k] x[t][k],
// A = the weights as stored (tile16, layout.hpp), B = the rows as MxRows (serve.hpp): MXFP4 and MXFP8 rows as they are, bf16
// and f32 rows as 4 and 6 E2M3 terms whose sum they are. A decoded to bf16 would cost more issue slots than the products save, and
// three bf16 planes of f32 rows three products at a quarter of the rate.
//
// A workgroup of WM x WN wavefronts computes MT x NT16 tiles of 16 x 16. A package is one term of a step of 128 values: the
// rows' chunks, and with the first term the weights' chunks and both sides' scale words. Packages arrive by LDS-DMA, DEPTH
// ahead, in rings of slots; every wavefront issues the same number of loads a package, so that one counted wait and one
// barrier hand a package over. A wavefront holds the weights of its tiles in registers over the terms of a step.
#pragma once
#include "serve.hpp"
#include "stream.hpp"

namespace moe {

// FMT: the rows' format (4 E2M1, 6 E2M3, 8 E4M3).
template <int FMT, int TERMS, int MT_, int NT_, int WM_, int WN_, int DEPTH_>
struct MxShape {
  static constexpr int kFmt = FMT, kTerms = TERMS, MT = MT_, NT = NT_, WM = WM_, WN = WN_, kDepth = DEPTH_;
  static constexpr int kWaves = WM * WN, TM = MT / WM, TN = NT / WN;
  static constexpr int kChunk = FMT == 4 ? 1024 : FMT == 6 ? 1536 : 2048;
  // 1 KB pieces of a package, and those a wavefront loads (the last ones again where they do not divide)
  static constexpr int kPiecesA = MT, kPiecesB = (NT * kChunk + 1023) / 1024, kPiecesSA = (MT + 3) / 4, kPiecesSB = (NT + 3) / 4;
  static constexpr int per(int n) { return (n + kWaves - 1) / kWaves; }
  static constexpr int kLoadA = per(kPiecesA), kLoadB = per(kPiecesB), kLoadS = per(kPiecesSA + kPiecesSB);
  static constexpr int loads(int term) { return kLoadB + (term == 0 ? kLoadA + kLoadS : 0); }
  // rings: packages i .. i + DEPTH are in LDS at once; a step's weights leave it for registers with its first package
  static constexpr int kSlotsB = kDepth + 1, kSlotsA = (kDepth + TERMS) / TERMS;
  static constexpr int kBytesA = kPiecesA * 1024, kBytesB = kPiecesB * 1024, kBytesS = (kPiecesSA + kPiecesSB) * 1024;
  static constexpr int kOffB = kSlotsA * kBytesA, kOffS = kOffB + kSlotsB * kBytesB, kLds = kOffS + kSlotsA * kBytesS;
  // loads of packages after the one needed that may be outstanding when package (., term) is awaited
  static constexpr int behind(int term) {
    int n = 0;
    for (int j = 1; j < kDepth; j++) n += loads((term + j) % TERMS);
    return n;
  }
  static constexpr int most() {
    int n = 0;
    for (int t = 0; t < TERMS; t++) n = behind(t) > n ? behind(t) : n;
    return n;
  }
  static_assert(kLds <= 160 * 1024 && most() <= 63 && MT % WM == 0 && NT % WN == 0, "rings");
};

template <class S>
__global__ __launch_bounds__(64 * S::kWaves) void k_mx_gemm(MxGemmArgs a) {
  extern __shared__ __align__(1024) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::WN, wn = wave % S::WN;
  const uint32_t nm = (a.d.tiles + S::MT - 1) / S::MT, nn = (a.r.tiles + S::NT - 1) / S::NT;
  const uint32_t split = blockIdx.x / (nm * nn), tile = blockIdx.x % (nm * nn);
  const uint32_t m0 = tile % nm * S::MT, n0 = tile / nm * S::NT;
  const uint32_t nb = a.d.nb, ns = a.d.ns, nq = a.d.nq;
  const uint32_t s_first = split * a.steps, s_last = min(s_first + a.steps, ns);
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

  // package (s, term) into slots sa, sb; steps past the last one load the last again
  auto issue = [&](uint32_t s, int term, uint32_t sa, uint32_t sb) {
    s = min(s, s_last - 1);
    if (term == 0) {
      const uint32_t in_tile = min((uint32_t)lane * 16, 256 * nb - 16 - s * 1024);  // (a last step may be short)
#pragma unroll
      for (int i = 0; i < S::kLoadA; i++)
        str_dma16(off_a[i] + in_tile, wa + (size_t)s * 1024, lds0 + sa * S::kBytesA + min(i * S::kWaves + wave, S::kPiecesA - 1) * 1024);
#pragma unroll
      for (int i = 0; i < S::kLoadS; i++) {
        const int p = min(i * S::kWaves + wave, S::kPiecesSA + S::kPiecesSB - 1);
        str_dma16(off_s[i], (p < S::kPiecesSA ? wsc : xsc) + (size_t)(s / 4) * 256, lds0 + S::kOffS + sa * S::kBytesS + p * 1024);
      }
    }
#pragma unroll
    for (int i = 0; i < S::kLoadB; i++)
      str_dma16(off_b[i], xb + ((size_t)s * S::kTerms + term) * S::kChunk,
                lds0 + S::kOffB + sb * S::kBytesB + min(i * S::kWaves + wave, S::kPiecesB - 1) * 1024);
  };

  f32x4 acc[S::TM][S::TN];
#pragma unroll
  for (int i = 0; i < S::TM; i++)
#pragma unroll
    for (int j = 0; j < S::TN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
  for (int d = 0; d < S::kDepth; d++) issue(s_first + d / S::kTerms, d % S::kTerms, d / S::kTerms % S::kSlotsA, d % S::kSlotsB);

  uint32_t slot_a = 0, slot_b = 0;  // of the package at hand
  uint32_t next_a = S::kDepth / S::kTerms % S::kSlotsA;  // of the step that the next first term belongs to
  if (S::kDepth % S::kTerms) next_a = (next_a + 1) % S::kSlotsA;
  for (uint32_t s = s_first; s < s_last; s++) {
    i32x8 A[S::TM];
    uint32_t sa[S::TM], sb[S::TN];
    str_static_for<0, S::kTerms>([&](auto term_) {
      constexpr int term = decltype(term_)::value;
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __builtin_amdgcn_s_waitcnt(vm_lgkm_wait(S::behind(term)));
      __builtin_amdgcn_s_barrier();
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      {  // DEPTH ahead, into the slots of the package before this one
        constexpr int ahead = (term + S::kDepth) % S::kTerms;
        issue(s + (term + S::kDepth) / S::kTerms, ahead, next_a, slot_b == 0 ? S::kSlotsB - 1 : slot_b - 1);
        if (ahead == 0) next_a = next_a + 1 == S::kSlotsA ? 0 : next_a + 1;
      }
      if constexpr (term == 0) {
        const uint8_t *pa = lds + slot_a * S::kBytesA, *ps = lds + S::kOffS + slot_a * S::kBytesS;
        const int sh = 8 * (s & 3);
#pragma unroll
        for (int i = 0; i < S::TM; i++) {
          const uint4 v = *(const uint4 *)(pa + (wm * S::TM + i) * 1024 + lane * 16);
          A[i] = i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
          sa[i] = *(const uint32_t *)(ps + (wm * S::TM + i) * 256 + lane * 4) >> sh;
        }
#pragma unroll
        for (int j = 0; j < S::TN; j++) sb[j] = *(const uint32_t *)(ps + S::kPiecesSA * 1024 + (wn * S::TN + j) * 256 + lane * 4) >> sh & 255;
        slot_a = slot_a + 1 == S::kSlotsA ? 0 : slot_a + 1;
      } else {  // 2^-5 a term (a NaN's 255 is the first one's alone: the codes are 0)
#pragma unroll
        for (int j = 0; j < S::TN; j++) sb[j] = (uint32_t)max((int)sb[j] - 5, 1);
      }
      const uint8_t *pb = lds + S::kOffB + slot_b * S::kBytesB;
#pragma unroll
      for (int j = 0; j < S::TN; j++) {
        const uint8_t *p = pb + (wn * S::TN + j) * S::kChunk + lane * 16;
        const uint4 v = *(const uint4 *)p;
        i32x8 B{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
        if constexpr (S::kFmt == 6) {
          const uint2 u = *(const uint2 *)(p - lane * 8 + 1024);
          B[4] = (int)u.x, B[5] = (int)u.y;
        } else if constexpr (S::kFmt == 8) {
          const uint4 u = *(const uint4 *)(p + 1024);
          B[4] = (int)u.x, B[5] = (int)u.y, B[6] = (int)u.z, B[7] = (int)u.w;
        }
        constexpr int kB = S::kFmt == 4 ? 4 : S::kFmt == 6 ? 2 : 0;
#pragma unroll
        for (int i = 0; i < S::TM; i++)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A[i], B, acc[i][j], 4, kB, 0, (int)sa[i], 0, (int)sb[j]);
      }
      slot_b = slot_b + 1 == S::kSlotsB ? 0 : slot_b + 1;
    });
  }
  __builtin_amdgcn_s_waitcnt(vm_wait(0));  // (no load may land once the workgroup's LDS is another's)

  // lane l: token 16 j + l % 16, rows 16 i + 4 (l / 16) ..
  const uint32_t R = a.d.rows;
#pragma unroll
  for (int i = 0; i < S::TM; i++) {
    const uint32_t mt = m0 + wm * S::TM + i, row = mt * 16 + (lane >> 4) * 4;
    if (mt >= a.d.tiles) continue;
    f32x4 b = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (a.bias && a.splits == 1) b = *(const f32x4 *)(a.bias + row);
#pragma unroll
    for (int j = 0; j < S::TN; j++) {
      const uint32_t t = (n0 + wn * S::TN + j) * 16 + (lane & 15);
      if (t >= a.r.tokens) continue;
      const f32x4 v = acc[i][j] + b;
      if (a.splits > 1) {
        *(f32x4 *)((float *)a.out + ((size_t)split * a.r.tokens + t) * R + row) = v;
      } else if (a.bf16) {
        uint16_t q[4];
#pragma unroll
        for (int x = 0; x < 4; x++) q[x] = __builtin_bit_cast(uint16_t, (__bf16)v[x]);
        *(uint2 *)((uint16_t *)a.out + (size_t)t * R + row) = __builtin_bit_cast(uint2, q);
      } else {
        *(f32x4 *)((float *)a.out + (size_t)t * R + row) = v;
      }
    }
  }
}

template <class S>
hipError_t launch_mx_shape(const MxGemmArgs &a, hipStream_t s) {
  static DynLdsOnce once;
  hipError_t e = ensure_dyn_lds(once, (const void *)k_mx_gemm<S>, S::kLds);
  if (e != hipSuccess) return e;
  const size_t nm = (a.d.tiles + S::MT - 1) / S::MT, nn = (a.r.tiles + S::NT - 1) / S::NT;
  if (nm * nn * a.splits > (size_t)1 << 22) return hipErrorInvalidValue;  // (a launch has less than 2^32 threads)
  return launch_own(k_mx_gemm<S>, dim3((unsigned)(nm * nn * a.splits)), dim3(64 * S::kWaves), S::kLds, s, a);
}

}  // namespace moe
