// bf16 matrix product of the dense operators on v_mfma_f32_16x16x32_bf16, f32 accumulation:
// D[m][n] = sum A[m][k] B[n][k], each operand K-contiguous or transposed in memory, with the
// operators' epilogues applied to the accumulators.
//
// A workgroup of WM x WN wavefronts computes a BM x BN tile in K-steps of 64 values. Both operands of
// a step arrive by LDS-DMA in one of two LDS slots while the other is computed on; one barrier a step.
// A K-contiguous operand lies in LDS as rows of 128 bytes whose 16-byte chunks are permuted by the
// row (chunk ^ row % 8), so that 8 lanes reading one chunk of 8 rows touch different banks. A
// transposed operand lies as its 64 rows of k, and the fragments are read by the transposing LDS
// load, whose 16 lanes take 4 rows x 32 bytes: the 32-byte pieces are permuted by the row.
#pragma once
#include "dense.hpp"
#include "stream.hpp"

namespace moe {

constexpr int kDenseStep = 64;  // k values per step

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

// exp(t) as 2^(t log2 e), the product in two parts so that a large |t| costs no bits.
__device__ __forceinline__ float dense_exp(float t) {
  const float a = t * 1.4426950408889634f;
  const float b = fmaxf(fmaf(t, 1.4426950408889634f, -a) + t * 1.925963e-8f, -1.0f);  // (NaN for an infinite t)
  return __builtin_amdgcn_exp2f(a) * fmaf(b, 0.6931471805599453f, 1.0f);
}

// The gated activation of one pair: G = min(g, limit), U = clamp(u, +-limit), s = sigmoid(1.702 G);
// h = (U + 1) G s. A NaN stays one.
struct DenseGate {
  float G, U, s;
  __device__ __forceinline__ DenseGate(float g, float u, float limit) {
    G = g > limit ? limit : g;
    U = rclamp(u, -limit, limit);
    s = __builtin_amdgcn_rcpf(1.0f + dense_exp(-1.702f * G));
  }
  __device__ __forceinline__ float h() const { return (U + 1.0f) * (G * s); }
};

// One operand's tile: R rows (of M or N) x 64 k, W wavefronts loading it.
template <int R, int W, bool TR>
struct DenseTile {
  static constexpr int kBytes = R * 128;
  static constexpr int kLoads = (R / 8 + W - 1) / W;  // LDS-DMAs of 1 KB per wavefront
  static constexpr bool kEven = R / 8 % W == 0;
  static constexpr int kPairs = R / 16;               // 32-byte pieces of a transposed row

  // piece of a transposed row that holds the logical piece q in row k
  static __device__ __forceinline__ int piece(int q, int k) {
    const int f = (k & 3) | ((k >> 1) & 4);
    const int mask = kPairs >= 8 ? ((q | 7) < kPairs ? 7 : (q | 3) < kPairs ? 3 : 0)
                                 : kPairs >= 4 ? ((q | 3) < kPairs ? 3 : 0) : kPairs >= 2 ? 1 : 0;
    return q ^ (f & mask);
  }

  uint32_t off[kLoads];  // byte offset of this lane's 16 bytes from the tile's base
  uint32_t part[kLoads]; // K-contiguous: first k of the lane's chunk; transposed: its row k

  // rows: valid rows from the tile's first; ld: bytes between stored rows
  __device__ __forceinline__ void init(int wave, int lane, int rows, size_t ld) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const int c = (i * W + wave) * 64 + lane;
      if constexpr (!TR) {
        const int row = c >> 3, ch = (c & 7) ^ (row & 7);
        off[i] = (uint32_t)((size_t)min(row, rows - 1) * ld);
        part[i] = ch * 8;
      } else {
        const int k = c / (R / 8), pos = c % (R / 8);
        int col = piece(pos >> 1, k) * 16 + (pos & 1) * 8;  // the permutation is its own inverse
        if (col >= rows) col = 0;
        off[i] = (uint32_t)(col * 2);
        part[i] = k;
      }
    }
  }
  // loads the step whose first k is at `base`; left: k values left in K from there
  __device__ __forceinline__ void load(const uint16_t *base, size_t ld, int left, uint32_t lds, int wave) const {
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      if (!kEven && (i * W + wave) * 8 >= R) continue;
      uint32_t o = off[i];
      if constexpr (!TR)
        o += ((int)part[i] < left ? part[i] : 0u) * 2;
      else
        o += (uint32_t)min((int)part[i], left - 1) * (uint32_t)ld;
      str_dma16(o, base, lds + (i * W + wave) * 1024);
    }
  }
  // zeroes the k values of the step past `left` (the last step of a K that is no multiple of 64)
  __device__ __forceinline__ static void zero_tail(uint8_t *lds, int left, int tid, int threads) {
    for (int c = tid; c < R * 8; c += threads) {
      bool past;
      if constexpr (!TR)
        past = (((c & 7) ^ ((c >> 3) & 7)) * 8) >= left;
      else
        past = c / (R / 8) >= left;
      if (past) *(uint4 *)(lds + c * 16) = uint4{0u, 0u, 0u, 0u};
    }
  }
  // MFMA operand of 16 rows from row0 (tile-relative), k slice kk (32 values)
  static __device__ __forceinline__ bf16x8 frag(const uint8_t *lds, int row0, int kk, int lane) {
    if constexpr (!TR) {
      const int row = row0 + (lane & 15), ch = kk * 4 + (lane >> 4);
      return *(const bf16x8 *)(lds + row * 128 + ((ch ^ (row & 7)) << 4));
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      const int i = lane & 15, k = kk * 32 + (lane >> 4) * 8 + (i >> 2);
      const int q = row0 >> 4;
      auto at = [&](int k) {
        return (__attribute__((address_space(3))) s16x4 *)(lds + k * (R * 2) + piece(q, k) * 32 + (i & 3) * 8);
      };
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(k));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at(k + 4));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

template <int BM, int BN, int WM, int WN, bool AT, bool BT, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void k_dense(const DenseArgs a) {
  constexpr int W = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  using TA = DenseTile<BM, W, AT>;
  using TB = DenseTile<BN, W, BT>;
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int kSlot = TA::kBytes + TB::kBytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int tiles_m = (a.M + BM - 1) / BM;
  const int tile = blockIdx.x;
  const int m0 = tile % tiles_m * BM, n0 = tile / tiles_m * BN;
  const int split = blockIdx.y;
  const int k_lo = split * a.k_split, k_hi = min(a.K, k_lo + a.k_split);
  const int nk = (k_hi - k_lo + kDenseStep - 1) / kDenseStep, steps = nk * a.n_pass;

  const uint32_t lds0 = str_lds(lds);
  TA la;
  TB lb;
  la.init(wave, lane, a.M - m0, a.lda * 2);
  lb.init(wave, lane, a.N - n0, a.ldb * 2);
  int pass = 0, k0 = k_lo;  // of the next step to load
  auto load = [&](int slot) {
    const uint16_t *A = a.A + ((a.pa >> 4 * pass) & 15) * a.a_plane + (AT ? (size_t)k0 * a.lda + m0 : (size_t)m0 * a.lda + k0);
    const uint16_t *B = a.B + ((a.pb >> 4 * pass) & 15) * a.b_plane + (BT ? (size_t)k0 * a.ldb + n0 : (size_t)n0 * a.ldb + k0);
    la.load(A, a.lda * 2, k_hi - k0, lds0 + slot * kSlot, wave);
    lb.load(B, a.ldb * 2, k_hi - k0, lds0 + slot * kSlot + TA::kBytes, wave);
    k0 += kDenseStep;
    if (k0 >= k_hi) {
      k0 = k_lo;
      pass++;
    }
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  load(0);
  int kt = 0;  // step within its pass
  for (int s = 0; s < steps; s++) {
    const int slot = s & 1;
    uint8_t *sl = lds + slot * kSlot;
    // this step's loads have landed, and the wavefront is done reading the other slot
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(vm_lgkm_wait(0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 1 < steps) load(slot ^ 1);
    const int left = k_hi - k_lo - kt * kDenseStep;
    kt = kt + 1 == nk ? 0 : kt + 1;
    if (left < kDenseStep) {
      TA::zero_tail(sl, left, tid, 64 * W);
      TB::zero_tail(sl + TA::kBytes, left, tid, 64 * W);
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt 0
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      bf16x8 fb[TN];
#pragma unroll
      for (int j = 0; j < TN; j++) fb[j] = TB::frag(sl + TA::kBytes, (wn * TN + j) * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const bf16x8 fa = TA::frag(sl, (wm * TM + i) * 16, kk, lane);
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa, fb[j], acc[i][j], 0, 0, 0);
      }
    }
  }

  // lane: column n = lane % 16 of each tile, rows m = lane / 16 * 4 + 0..3
  const int mw = m0 + wm * TM * 16 + (lane >> 4) * 4, nw = n0 + wn * TN * 16 + (lane & 15);
  if constexpr (EPI == DENSE_STORE) {
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int n = nw + j * 16;
      if (n >= a.N) continue;
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const int m = mw + i * 16;
        if (m >= a.M) continue;
        float4 v = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        if (a.bias) {
          const float4 b = *(const float4 *)(a.bias + m);
          v.x += b.x, v.y += b.y, v.z += b.z, v.w += b.w;
        }
        const size_t at = (size_t)n * a.ldo + m;
        if (a.out_mode == 0) {
          const uint2 u = {dense_bf16(v.x) | (uint32_t)dense_bf16(v.y) << 16, dense_bf16(v.z) | (uint32_t)dense_bf16(v.w) << 16};
          *(uint2 *)((uint16_t *)a.out + at) = u;
        } else {
          float4 *o = (float4 *)((float *)a.out + split * a.split_stride + at);
          if (a.out_mode == 2) {
            const float4 b = *o;
            v.x += b.x, v.y += b.y, v.z += b.z, v.w += b.w;
          }
          *o = v;
        }
      }
    }
  } else if constexpr (EPI == DENSE_GATE || EPI == DENSE_GATE_RAW) {
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int n = nw + j * 16;
      if (n >= a.N) continue;
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const int m = mw + i * 16;
        if (m >= a.M) continue;
        float4 v = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        if (a.bias) {
          const float4 b = *(const float4 *)(a.bias + m);
          v.x += b.x, v.y += b.y, v.z += b.z, v.w += b.w;
        }
        if constexpr (EPI == DENSE_GATE_RAW) {
          *(float4 *)(a.gu + (size_t)n * a.M + m) = v;
        } else {
          const float h0 = DenseGate(v.x, v.y, a.limit).h(), h1 = DenseGate(v.z, v.w, a.limit).h();
          uint16_t *o = a.h + (size_t)n * a.ldh + m / 2;
          if (a.planes == 1) {
            *(uint32_t *)o = dense_bf16(h0) | (uint32_t)dense_bf16(h1) << 16;
          } else {
            uint16_t p0[kPlanes], p1[kPlanes];
            dense_split(h0, p0);
            dense_split(h1, p1);
#pragma unroll
            for (int p = 0; p < kPlanes; p++) *(uint32_t *)(o + p * a.h_plane) = p0[p] | (uint32_t)p1[p] << 16;
          }
        }
      }
    }
  } else if constexpr (EPI == DENSE_DGATE) {
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const int m = mw + i * 16;
      float db[8];
#pragma unroll
      for (int r = 0; r < 8; r++) db[r] = 0.0f;
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const int n = nw + j * 16;
        if (n >= a.N || m >= a.M) continue;
        const float *row = a.gu + (size_t)n * a.M * 2 + 2 * m;
        const float4 g01 = *(const float4 *)row, g23 = *(const float4 *)(row + 4);
        const float gate[4] = {g01.x, g01.z, g23.x, g23.z}, up[4] = {g01.y, g01.w, g23.y, g23.w};
        float d[8], hv[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const DenseGate g(gate[r], up[r], a.limit);
          const float dh = acc[i][j][r];
          hv[r] = g.h();
          d[2 * r] = gate[r] > a.limit ? 0.0f : dh * (g.U + 1.0f) * (g.s * (1.0f + 1.702f * (g.G * (1.0f - g.s))));
          d[2 * r + 1] = fabsf(up[r]) > a.limit ? 0.0f : dh * (g.G * g.s);
        }
#pragma unroll
        for (int r = 0; r < 8; r++) db[r] += d[r];
        for (int p = 0; p < a.planes; p++) {  // each plane takes what the planes before it left
          uint16_t q[8], e[4];
#pragma unroll
          for (int r = 0; r < 8; r++) {
            q[r] = dense_bf16(d[r]);
            d[r] = isfinite(bf16_to_f32(q[r])) ? d[r] - bf16_to_f32(q[r]) : 0.0f;
          }
#pragma unroll
          for (int r = 0; r < 4; r++) {
            e[r] = dense_bf16(hv[r]);
            hv[r] = isfinite(bf16_to_f32(e[r])) ? hv[r] - bf16_to_f32(e[r]) : 0.0f;
          }
          *(uint4 *)(a.dgu + p * a.dgu_plane + (size_t)n * a.M * 2 + 2 * m) = __builtin_bit_cast(uint4, q);
          *(uint2 *)(a.h + p * a.h_plane + (size_t)n * a.ldh + m) = __builtin_bit_cast(uint2, e);
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
          float *o = a.db_part + (size_t)(tile / tiles_m * WN + wn) * a.M * 2 + 2 * m;
          *(float4 *)o = make_float4(db[0], db[1], db[2], db[3]);
          *(float4 *)(o + 4) = make_float4(db[4], db[5], db[6], db[7]);
        }
      }
    }
  } else if constexpr (EPI == DENSE_STATS) {
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int n = nw + j * 16;
      const int want = n < a.N ? a.targets[n] : -1;
      float mx = -INFINITY;
      bool nan = false;
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int m = mw + i * 16 + r;
          if (m >= a.M) continue;
          const float l = acc[i][j][r];
          mx = fmaxf(mx, l);
          nan |= l != l;
          if (a.v0 + m == want) a.picked[n] = l;
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      // no value above minus infinity: every exponential is 0 against a base of 0
      const float base = mx == -INFINITY ? 0.0f : mx;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (mw + i * 16 + r < a.M) sum += dense_exp(acc[i][j][r] - base);
      if (nan) sum = NAN;
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lane < 16 && n < a.N) a.stats[(size_t)(tile % tiles_m * WM + wm) * a.N + n] = make_float2(mx, sum);
    }
  } else {
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int n = nw + j * 16;
      if (n >= a.N) continue;
      const int t = a.targets[n];
      const float lse = a.lse[n], scale = a.dloss[n];
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const int m = mw + i * 16;
        if ((size_t)m >= a.ld_dl) continue;
        float d[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
          d[r] = scale * (dense_exp(acc[i][j][r] - lse) - (a.v0 + m + r == t ? 1.0f : 0.0f));
          if (t >= a.vocab) d[r] = NAN;
          if (t < 0 || m + r >= a.M) d[r] = 0.0f;  // ignored token, padding column
        }
        for (int p = 0; p < a.planes; p++) {
          uint16_t q[4];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            q[r] = dense_bf16(d[r]);
            d[r] = isfinite(bf16_to_f32(q[r])) ? d[r] - bf16_to_f32(q[r]) : 0.0f;
          }
          *(uint2 *)(a.dl + p * a.dl_plane + (size_t)n * a.ld_dl + m) = __builtin_bit_cast(uint2, q);
        }
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, bool AT, bool BT, int EPI>
hipError_t launch_dense_as(const DenseArgs &a, hipStream_t st) {
  static DynLdsOnce once;
  const size_t bytes = 2 * (BM + BN) * 128;
  auto kernel = k_dense<BM, BN, WM, WN, AT, BT, EPI>;
  hipError_t e = ensure_dyn_lds(once, (const void *)kernel, bytes);
  if (e != hipSuccess) return e;
  const size_t tiles = (size_t)((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  if (tiles > 0x7FFFFFFF || a.splits > 65535) return hipErrorInvalidValue;
  kernel<<<dim3((unsigned)tiles, a.splits), 64 * WM * WN, bytes, st>>>(a);
  return hipGetLastError();
}

}  // namespace moe
