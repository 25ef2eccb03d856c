// The dense products of few rows (up to 8, a row's planes counted): the weights stream once through
// registers, no LDS.
//
// A workgroup takes 8 to 24 rows of A; its 8 wavefronts take the K-steps of 64 values in turn, each with the
// loads of its next 6 steps under way, and their sums join in LDS, in order. Bound by the weights' bytes
// and the latency of the first of them: one row of 2880 x 2880 weights (33 MB of gate and up, 16.6 MB
// down) takes 9.0 and 4.9 us, both 13.3 with the launches (10.1 and 5.5, 15.0, with 16 rows a workgroup; 10.6 and
// 8.3, with the sum of its K parts, through the LDS rings of dense_gemm.hpp).
#include "dense_gemm.hpp"
#include "dense_launch.hpp"

namespace moe {
namespace {

constexpr int kWaves = 8, kAhead = 6;

template <int ROWS, int EPI>
__global__ __launch_bounds__(64 * kWaves) void k_dense_few(const DenseArgs a) {
  constexpr int kTiles = (ROWS + 15) / 16;
  __shared__ float s_sum[kWaves][16][16 * kTiles + 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = blockIdx.x * ROWS, rows_b = a.N * a.stack, at = lane >> 4;
  const int row_b = min(lane & 15, rows_b - 1);  // of the stacked planes, which may lie in every other slot
  const uint16_t *A[kTiles], *B = a.B + (size_t)(row_b + row_b / a.N * a.N * (a.stack_step - 1)) * a.ldb;
#pragma unroll
  for (int t = 0; t < kTiles; t++)  // (of a part of a tile the lanes past it read its last row)
    A[t] = a.A + (size_t)min(m0 + min(t * 16 + (lane & 15), ROWS - 1), a.M - 1) * a.lda;
  const int steps = (a.K + kDenseStep - 1) / kDenseStep;
  f32x4 acc[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = wave; s0 < steps; s0 += kWaves * kAhead) {
    uint4 fa[kAhead][2][kTiles], fb[kAhead][2];
#pragma unroll
    for (int i = 0; i < kAhead; i++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int k = (s0 + i * kWaves) * kDenseStep + h * kDenseHalf + at * 8, c = min(k, a.K - 8);
        const bool in = k < a.K;  // (K is a multiple of 8)
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
          fa[i][h][t] = *(const uint4 *)(A[t] + c);
          if (!in) fa[i][h][t] = uint4{0u, 0u, 0u, 0u};
        }
        fb[i][h] = *(const uint4 *)(B + c);
        if (!in) fb[i][h] = uint4{0u, 0u, 0u, 0u};
      }
#pragma unroll
    for (int i = 0; i < kAhead; i++)
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int t = 0; t < kTiles; t++)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(fa[i][h][t]), as_bf16x8(fb[i][h]), acc[t], 0, 0, 0);
  }
#pragma unroll
  for (int t = 0; t < kTiles; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) s_sum[wave][lane & 15][t * 16 + at * 4 + r] = acc[t][r];
  __syncthreads();
  // the sum of the wavefronts' parts, and of a row's planes
  auto sum = [&](int n, int m) __attribute__((always_inline)) {
    float v = 0.0f;
    for (int p = 0; p < a.stack; p++)
#pragma unroll
      for (int w = 0; w < kWaves; w++) v += s_sum[w][p * a.N + n][m];
    return v + (a.bias ? a.bias[m0 + m] : 0.0f);
  };
  if constexpr (EPI == DENSE_STORE) {
    const int n = threadIdx.x / ROWS, m = threadIdx.x % ROWS;
    if (n < a.N && m0 + m < a.M) {
      const float v = sum(n, m);
      const size_t o = (size_t)n * a.ldo + m0 + m;
      if (a.out_mode == 0)
        ((uint16_t *)a.out)[o] = dense_bf16(v);
      else
        ((float *)a.out)[o] = v;
    }
  } else {
    const int n = threadIdx.x / (ROWS / 2), i = threadIdx.x % (ROWS / 2);
    if (n < a.N && m0 + 2 * i < a.M) {
      DenseGate g;
      g.set<false>(sum(n, 2 * i), sum(n, 2 * i + 1), a.limit);
      uint16_t q[kPlanes];
      dense_split(g.h(), q);
      for (int p = 0; p < a.planes; p++)
        dense_slots<false>(a.h_where, p, q[p], [&](size_t at, uint16_t v) { a.h[at * a.h_slot + (size_t)n * a.ldh + m0 / 2 + i] = v; });
    }
  }
}

template <int ROWS>
hipError_t launch_few(const DenseShape &s, const DenseArgs &a, hipStream_t st) {
  const unsigned grid = (unsigned)((a.M + ROWS - 1) / ROWS);
  return launch_own(s.epi == DENSE_GATE ? k_dense_few<ROWS, DENSE_GATE> : k_dense_few<ROWS, DENSE_STORE>, grid, 64 * kWaves, 0, st, a);
}

}  // namespace

hipError_t launch_dense_few(const DenseShape &s, const DenseArgs &a, hipStream_t st) {
  switch (dense_few_rows(s, a)) {
    case 8: return launch_few<8>(s, a, st);
    case 12: return launch_few<12>(s, a, st);
    case 16: return launch_few<16>(s, a, st);
    case 24: return launch_few<24>(s, a, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace moe
