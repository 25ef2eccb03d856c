// Host interface of the kernels behind include/moe_serve.h: MXFP4 quantisation (mx_quant.hip), products with
// a resident MXFP4 matrix (mx_gemm.hip), routing rules (route_rule.hip), sampling (sample.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/moe_serve.h"
#include "layout.hpp"

namespace moe {

hipError_t launch_mx4_quantize(const void *x, bool bf16, size_t n, size_t cols, uint8_t *blocks, uint8_t *scales, hipStream_t s);

// What a product makes of its rows: tiles of 16 rows x steps of 128 values as the MFMA's B operand takes them. Step s of tile n lies
// at ((n ns + s) terms) * chunk bytes, one chunk a term: lane l = 16 g + j holds block 4 s + g of row 16 n + j, in planes of 16
// (and 8 or 16) bytes a lane; bf16 rows' chunk is four planes of 8 values a lane. Behind the tiles (but of bf16 rows), a scale word per
// (tile, 4 steps, lane), byte i that of step 4 q + i: the weights' layout (layout.hpp). All terms share the byte: an E2M3 term t's
// is 5 t below it, at least 1.
struct MxRows {
  int type;     // MOE_F32, MOE_BF16, MOE_MXFP8, MOE_MXFP4
  uint32_t tokens, nb, ns, nq, tiles;
  int terms, chunk;  // terms a value, bytes of a chunk
};
inline MxRows mx_rows(int type, size_t tokens, size_t cols) {
  MxRows r{};
  r.type = type;
  r.tokens = (uint32_t)tokens;
  r.nb = (uint32_t)(cols / 32);
  r.ns = (r.nb + 3) / 4;
  r.nq = (r.ns + 3) / 4;
  r.tiles = (uint32_t)((tokens + 15) / 16);
  r.terms = type == MOE_F32 ? 6 : type == MOE_MXFP8 ? 2 : 1;
  r.chunk = type == MOE_MXFP4 ? 1024 : type == MOE_MXFP8 ? 2048 : type == MOE_BF16 ? 4096 : 1536;
  return r;
}
inline size_t mx_rows_code_bytes(const MxRows &r) { return (size_t)r.tiles * r.ns * r.terms * r.chunk; }
inline size_t mx_rows_scale_bytes(const MxRows &r) { return r.type == MOE_BF16 ? 0 : (size_t)r.tiles * r.nq * 256; }
hipError_t launch_mx_rows(const MxRows &r, const void *x, const uint8_t *x_scales, uint8_t *codes, uint32_t *scales, hipStream_t s);

struct MxGemmArgs {
  const uint8_t *w;      // resident matrix (layout.hpp)
  PackDims d;
  MxRows r;
  const uint8_t *codes;  // rows (MxRows)
  const uint32_t *scales;
  const float *bias;     // [rows] or NULL
  void *out;             // [tokens][rows]
  bool bf16;
  int strip;             // set by the launch
};
hipError_t launch_mx_gemm(const MxGemmArgs &a, hipStream_t s);
// The form for few rows (mx_few.hip).
hipError_t launch_mx_few(const MxGemmArgs &a, hipStream_t s);
// Few rows x without MxRows (a.codes, a.scales): bf16 rows, or the terms of f32 rows, that fit the MFMA's 16 columns and 64 KB of LDS.
constexpr size_t mx_one_rows(size_t nb, size_t tokens) { return ((nb + 3) / 4 * 16 + 1) * 16 * tokens; }
constexpr size_t mx_one_lds(size_t nb, size_t columns) { return (nb + 3) / 4 * 4 * columns * 28 + 8 * 64 * 16 + 1024; }
inline bool mx_one_takes(int type, size_t tokens, size_t cols) {
  if (type == MOE_BF16) return tokens <= 16 && mx_one_rows(cols / 32, tokens) + 16 * 1024 <= 64 * 1024;
  return type == MOE_F32 && tokens <= 2 && mx_one_lds(cols / 32, 6 * tokens) <= 64 * 1024;
}
hipError_t launch_mx_one(const MxGemmArgs &a, const void *x, hipStream_t s);

struct RouteRule {
  int score, normalize, k, groups, top_groups, two;
  float scale;
  const float *bias;
};
hipError_t launch_route_rule(const RouteRule &r, const float *logits, size_t T, int E, int32_t *idx, float *w, int32_t *counts, hipStream_t s);
hipError_t launch_route_rule_backward(const RouteRule &r, const float *logits, const int32_t *idx, const float *dw, size_t T, int E, float *dl,
                                      hipStream_t s);

// Bits of the largest logit's mass in a row of V: 44, fewer where the sum of V such masses would pass 2^62 (V at most 2^28).
constexpr int sample_shift(size_t V) {
  int s = 44;
  while (V > (size_t)1 << (62 - s)) s--;
  return s;
}
// Logits of a row that a workgroup of 512 threads takes in the launch that looks for the largest, and rows at once: a launch has less than
// 2^32 threads.
constexpr size_t kSampleSpan = 4 * 2048;
constexpr size_t sample_rows(size_t V) {
  const size_t rows = (((size_t)1 << 23) - 1) / ((V + kSampleSpan - 1) / kSampleSpan);
  return rows < 4096 ? rows : 4096;
}
struct SampleArgs {
  moe_sampling rule;
  const float *logits;
  size_t ld;
  const float *u;
  uint32_t T, V;
  int32_t *tokens;
  float *logprob;
  // workspace, sized by sample_workspace
  void *work;
};
size_t sample_workspace(size_t T, size_t V);
hipError_t launch_sample(const SampleArgs &a, hipStream_t s);

}  // namespace moe
