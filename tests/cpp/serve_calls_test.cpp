// The calls of include/moe_serve.h replayed on the host: csrc/serve_api.cpp as it is, over launches and allocations that
// only note what they would read and write.
//   serve_calls_test refusals   calls that must be refused before anything is launched or allocated
//   serve_calls_test calls      calls of drawn sizes: every launch stays in the caller's buffers and the workspace, the pieces
//                               of a call cover each output once, and what a piece reads of the workspace it wrote
#include <cmath>
#include <cstdio>
#include <cstring>
#include <map>
#include <random>
#include <string>
#include <vector>

#include "../../silentotithrandousha_amd/csrc/call.hpp"
#include "../../silentotithrandousha_amd/csrc/serve.hpp"

using namespace moe;

struct moe_ctx {
  DenseCtx d;
};

namespace {

std::string g_error;
long g_faults, g_launches, g_allocations;
bool g_capturing;

void fault(const char *what) {
  if (g_faults++ < 20) printf("FAULT %s\n", what);
}

struct Buffer {
  size_t bytes;
  std::vector<std::pair<uintptr_t, uintptr_t>> written;
};
std::map<uintptr_t, Buffer> g_buffers;
uintptr_t g_next = (uintptr_t)1 << 40;

void *buffer(size_t bytes) {
  const uintptr_t at = g_next;
  g_next += (bytes + 0x1FFFFF) & ~(uintptr_t)0xFFFFF;
  g_buffers[at].bytes = bytes;
  return (void *)at;
}
Buffer *holding(const void *p, size_t bytes) {
  auto it = g_buffers.upper_bound((uintptr_t)p);
  if (it == g_buffers.begin()) return nullptr;
  --it;
  return (uintptr_t)p + bytes <= it->first + it->second.bytes ? &it->second : nullptr;
}
void read(const void *p, size_t bytes) {
  if (bytes && !holding(p, bytes)) fault("a read outside the buffers");
}
void write(const void *p, size_t bytes) {
  Buffer *b = holding(p, bytes);
  if (!b) return fault("a write outside the buffers");
  b->written.push_back({(uintptr_t)p, (uintptr_t)p + bytes});
}
// every byte of an output once
void whole(const void *p, size_t bytes) {
  auto &w = g_buffers[(uintptr_t)p].written;
  uintptr_t at = (uintptr_t)p;
  for (auto &v : w) {
    if (v.first != at) fault("pieces that do not join");
    at = v.second;
  }
  if (at != (uintptr_t)p + bytes) fault("an output that is not written whole");
}

struct {
  const void *codes, *scales;
  size_t tokens;
} g_rows;

}  // namespace

namespace moe {
int api_fail(int code, const char *msg) {
  g_error = msg;
  return code;
}
int dense_ctx(moe_ctx *c, DenseCtx *d) {
  if (!c) return fail(MOE_ERR_INVALID, "null context");
  *d = c->d;
  return MOE_OK;
}
hipError_t launch_mx4_quantize(const void *x, bool bf16, size_t n, size_t cols, uint8_t *blocks, uint8_t *scales, hipStream_t) {
  g_launches++;
  read(x, n * cols * (bf16 ? 2 : 4));
  write(blocks, n * cols / 2);
  write(scales, n * cols / 32);
  return hipSuccess;
}
hipError_t launch_mx_rows(const MxRows &r, const void *x, const uint8_t *x_scales, uint8_t *codes, uint32_t *scales, hipStream_t) {
  g_launches++;
  const size_t values = (size_t)r.tokens * r.nb * 32;
  read(x, r.type == MOE_F32 ? values * 4 : r.type == MOE_BF16 ? values * 2 : r.type == MOE_MXFP8 ? values : values / 2);
  if (r.type >= MOE_MXFP8) read(x_scales, values / 32);
  write(codes, mx_rows_code_bytes(r));
  write(scales, mx_rows_scale_bytes(r));
  if ((size_t)r.tiles * r.ns > (size_t)1 << 25 || 16 * (size_t)r.ns * r.terms * r.chunk >> 32) fault("a piece above what the kernels take");
  if ((uintptr_t)codes % 256 || (uintptr_t)scales % 256 || !(codes + mx_rows_code_bytes(r) <= (uint8_t *)scales)) fault("the workspace's parts");
  g_rows = {codes, scales, r.tokens};
  return hipSuccess;
}
static hipError_t product(const MxGemmArgs &a) {
  g_launches++;
  read(a.w, pack_weight_bytes(a.d));
  if (a.bias) read(a.bias, (size_t)a.d.rows * 4);
  write(a.out, (size_t)a.r.tokens * a.d.rows * (a.bf16 ? 2 : 4));
  return hipSuccess;
}
hipError_t launch_mx_gemm(const MxGemmArgs &a, hipStream_t) {
  if (a.codes != g_rows.codes || a.scales != g_rows.scales || a.r.tokens != g_rows.tokens) fault("rows of another piece");
  return product(a);
}
hipError_t launch_mx_one(const MxGemmArgs &a, const void *x, hipStream_t) {
  read(x, (size_t)a.r.tokens * a.r.nb * 32 * (a.r.type == MOE_F32 ? 4 : 2));
  if ((size_t)a.r.tokens * a.r.terms > 16) fault("more terms than columns");
  return product(a);
}
hipError_t launch_route_rule(const RouteRule &r, const float *logits, size_t T, int E, int32_t *idx, float *w, int32_t *counts, hipStream_t) {
  g_launches++;
  read(logits, T * E * 4);
  if (r.bias) read(r.bias, (size_t)E * 4);
  if (T) write(idx, T * r.k * 4), write(w, T * r.k * 4);
  if (counts) write(counts, (size_t)E * 4);
  return hipSuccess;
}
hipError_t launch_route_rule_backward(const RouteRule &r, const float *logits, const int32_t *idx, const float *dw, size_t T, int E, float *dl,
                                      hipStream_t) {
  g_launches++;
  read(logits, T * E * 4), read(idx, T * r.k * 4), read(dw, T * r.k * 4);
  write(dl, T * E * 4);
  return hipSuccess;
}
size_t sample_workspace(size_t T, size_t V) { return T * 57000 + T * ((V + 2047) / 2048) * 12; }
hipError_t launch_sample(const SampleArgs &a, hipStream_t) {
  g_launches++;
  read(a.logits, ((size_t)(a.T - 1) * a.ld + a.V) * 4);
  read(a.u, (size_t)a.T * 4);
  for (const void *p : {(const void *)a.rule.temperature, (const void *)a.rule.top_k, (const void *)a.rule.top_p, (const void *)a.rule.min_p})
    if (p) read(p, (size_t)a.T * 4);
  write(a.work, sample_workspace(a.T, a.V));
  write(a.tokens, (size_t)a.T * 4);
  if (a.logprob) write(a.logprob, (size_t)a.T * 4);
  return hipSuccess;
}
}  // namespace moe

extern "C" {
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
  *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t bytes) {
  g_allocations++;
  *p = buffer(bytes);
  return hipSuccess;
}
hipError_t hipFree(void *p) {
  g_buffers.erase((uintptr_t)p);
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "error"; }
}

namespace {

DenseWork g_work;
moe_ctx g_ctx{};

template <class T = uint8_t>
T *device(size_t bytes) {
  return (T *)buffer(bytes);
}

int refusals() {
  int wrong = 0, n = 0;
  auto refused = [&](int rc, const char *says, int code = MOE_ERR_INVALID) {
    n++;
    if (rc != code || g_error.find(says) == std::string::npos || g_launches || g_allocations) {
      wrong++;
      printf("call %d: status %d, \"%s\" (not \"%s\")\n", n, rc, g_error.c_str(), says);
    }
    g_launches = 0;
    g_error.clear();
  };
  moe_ctx *c = &g_ctx;
  uint8_t *x = device(4096), *y = device(4096), *s = device(4096);
  float *xf = (float *)x, *yf = (float *)y, *sf = (float *)s;
  int32_t *yi = (int32_t *)y, *si = (int32_t *)s;
  auto quantize = [&](const void *x, int dtype, size_t n, size_t cols, uint8_t *b, uint8_t *s) {
    return moe_mxfp4_quantize_device(c, x, dtype, n, cols, b, s, nullptr);
  };
  refused(moe_mxfp4_quantize_device(nullptr, x, 0, 1, 32, y, s, nullptr), "null context");
  refused(quantize(x, 2, 1, 32, y, s), "dtype 2");
  refused(quantize(x, -1, 1, 32, y, s), "dtype -1");
  for (size_t cols : {(size_t)0, (size_t)1, (size_t)33, ((size_t)1 << 20) + 32, (size_t)-32}) refused(quantize(x, 0, 1, cols, y, s), "cols");
  for (size_t rows : {((size_t)1 << 24) + 1, (size_t)-1}) refused(quantize(x, 0, rows, 32, y, s), "n_rows");
  refused(quantize(nullptr, 0, 1, 32, y, s), "null");
  refused(quantize(x, 0, 1, 32, nullptr, s), "null");
  refused(quantize(x, 0, 1, 32, y, nullptr), "null");
  refused(quantize(x + 4, 0, 1, 32, y, s), "aligned");
  refused(quantize(x, 0, 1, 32, y + 8, s), "aligned");
  refused(quantize(x, 0, 1, 32, x, s), "an output is also an input");
  refused(quantize(x, 0, 1, 32, y, y), "two outputs");

  auto matmul = [&](const void *p, size_t rows, size_t cols, const void *bias, const void *x, int x_type, const void *xs, size_t T, void *y, int dtype) {
    return moe_mxfp4_matmul_device(c, (const uint8_t *)p, rows, cols, (const float *)bias, x, x_type, (const uint8_t *)xs, T, y, dtype, nullptr);
  };
  for (int t : {-1, 4}) refused(matmul(s, 16, 32, nullptr, x, t, nullptr, 1, y, 0), "x_type");
  for (int t : {-1, 2, 3}) refused(matmul(s, 16, 32, nullptr, x, 0, nullptr, 1, y, t), "dtype");
  for (size_t rows : {(size_t)0, (size_t)15, ((size_t)1 << 24) + 16, (size_t)-16}) refused(matmul(s, rows, 32, nullptr, x, 0, nullptr, 1, y, 0), "rows");
  for (size_t cols : {(size_t)0, (size_t)48, ((size_t)1 << 20) + 32}) refused(matmul(s, 16, cols, nullptr, x, 0, nullptr, 1, y, 0), "cols");
  refused(matmul(s, 16, 32, nullptr, x, 0, nullptr, ((size_t)1 << 20) + 1, y, 0), "n_tokens");
  refused(matmul(s, 16, 32, nullptr, x, MOE_MXFP4, nullptr, 1, y, 0), "x_scales");
  refused(matmul(nullptr, 16, 32, nullptr, x, 0, nullptr, 1, y, 0), "null");
  refused(matmul(s, 16, 32, nullptr, nullptr, 0, nullptr, 1, y, 0), "null");
  refused(matmul(s, 16, 32, nullptr, x, 0, nullptr, 1, nullptr, 0), "null");
  refused(matmul(s + 4, 16, 32, nullptr, x, 0, nullptr, 1, y, 0), "aligned");
  refused(matmul(s, 16, 32, s + 4, x, 0, nullptr, 1, y, 0), "aligned");
  refused(matmul(s, 16, 32, nullptr, x + 8, 0, nullptr, 1, y, 0), "aligned");
  refused(matmul(s, 16, 32, nullptr, x, 0, nullptr, 1, y + 4, 0), "aligned");
  refused(matmul(s, 16, 32, nullptr, x, 0, nullptr, 1, x, 0), "an output is also an input");
  refused(matmul(s, 16, 32, y, x, 0, nullptr, 1, y, 0), "an output is also an input");
  refused(matmul(s, 16, 32, nullptr, x, MOE_MXFP4, y, 1, y, 0), "an output is also an input");
  g_capturing = true;
  refused(matmul(s, 16, 32, nullptr, x, 0, nullptr, 3, y, 0), "workspace", MOE_ERR_STATE);
  g_capturing = false;

  const moe_routing good{0, 1, 2, 0, 0, 0, 1.0f, nullptr};
  auto rule = [&](auto change) {
    moe_routing r = good;
    change(r);
    return r;
  };
  auto route = [&](const moe_routing &r, size_t E = 8, size_t T = 1) { return moe_route_device(c, &r, xf, T, E, yi, sf, nullptr, nullptr); };
  auto back = [&](const moe_routing &r, size_t E = 8, size_t T = 1) { return moe_route_backward_device(c, &r, xf, si, sf, T, E, yf, nullptr); };
  auto both = [&](const moe_routing &r, const char *says, size_t E = 8, size_t T = 1) {
    refused(route(r, E, T), says);
    refused(back(r, E, T), says);
  };
  for (size_t k : {(size_t)0, (size_t)9, (size_t)33, (size_t)-1}) both(rule([&](auto &r) { r.top_k = k; }), "top_k");
  both(rule([](auto &r) { r.top_k = 33; }), "top_k", 1024);
  for (int v : {-1, 2}) both(rule([&](auto &r) { r.score = v; }), "score");
  for (float v : {(float)NAN, (float)INFINITY, (float)-INFINITY}) both(rule([&](auto &r) { r.scale = v; }), "scale");
  both(rule([](auto &r) { r.n_groups = 3, r.top_groups = 1; }), "n_groups");
  both(rule([](auto &r) { r.n_groups = 65, r.top_groups = 1, r.top_k = 1; }), "n_groups", 130);
  both(rule([](auto &r) { r.n_groups = (size_t)-1, r.top_groups = 1; }), "n_groups");
  for (size_t g : {(size_t)0, (size_t)5}) both(rule([&](auto &r) { r.n_groups = 4, r.top_groups = g; }), "top_groups");
  both(rule([](auto &r) { r.n_groups = 4, r.top_groups = 1, r.top_k = 3; }), "top_k");
  both(rule([](auto &r) { r.n_groups = 4, r.top_groups = 2, r.group_score = 2; }), "group_score");
  both(rule([&](auto &r) { r.bias = (const float *)(x + 2); }), "aligned");
  for (size_t E : {(size_t)0, (size_t)1025, (size_t)-1}) both(good, "n_experts", E);
  both(good, "n_tokens", 8, ((size_t)1 << 20) + 1);
  refused(moe_route_device(c, nullptr, xf, 1, 8, yi, sf, nullptr, nullptr), "null rule");
  refused(moe_route_device(c, &good, nullptr, 1, 8, yi, sf, nullptr, nullptr), "null");
  refused(moe_route_device(c, &good, xf, 1, 8, nullptr, sf, nullptr, nullptr), "null");
  refused(moe_route_device(c, &good, xf, 1, 8, yi, nullptr, nullptr, nullptr), "null");
  refused(moe_route_device(c, &good, (float *)(x + 2), 1, 8, yi, sf, nullptr, nullptr), "aligned");
  refused(moe_route_device(c, &good, xf, 1, 8, yi, sf, (int32_t *)(x + 2), nullptr), "aligned");
  refused(moe_route_device(c, &good, xf, 1, 8, (int32_t *)(y + 1), sf, nullptr, nullptr), "aligned");
  refused(moe_route_device(c, &good, xf, 1, 8, yi, yf, nullptr, nullptr), "two outputs");
  refused(moe_route_device(c, &good, xf, 1, 8, yi, sf, yi, nullptr), "two outputs");
  refused(moe_route_device(c, &good, xf, 1, 8, (int32_t *)x, sf, nullptr, nullptr), "an output is also an input");
  const moe_routing biased = rule([&](auto &r) { r.bias = sf; });
  refused(moe_route_device(c, &biased, xf, 1, 8, yi, sf, nullptr, nullptr), "an output is also an input");
  refused(moe_route_device(c, &biased, nullptr, 0, 8, nullptr, nullptr, si, nullptr), "an output is also an input");
  refused(moe_route_backward_device(c, nullptr, xf, si, sf, 1, 8, yf, nullptr), "null rule");
  refused(moe_route_backward_device(c, &good, nullptr, si, sf, 1, 8, yf, nullptr), "null");
  refused(moe_route_backward_device(c, &good, xf, nullptr, sf, 1, 8, yf, nullptr), "null");
  refused(moe_route_backward_device(c, &good, xf, si, nullptr, 1, 8, yf, nullptr), "null");
  refused(moe_route_backward_device(c, &good, xf, si, sf, 1, 8, nullptr, nullptr), "null");
  refused(moe_route_backward_device(c, &good, xf, si, sf, 1, 8, sf, nullptr), "an output is also an input");
  refused(moe_route_backward_device(c, &good, xf, si, sf, 1, 8, (float *)(y + 2), nullptr), "aligned");

  moe_sampling none{};
  auto sample = [&](const moe_sampling &r, size_t T, size_t V, size_t ld) { return moe_sample_device(c, &r, xf, ld, yf, T, V, si, nullptr, nullptr); };
  refused(sample(none, 1, 8, 7), "ld");
  refused(sample(none, 1, 0, 8), "vocab");
  refused(sample(none, 1, ((size_t)1 << 28) + 1, ((size_t)1 << 28) + 1), "vocab");
  refused(sample(none, ((size_t)1 << 20) + 1, 8, 8), "n_tokens");
  refused(sample(moe_sampling{(const float *)(x + 1), nullptr, nullptr, nullptr}, 1, 8, 8), "aligned");
  refused(sample(moe_sampling{nullptr, (const int32_t *)(x + 2), nullptr, nullptr}, 1, 8, 8), "aligned");
  refused(sample(moe_sampling{nullptr, nullptr, nullptr, sf}, 1, 8, 8), "an output is also an input");
  refused(moe_sample_device(c, nullptr, xf, 8, yf, 1, 8, si, nullptr, nullptr), "null rule");
  refused(moe_sample_device(c, &none, nullptr, 8, yf, 1, 8, si, nullptr, nullptr), "null");
  refused(moe_sample_device(c, &none, xf, 8, nullptr, 1, 8, si, nullptr, nullptr), "null");
  refused(moe_sample_device(c, &none, xf, 8, yf, 1, 8, nullptr, nullptr, nullptr), "null");
  refused(moe_sample_device(c, &none, xf, 8, yf, 1, 8, yi, nullptr, nullptr), "an output is also an input");
  refused(moe_sample_device(c, &none, xf, 8, yf, 1, 8, si, sf, nullptr), "two outputs");
  refused(moe_sample_device(c, &none, (float *)(x + 2), 8, yf, 1, 8, si, nullptr, nullptr), "aligned");
  g_capturing = true;
  refused(sample(none, 1, 8, 8), "workspace", MOE_ERR_STATE);
  g_capturing = false;
  printf("%d refusals, %d wrong\n", n, wrong);
  return wrong != 0;
}

int calls() {
  std::mt19937_64 rng(1);
  auto draw = [&](double most) { return (size_t)std::floor(std::exp(std::uniform_real_distribution<double>(0, std::log(most + 1))(rng))); };
  auto clear = [&] {
    for (auto it = g_buffers.begin(); it != g_buffers.end();)
      it = it->first == (uintptr_t)g_work.p ? (it->second.written.clear(), std::next(it)) : g_buffers.erase(it);
  };
  auto fine = [&](int rc) {
    if (rc) fault(g_error.c_str());
  };
  for (int i = 0; i < 20000; i++) {
    const size_t T = draw(1 << 20), rows = 16 * draw(1 << 12), cols = 32 * draw(i % 3 ? 256 : 1 << 15);
    const int type = (int)(rng() % 4), dtype = (int)(rng() % 2);
    const size_t el = dtype ? 2 : 4;
    {
      const PackDims d = pack_dims(rows, cols);
      const size_t xb = T * cols * (type == MOE_F32 ? 8 : type == MOE_BF16 ? 4 : type == MOE_MXFP8 ? 2 : 1) / 2;
      const bool behind = type == MOE_MXFP8 && rng() % 2;
      void *y = buffer(T * rows * el);
      fine(moe_mxfp4_matmul_device(&g_ctx, device(pack_weight_bytes(d) + pack_scale_bytes(d)), rows, cols, rng() % 2 ? device<float>(rows * 4) : nullptr,
                                   buffer(xb + (behind ? T * cols / 32 : 0)), type, type < MOE_MXFP8 || behind ? nullptr : device(T * cols / 32), T, y,
                                   dtype, nullptr));
      whole(y, T * rows * el);
      clear();
    }
    {
      const size_t n = T;
      uint8_t *b = device(n * cols / 2), *s = device(n * cols / 32);
      fine(moe_mxfp4_quantize_device(&g_ctx, buffer(n * cols * el), dtype, n, cols, b, s, nullptr));
      whole(b, n * cols / 2);
      whole(s, n * cols / 32);
      clear();
    }
    {
      const size_t V = draw(1 << 20), ld = V + rng() % 100, t = std::min<size_t>(T, 20000);
      auto some = [&] { return rng() % 2 ? buffer(t * 4) : nullptr; };
      const moe_sampling r{(float *)some(), (int32_t *)some(), (float *)some(), (float *)some()};
      int32_t *tokens = device<int32_t>(t * 4);
      float *lp = (float *)some();
      fine(moe_sample_device(&g_ctx, &r, device<float>(((t - 1) * ld + V) * 4), ld, device<float>(t * 4), t, V, tokens, lp, nullptr));
      whole(tokens, t * 4);
      if (lp) whole(lp, t * 4);
      clear();
    }
  }
  printf("faults %ld\n", g_faults);
  return g_faults ? 3 : 0;
}

}  // namespace

int main(int argc, char **argv) {
  g_ctx.d.H = 32;
  g_ctx.d.work = &g_work;
  const std::string what = argc > 1 ? argv[1] : "";
  return what == "refusals" ? refusals() : what == "calls" ? calls() : 2;
}
