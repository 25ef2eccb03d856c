// The serving operators through the C++ mirror (silentotithrandousha_amd/host/gpu_moe_dispatcher.hpp): a head quantised to
// MXFP4, its product, the choice of experts and a token from the results, each against plain loops.
//   serve_mirror_test cpu   what needs no device
//   serve_mirror_test gpu   the run
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>

#include "../../silentotithrandousha_amd/host/gpu_moe_dispatcher.hpp"

using namespace silentot;

static int failures = 0;
#define EXPECT(c, ...)                                 \
  do {                                                 \
    if (!(c)) {                                        \
      std::printf("FAIL %s:%d: ", __FILE__, __LINE__); \
      std::printf(__VA_ARGS__);                        \
      std::printf("\n");                               \
      failures++;                                      \
    }                                                  \
  } while (0)

template <class F>
static bool panics(F &&f) {
  try {
    f();
  } catch (const MoePanic &e) {
    return e.status == MOE_ERR_INVALID;
  }
  return false;
}

static int run_cpu() {
  GpuMoeDispatcher none;  // without a context every call is an error, not a crash
  EXPECT(panics([&] { none.mxfp4_quantize_device(nullptr, MOE_F32, 1, 32, nullptr, nullptr); }), "quantise");
  EXPECT(panics([&] { none.mxfp4_matmul_device(nullptr, 16, 32, nullptr, nullptr, MOE_MXFP4, nullptr, 1, nullptr, MOE_F32); }), "product");
  EXPECT(panics([&] { none.route_device(moe_routing{}, nullptr, 1, 8, nullptr, nullptr); }), "route");
  EXPECT(panics([&] { none.route_backward_device(moe_routing{}, nullptr, nullptr, nullptr, 1, 8, nullptr); }), "route's gradient");
  EXPECT(panics([&] { none.sample_device(moe_sampling{}, nullptr, 8, nullptr, 1, 8, nullptr); }), "sample");
  std::printf("cpu: %s\n", failures ? "FAILED" : "ok");
  return failures ? 1 : 0;
}

template <class T>
struct Device {
  T *p = nullptr;
  size_t n;
  explicit Device(size_t n) : n(n) { moe_check(moe_device_alloc(n * sizeof(T), (void **)&p)); }
  explicit Device(const std::vector<T> &v) : Device(v.size()) { moe_check(moe_memcpy_h2d(p, v.data(), n * sizeof(T))); }
  Device(const Device &) = delete;
  ~Device() { moe_device_free(p); }
  std::vector<T> get() const {
    std::vector<T> v(n);
    moe_check(moe_memcpy_d2h(v.data(), p, n * sizeof(T)));
    return v;
  }
};

static int run_gpu() {
  const size_t T = 5, H = 64, R = 48, K = 3;
  auto d = GpuMoeDispatcher::create(H, 32, 7.0f).unwrap();
  std::mt19937 rng(1);
  std::normal_distribution<float> normal;
  std::vector<float> x(T * H), w(R * H), u(T), dw(T * K);
  for (auto &v : x) v = normal(rng);
  for (auto &v : w) v = normal(rng) / 8;
  for (auto &v : dw) v = normal(rng);
  for (size_t t = 0; t < T; t++) u[t] = (t + 0.5f) / T;
  Device<float> dx(x), dweights(w), y(T * R), du(u), weights(T * K), ddw(dw), dl(T * R), logprob(T);
  Device<uint8_t> blocks(R * H / 2), scales(R * H / 32), packed(GpuMoeDispatcher::mxfp4_packed_size(R, H));
  Device<int32_t> idx(T * K), counts(R), tokens(T);
  const moe_routing rule{MOE_SCORE_SOFTMAX, 1, K, 0, 0, 0, 1.0f, nullptr};
  d.mxfp4_quantize_device(dweights.p, MOE_F32, R, H, blocks.p, scales.p);
  d.mxfp4_pack_device(blocks.p, scales.p, R, H, packed.p);
  d.mxfp4_matmul_device(packed.p, R, H, nullptr, dx.p, MOE_F32, nullptr, T, y.p, MOE_F32);
  d.route_device(rule, y.p, T, R, idx.p, weights.p, counts.p);
  d.route_backward_device(rule, y.p, idx.p, ddw.p, T, R, dl.p);
  d.sample_device(moe_sampling{}, y.p, R, du.p, T, R, tokens.p, logprob.p);
  d.synchronize();
  const float code[8] = {0, 0.5f, 1, 1.5f, 2, 3, 4, 6};
  const auto b = blocks.get(), s = scales.get();
  const auto logits = y.get(), weight = weights.get(), grad = dl.get(), lp = logprob.get();
  const auto expert = idx.get(), token = tokens.get(), count = counts.get();
  std::vector<double> q(R * H);
  for (size_t i = 0; i < R * H; i++) {
    const int c = b[i / 2] >> 4 * (i & 1) & 15;
    q[i] = std::ldexp((c & 8 ? -1.0 : 1.0) * code[c & 7], s[i / 32] - 127);
    // (codes of up to 6 have steps of up to 2, and values of up to 8 are cut to 6; the scale is an eighth to a quarter of the largest)
    double top = 0;
    for (size_t j = i / 32 * 32; j < i / 32 * 32 + 32; j++) top = std::max(top, (double)std::fabs(w[j]));
    EXPECT(std::fabs(q[i] - w[i]) <= top / 4 + 1e-12, "weight %zu: %g for %g", i, q[i], w[i]);
  }
  int32_t chosen = 0;
  for (int32_t c : count) chosen += c;
  EXPECT(chosen == (int32_t)(T * K), "counts add up to %d", chosen);
  for (size_t t = 0; t < T; t++) {
    double sum = 0, top = 0, mean = 0;
    for (size_t r = 0; r < R; r++) {
      double v = 0, mag = 0;
      for (size_t h = 0; h < H; h++) v += q[r * H + h] * x[t * H + h], mag += std::fabs(q[r * H + h] * x[t * H + h]);
      EXPECT(std::fabs(v - logits[t * R + r]) <= 1e-6 * mag, "logit %zu %zu: %g for %g", t, r, logits[t * R + r], v);
      sum += std::exp((double)logits[t * R + r]);
    }
    for (size_t j = 0; j < K; j++) {
      const float l = logits[t * R + expert[t * K + j]];
      size_t above = 0;
      for (size_t r = 0; r < R; r++) above += logits[t * R + r] > l;
      EXPECT(above == j, "expert %zu of token %zu has %zu above it", j, t, above);
      top += std::exp((double)l);
    }
    for (size_t j = 0; j < K; j++) {
      const double p = std::exp((double)logits[t * R + expert[t * K + j]]) / top;
      EXPECT(std::fabs(weight[t * K + j] - p) <= 1e-7, "weight %zu %zu", t, j);
      mean += p * dw[t * K + j];
    }
    for (size_t r = 0; r < R; r++) {
      double g = 0;
      for (size_t j = 0; j < K; j++)
        if (expert[t * K + j] == (int32_t)r) g = std::exp((double)logits[t * R + r]) / top * (dw[t * K + j] - mean);
      EXPECT(std::fabs(grad[t * R + r] - g) <= 1e-6, "gradient %zu %zu", t, r);
    }
    double run = 0;
    size_t at = 0;
    while ((run += std::exp((double)logits[t * R + at])) <= u[t] * sum) at++;
    EXPECT(token[t] == (int32_t)at, "token %zu: %d for %zu", t, token[t], at);
    EXPECT(std::fabs(lp[t] - (logits[t * R + at] - std::log(sum))) <= 1e-6, "probability of token %zu", t);
  }
  std::printf("gpu: %s\n", failures ? "FAILED" : "ok");
  return failures ? 1 : 0;
}

int main(int argc, char **argv) { return argc > 1 && !std::strcmp(argv[1], "gpu") ? run_gpu() : run_cpu(); }
