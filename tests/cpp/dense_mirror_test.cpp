// The dense operators through the C++ mirror (silentotithrandousha_amd/host/gpu_moe_dispatcher.hpp): one training step of a
// block under the LM head, each result against plain loops in 64 bits.
//   dense_mirror_test cpu   what needs no device
//   dense_mirror_test gpu   the step
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
  EXPECT(GpuMoeDispatcher::act8_bytes(3, 64) == 3 * 64 + 3 * 2, "bytes of a checkpoint");
  EXPECT(GpuMoeDispatcher::act8_bytes(0, 64) == 0, "no rows");
  EXPECT(panics([] { GpuMoeDispatcher::act8_bytes(3, 33); }), "33 columns");
  EXPECT(panics([] { GpuMoeDispatcher::act8_bytes(3, 0); }), "no columns");
  GpuMoeDispatcher none;  // without a context every call is an error, not a crash
  EXPECT(panics([&] { none.act8_pack_device(nullptr, MOE_F32, 1, 32, nullptr); }), "pack");
  EXPECT(panics([&] { none.act8_unpack_device(nullptr, 1, 32, nullptr, MOE_F32); }), "unpack");
  EXPECT(panics([&] { none.lm_head_loss_device(nullptr, MOE_F32, nullptr, 1, 1, nullptr, nullptr); }), "loss");
  EXPECT(panics([&] { none.ffn_forward_device(moe_ffn{}, nullptr, MOE_F32, 1, nullptr); }), "block");
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

// sums of up to 300 products in f32, of three bf16 terms each, and a few functions: 2^-12 of the magnitudes
static void close(const char *what, const std::vector<float> &got, const std::vector<double> &want, const std::vector<double> &size) {
  for (size_t i = 0; i < got.size(); i++)
    if (!(std::fabs(got[i] - want[i]) <= size[i] / 4096)) {
      EXPECT(false, "%s[%zu]: %g against %g", what, i, got[i], want[i]);
      return;
    }
}

static int run_gpu() {
  const size_t T = 5, H = 64, I = 40, V = 300;
  const double C = 7.0;
  std::mt19937 rng(1);
  std::normal_distribution<float> normal;
  auto values = [&](size_t n, float scale) {
    std::vector<float> v(n);
    for (float &x : v) x = normal(rng) * scale;
    return v;
  };
  auto weights = [&](size_t n, float scale, std::vector<double> &exact) {
    std::vector<uint16_t> w(n);
    exact.resize(n);
    for (size_t i = 0; i < n; i++) {
      const float f = normal(rng) * scale;
      uint32_t u;
      std::memcpy(&u, &f, 4);
      u &= 0xFFFF0000u;
      w[i] = (uint16_t)(u >> 16);
      float r;
      std::memcpy(&r, &u, 4);
      exact[i] = r;
    }
    return w;
  };
  std::vector<double> wgu, wd, wl;
  Device<uint16_t> gate_up(weights(2 * I * H, 0.15f, wgu)), down(weights(H * I, 0.15f, wd)), head(weights(V * H, 0.2f, wl));
  const auto xh = values(T * H, 1.0f), bg = values(2 * I, 0.1f), bd = values(H, 0.1f);
  Device<float> x(xh), bias(bg), bias_down(bd), y(T * H), loss(T), lse(T), dy(T * H), dw(V * H), dloss(std::vector<float>(T, 1.0f / T)), back(T * H);
  Device<float> dx(T * H), dgu(2 * I * H), dbg(2 * I), dd(H * I), dbd(H);
  std::vector<int32_t> targets{3, -1, 299, 0, 150};
  Device<int32_t> t(targets);
  auto d = GpuMoeDispatcher::create(H, 32, (float)C).unwrap();
  Device<uint8_t> kept(GpuMoeDispatcher::act8_bytes(T, H)), again(GpuMoeDispatcher::act8_bytes(T, H));
  const moe_ffn block{I, gate_up.p, bias.p, down.p, bias_down.p};
  d.init_lm_head_bf16_device(head.p, V);
  d.ffn_forward_device(block, x.p, MOE_F32, T, y.p, kept.p);
  d.lm_head_loss_device(y.p, MOE_F32, t.p, T, V, loss.p, lse.p);
  d.lm_head_loss_backward_device(y.p, MOE_F32, t.p, lse.p, dloss.p, T, V, dy.p, dw.p);
  d.ffn_backward_device(block, kept.p, MOE_MXFP8, dy.p, MOE_F32, T, moe_ffn_grads{dx.p, dgu.p, dbg.p, dd.p, dbd.p});
  d.act8_pack_device(x.p, MOE_F32, T, H, again.p);
  d.act8_unpack_device(again.p, T, H, back.p, MOE_F32);
  d.synchronize();
  EXPECT(kept.get() == again.get(), "the forward pass's checkpoint is the packed rows");
  const auto x8 = back.get();
  for (size_t i = 0; i < T * H; i++) EXPECT(std::fabs(x8[i] - xh[i]) <= std::fabs(xh[i]) / 16 + 0.01, "a checkpoint's value %zu", i);

  // h of rows, and the block's result
  auto hidden = [&](const std::vector<float> &rows, std::vector<double> &g, std::vector<double> &u) {
    std::vector<double> h(T * I);
    g.assign(T * I, 0), u.assign(T * I, 0);
    for (size_t r = 0; r < T; r++)
      for (size_t i = 0; i < I; i++) {
        double a = bg[2 * i], b = bg[2 * i + 1];
        for (size_t k = 0; k < H; k++) a += rows[r * H + k] * wgu[2 * i * H + k], b += rows[r * H + k] * wgu[(2 * i + 1) * H + k];
        g[r * I + i] = a, u[r * I + i] = b;
        const double G = std::fmin(a, C), U = std::fmax(std::fmin(b, C), -C);
        h[r * I + i] = (U + 1) * G / (1 + std::exp(-1.702 * G));
      }
    return h;
  };
  std::vector<double> g, u;
  const auto h = hidden(xh, g, u);
  std::vector<double> want(T * H), size(T * H);
  for (size_t r = 0; r < T; r++)
    for (size_t k = 0; k < H; k++) {
      double v = bd[k], m = std::fabs(v) + 1;
      for (size_t i = 0; i < I; i++) v += h[r * I + i] * wd[k * I + i], m += std::fabs(h[r * I + i] * wd[k * I + i]);
      want[r * H + k] = v, size[r * H + k] = m;
    }
  close("y", y.get(), want, size);

  // loss and its gradient of the rows that the block returned
  const auto yr = y.get();
  std::vector<double> wl_loss(T), one(T, 16.0), wdy(T * H), sdy(T * H, 1e-3);
  for (size_t r = 0; r < T; r++) {
    std::vector<double> l(V);
    double sum = 0;
    for (size_t v = 0; v < V; v++) {
      for (size_t k = 0; k < H; k++) l[v] += yr[r * H + k] * wl[v * H + k];
      sum += std::exp(l[v]);
    }
    wl_loss[r] = targets[r] < 0 ? 0 : std::log(sum) - l[targets[r]];
    for (size_t v = 0; v < V && targets[r] >= 0; v++) {
      const double p = (std::exp(l[v]) / sum - (v == (size_t)targets[r])) / T;
      for (size_t k = 0; k < H; k++) wdy[r * H + k] += p * wl[v * H + k], sdy[r * H + k] += std::fabs(p * wl[v * H + k]);
    }
  }
  close("loss", loss.get(), wl_loss, one);
  close("dy", dy.get(), wdy, sdy);

  // the bias gradients and dx at the checkpoint's values
  const auto dyr = dy.get();
  hidden(x8, g, u);
  std::vector<double> wb(H), sb(H, 1e-3), wg(2 * I), sg(2 * I, 1e-3), wdx(T * H), sdx(T * H, 1e-3);
  for (size_t r = 0; r < T; r++)
    for (size_t k = 0; k < H; k++) wb[k] += dyr[r * H + k], sb[k] += std::fabs(dyr[r * H + k]);
  for (size_t r = 0; r < T; r++)
    for (size_t i = 0; i < I; i++) {
      double dh = 0, mh = 0;
      for (size_t k = 0; k < H; k++) dh += dyr[r * H + k] * wd[k * I + i], mh += std::fabs(dyr[r * H + k] * wd[k * I + i]);
      const double a = g[r * I + i], b = u[r * I + i], G = std::fmin(a, C), U = std::fmax(std::fmin(b, C), -C), s = 1 / (1 + std::exp(-1.702 * G));
      const double da = a > C ? 0 : dh * (U + 1) * s * (1 + 1.702 * G * (1 - s)), db = std::fabs(b) > C ? 0 : dh * G * s;
      const double m = mh * (std::fabs(U) + 1) * (std::fabs(G) + 1);
      wg[2 * i] += da, wg[2 * i + 1] += db, sg[2 * i] += m, sg[2 * i + 1] += m;
      for (size_t k = 0; k < H; k++) {
        wdx[r * H + k] += da * wgu[2 * i * H + k] + db * wgu[(2 * i + 1) * H + k];
        sdx[r * H + k] += m * (std::fabs(wgu[2 * i * H + k]) + std::fabs(wgu[(2 * i + 1) * H + k]));
      }
    }
  close("down_bias", dbd.get(), wb, sb);
  close("gate_up_bias", dbg.get(), wg, sg);
  close("dx", dx.get(), wdx, sdx);
  EXPECT(panics([&] { d.act8_pack_device(x.p, MOE_MXFP8, T, H, again.p); }), "a checkpoint of a checkpoint");
  std::printf("gpu: %s\n", failures ? "FAILED" : "ok");
  return failures ? 1 : 0;
}

int main(int argc, char **argv) {
  try {
    return argc > 1 && std::string(argv[1]) == "gpu" ? run_gpu() : run_cpu();
  } catch (const std::exception &e) {
    std::printf("exception: %s\n", e.what());
    return 2;
  }
}
