// The bounds of include/moe_serve.h's calls at the ends of what it allows, over the launches that serve_calls_test.cpp notes.
//   serve_bounds_test shift   a row's masses sum up within 64 bits, and have as many bits as that leaves
//   serve_bounds_test rows    rows of the widest vocabularies go in launches of less than 2^32 threads, each row once
//   serve_bounds_test terms   a product's workspace: fewer tokens at a time of above 65536 columns
//   serve_bounds_test alone   which products need no workspace, and so may be captured first
#define main serve_calls_main
#include "serve_calls_test.cpp"
#undef main

namespace {

int wrong;
void check(bool ok, const char *what, size_t a, size_t b = 0) {
  if (!ok && wrong++ < 20) printf("WRONG %s: %zu %zu\n", what, a, b);
}

void shift() {
  auto one = [](size_t V) {
    const int s = sample_shift(V);
    const unsigned __int128 all = (unsigned __int128)V << s;
    check(s >= 34 && s <= 44 && all <= (unsigned __int128)1 << 62, "a sum above 2^62", V, s);
    check(s == 44 || all * 2 > (unsigned __int128)1 << 62, "fewer bits than there are", V, s);
  };
  for (size_t V = 1; V < 3000; V++) one(V);
  for (int e = 12; e <= 28; e++)
    for (long off : {-3L, -2L, -1L, 0L, 1L, 2L, 3L, 100L})
      if (((size_t)1 << e) + off <= (size_t)1 << 28) one(((size_t)1 << e) + off);
  for (size_t V : {(size_t)201088, (size_t)1200000, (size_t)1300000, (size_t)1500000, ((size_t)1 << 28) - 1}) one(V);
  std::mt19937_64 rng(2);
  for (int i = 0; i < 100000; i++) one(1 + rng() % ((size_t)1 << 28));
}

void rows() {
  // (sizes whose logits no card holds: a bound of the call alone)
  for (size_t V : {(size_t)1, (size_t)8192, (size_t)201088, (size_t)1 << 23, (size_t)1 << 24, ((size_t)1 << 24) + 1, ((size_t)1 << 28) - 1, (size_t)1 << 28})
    for (size_t T : {(size_t)1, (size_t)255, (size_t)256, (size_t)257, (size_t)4096, (size_t)4097, (size_t)20000}) {
      const moe_sampling r{};
      int32_t *tokens = device<int32_t>(T * 4);
      if (moe_sample_device(&g_ctx, &r, device<float>(T * V * 4), V, device<float>(T * 4), T, V, tokens, nullptr, nullptr)) fault(g_error.c_str());
      for (auto &w : g_buffers[(uintptr_t)tokens].written) {
        const size_t n = (w.second - w.first) / 4, groups = (V + 8191) / 8192;
        check(n <= 4096 && groups * n * 512 < (size_t)1 << 32, "a launch's threads", V, n);
      }
      whole(tokens, T * 4);
      check(V > (size_t)1 << 23 || g_buffers[(uintptr_t)tokens].written.size() == (T + 4095) / 4096, "pieces of an ordinary call", V, T);
    }
}

void terms() {
  for (size_t cols : {(size_t)1 << 20, ((size_t)1 << 20) - 32, (size_t)100000, (size_t)65536 + 32, (size_t)65536, (size_t)2880})
    for (size_t T : {(size_t)65536, (size_t)65537, (size_t)40000, (size_t)5000})
      for (int type : {(int)MOE_F32, (int)MOE_BF16, (int)MOE_MXFP8, (int)MOE_MXFP4}) {
        const PackDims d = pack_dims(16, cols);
        void *y = buffer(T * 64);
        g_work = DenseWork{};
        if (moe_mxfp4_matmul_device(&g_ctx, device(pack_weight_bytes(d) + pack_scale_bytes(d)), 16, cols, nullptr, buffer(T * cols * 4), type,
                                    device(T * cols / 32), T, y, MOE_F32, nullptr))
          fault(g_error.c_str());
        whole(y, T * 64);
        size_t largest = 0;
        for (auto &w : g_buffers[(uintptr_t)y].written) largest = std::max(largest, (w.second - w.first) / 64);
        check(largest * cols <= (size_t)1 << 32 && largest <= 65536, "tokens at a time", cols, largest);
        check(cols > 65536 || largest == std::min<size_t>(T, 65536), "pieces of an ordinary call", cols, largest);
        check(g_work.cap < (size_t)20 << 30, "workspace", cols, g_work.cap);
      }
}

void alone() {
  g_capturing = true;
  auto one = [](int type, size_t T, size_t cols, bool none) {
    g_work = DenseWork{};
    const PackDims d = pack_dims(16, cols);
    void *y = buffer(T * 64);
    const int rc = moe_mxfp4_matmul_device(&g_ctx, device(pack_weight_bytes(d) + pack_scale_bytes(d)), 16, cols, nullptr, buffer(T * cols * 4), type,
                                           device(T * cols), T, y, MOE_F32, nullptr);
    check(rc == (none ? MOE_OK : MOE_ERR_STATE) && !g_work.p, "a product's workspace", T, cols);
    if (none) whole(y, T * 64);
  };
  one(MOE_F32, 1, 32, true), one(MOE_F32, 1, 10624, true), one(MOE_F32, 2, 5248, true);
  one(MOE_F32, 1, 10624 + 32, false), one(MOE_F32, 2, 5248 + 32, false), one(MOE_F32, 3, 32, false);
  // rows of 2 cols, rounded up to 256, and 16 bytes: 48 KB in all
  for (size_t T = 1; T <= 16; T++)
    for (size_t cols = 32; cols <= 32768; cols += 32) one(MOE_BF16, T, cols, T * ((2 * cols + 255) / 256 * 256 + 16) <= 48 * 1024);
  one(MOE_BF16, 17, 32, false);
  one(MOE_MXFP8, 1, 32, false), one(MOE_MXFP4, 1, 32, false);
  g_capturing = false;
}

}  // namespace

int main(int argc, char **argv) {
  g_ctx.d.H = 32;
  g_ctx.d.work = &g_work;
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "shift")
    shift();
  else if (what == "rows")
    rows();
  else if (what == "terms")
    terms();
  else if (what == "alone")
    alone();
  else
    return 2;
  printf("wrong %d, faults %ld\n", wrong, g_faults);
  return wrong || g_faults ? 3 : 0;
}
