// The bounds of include/moe_serve.h's calls at the ends of what it allows, over the launches that serve_calls_test.cpp notes.
//   serve_bounds_test shift   a row's masses sum up within 64 bits, and have as many bits as that leaves
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

}  // namespace

int main(int argc, char **argv) {
  g_ctx.d.H = 32;
  g_ctx.d.work = &g_work;
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "shift")
    shift();
  else
    return 2;
  printf("wrong %d, faults %ld\n", wrong, g_faults);
  return wrong || g_faults ? 3 : 0;
}
