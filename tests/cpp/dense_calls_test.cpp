// The calls of include/moe_dense.h replayed on the host: csrc/dense_api.cpp and dense_plan.cpp as they are, over launches
// and allocations that only note what they would read and write. Of every launch it is checked that
//   * what it reads and writes lies in the caller's buffers or in the workspace, and what it writes is not what it reads;
//   * what it reads of the workspace, an earlier launch of the same call wrote;
//   * the slots of f32 rows hold the planes that the product takes them for, with infinities where they may be.
// The form of every launch (tile, layout, planes, K parts, ...) is printed, so that a test can tell which of them its
// sizes take.
//   dense_calls_test calls [BYTES] < lines   a line a call: its forms; no workspace may be above BYTES
//   dense_calls_test refusals           calls that must be refused before anything is launched
//   dense_calls_test growth             the workspace over calls of rising lengths
//   dense_calls_test draw N SEED        the forms of N drawn calls, each with the cheapest call that takes it
//   dense_calls_test plant WHAT < lines the same as `calls` with a mistake: must find it
//   dense_calls_test checks             products that the kernels could not store in their pieces: each must be refused
// Lines: "loss T H V dtype", "lossgrad T H V dtype dx dw", "ffn T H I dtype x8", "ffngrad T H I dtype kept mask" (mask: bits
// of the gradients of x, gate_up, gate_up_bias, down, down_bias).
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <iostream>
#include <iterator>
#include <map>
#include <random>
#include <set>
#include <sstream>
#include <string>
#include <vector>

#include "../../include/moe_dense.h"
#include "../../silentotithrandousha_amd/csrc/dense_plan.hpp"

using namespace moe;

struct moe_ctx {
  DenseCtx d;
};

namespace {

std::string g_plant;
std::string g_error;  // what moe_last_error would say
long g_faults;

void fault(const char *what) {
  if (g_faults++ < 20) printf("FAULT %s\n", what);
}

// ---- memory: buffers of the caller and the workspace, what was written, the planes that slots hold
struct Buffer {
  uintptr_t at;
  size_t bytes;
  bool work;
};
std::vector<Buffer> g_buffers;
std::vector<std::pair<uintptr_t, uintptr_t>> g_written;  // intervals of the workspace, merged
struct Slot {
  size_t bytes;
  int plane;  // -1: a value itself
  bool infinite;  // it holds infinities
};
std::map<uintptr_t, Slot> g_slots;
uintptr_t g_next = (uintptr_t)1 << 40;

uintptr_t buffer(size_t bytes, bool work = false) {
  const uintptr_t at = g_next;
  g_next += (bytes + 0x1FFFFF) & ~(uintptr_t)0xFFFFF;
  g_buffers.push_back({at, bytes, work});
  return at;
}
const Buffer *holding(uintptr_t at, size_t bytes) {
  for (const Buffer &b : g_buffers)
    if (at >= b.at && at + bytes <= b.at + b.bytes) return &b;
  return nullptr;
}
struct Range {
  uintptr_t at;
  size_t bytes;
};
std::vector<Range> g_reads, g_writes;  // of the launch under way

void read(const void *p, size_t bytes) {
  const uintptr_t at = (uintptr_t)p;
  const Buffer *b = holding(at, bytes);
  if (!b) return fault("a read outside the buffers");
  g_reads.push_back({at, bytes});
  if (!b->work) return;
  for (auto &w : g_written)
    if (at >= w.first && at + bytes <= w.second) return;
  fault("a read of workspace that nothing wrote");
}
void write(const void *p, size_t bytes) {
  const uintptr_t at = (uintptr_t)p;
  if (!holding(at, bytes)) return fault("a write outside the buffers");
  g_writes.push_back({at, bytes});
}
// rows of a matrix: n rows of `cols` elements, `ld` between them
size_t extent(size_t n, size_t cols, size_t ld, size_t el) { return ((n - 1) * ld + cols) * el; }
size_t up8(size_t v) { return (v + 7) / 8 * 8; }

long g_launches;

void launched() {
  g_launches++;
  for (const Range &w : g_writes) {
    for (const Range &r : g_reads)
      if (w.at < r.at + r.bytes && r.at < w.at + w.bytes) fault("a launch writes what it reads");
    for (const Range &v : g_writes)
      if (&v != &w && w.at < v.at + v.bytes && v.at < w.at + w.bytes) fault("a launch writes twice to a place");
  }
  for (const Range &w : g_writes) {
    uintptr_t lo = w.at, hi = w.at + w.bytes;
    std::vector<std::pair<uintptr_t, uintptr_t>> keep;
    for (auto &v : g_written) {
      if (v.second < lo || v.first > hi)
        keep.push_back(v);
      else
        lo = std::min(lo, v.first), hi = std::max(hi, v.second);
    }
    keep.push_back({lo, hi});
    g_written = keep;
  }
  g_reads.clear(), g_writes.clear();
}

// values in planes, in slots of `bytes`
void write_slots(void *out, uint32_t where, int planes, size_t bytes) {
  for (int p = 0; p < planes; p++)
    for (uint32_t m = where >> 8 * p & 255, all = m; m; m &= m - 1) {
      const int s = __builtin_ctz(m);
      char *at = (char *)out + (size_t)s * bytes;
      write(at, bytes);
      g_slots[(uintptr_t)at] = {bytes, planes == 1 ? -1 : p, planes == 1 || (p == 0 && (all >> s) == 1)};
    }
}
const Slot *slot_at(const void *p, size_t bytes) {
  auto it = g_slots.find((uintptr_t)p);
  return it != g_slots.end() && it->second.bytes >= bytes ? &it->second : nullptr;
}

// a launch counts its threads in 32 bits
void grid(size_t tiles, const DenseTileDims &d) {
  if (tiles * 64 * d.wm * d.wn >> 32) fault("a grid of more threads than a launch has");
}

// ---- forms
std::set<std::string> g_forms;
void form(const std::string &s) { g_forms.insert(s); }
const char *epi_name(DenseEpi e) {
  const char *n[] = {"store", "gate", "dgate", "stats", "dlogits"};
  return n[e];
}

// B as a product reads it: its planes, lowest first, one of them with the infinities
void read_b(const DenseShape &s, const DenseArgs &a) {
  const size_t rows = s.bt ? (size_t)a.K : (size_t)a.N, cols = s.bt ? up8(a.N) : up8(a.K);
  const size_t one = extent(rows, cols, a.ldb, 2);
  if (a.stack > 1) {
    std::set<int> planes;
    for (int i = 0; i < a.stack; i++) {
      const uint16_t *p = a.B + (size_t)i * a.stack_step * a.b_slot;
      read(p, one);
      const Slot *t = slot_at(p, one);
      if (!t || t->plane < 0 || t->infinite != (t->plane == 0)) {
        fault("a stacked slot that is no plane, or not the last of its plane");
        continue;
      }
      planes.insert(t->plane);
      if (i == a.stack - 1 && t->plane != 0) fault("the first plane is not the last row of the stack");
    }
    if (planes.size() != (size_t)kPlanes) fault("the stack does not hold every plane");
    if (a.b_slot != rows * a.ldb) fault("stacked slots whose rows do not follow each other");
    return;
  }
  if (a.b_planes > 1) {
    for (int i = 0; i < a.b_planes; i++) {
      const uint16_t *p = a.B + (size_t)(a.pb >> 4 * i & 15) * a.b_slot;
      read(p, one);
      const Slot *t = slot_at(p, one);
      if (!t || t->plane != kPlanes - 1 - i || t->infinite != (t->plane == 0)) fault("a slot that does not hold the plane it is taken for");
    }
    return;
  }
  read(a.B, one);
}

// the pairs of a gradient's slots
void read_gradient(const DenseArgs &a) {
  const size_t A = extent(a.K, up8(a.M), a.lda, 2), B = extent(a.K, up8(a.N), a.ldb, 2);
  read(a.A, A);
  read(a.B, B);
  const Slot *x = slot_at(a.A, 0), *y = slot_at(a.B, 0);
  if (!y || y->plane < 0) return;  // rows of one plane (a caller's, or copies without planes)
  std::multiset<std::pair<int, int>> pairs;
  const char *pa = (const char *)a.A, *pb = (const char *)a.B;
  size_t k = 0;
  while (k < (size_t)a.K) {
    x = slot_at(pa, 0), y = slot_at(pb, 0);
    if (!x || !y || x->bytes / (a.lda * 2) != y->bytes / (a.ldb * 2)) return fault("a gradient over slots of different rows");
    pairs.insert({x->plane, y->plane});
    if (x->plane >= 0 && (x->infinite || y->infinite) && !(x->infinite && y->infinite)) fault("an infinity meets a lower plane");
    k += x->bytes / (a.lda * 2);
    pa += x->bytes, pb += y->bytes;
  }
  const std::multiset<std::pair<int, int>> six{{0, 0}, {0, 1}, {1, 0}, {1, 1}, {0, 2}, {2, 0}}, copies{{-1, 0}, {-1, 1}, {-1, 2}};
  if (k != (size_t)a.K || (pairs != six && pairs != copies)) fault("a gradient whose pairs of planes are not those above 2^-24");
}

void note(const DenseShape &s, DenseArgs a) {
  if (s.bt) {
    read_gradient(a);
  } else {
    const size_t rows = s.at ? (size_t)a.K : (size_t)a.M, cols = s.at ? up8(a.M) : up8(a.K);
    read(a.A, extent(rows, cols, a.lda, 2));
    read_b(s, a);
  }
  if (a.bias) read(a.bias, (size_t)a.M * 4);
  const bool planes = a.b_planes > 1 || a.stack > 1;
  const size_t N = a.N, M = a.M;
  switch (s.epi) {
    case DENSE_STORE:
      if (a.scale) read(a.scale, 4);
      for (int p = 0; p < a.splits; p++) {
        const size_t el = a.out_mode ? 4 : 2, bytes = extent(N, M, a.ldo, el);
        write((char *)a.out + (size_t)p * a.split_stride * 4, bytes);
      }
      break;
    case DENSE_GATE:
      if ((a.planes > 1) != planes) fault("planes of the result beside rows of one");
      write_slots(a.h, a.h_where, a.planes, N * a.ldh * 2);
      if (a.h_slot != N * a.ldh && a.planes > 1) fault("slots of h that leave room");
      break;
    case DENSE_DGATE:
      read(a.gu, N * 2 * M * 4);
      write_slots(a.h, a.h_where, a.planes, N * a.ldh * 2);
      write_slots(a.dgu, a.dgu_where, a.planes, N * 2 * M * 2);
      if (a.db_part) write(a.db_part, (size_t)dense_parts(s, a) * 2 * M * 4);
      break;
    case DENSE_STATS:
      read(a.targets, N * 4);
      write(a.stats, (size_t)dense_parts(s, a) * N * 8);
      write(a.picked, N * 4);
      break;
    case DENSE_DLOGITS:
      read(a.targets, N * 4), read(a.lse, N * 4), read(a.dloss, N * 4), read(a.scale, 4);
      // (the columns past the piece's own up to the next 8 are written as zeros; the others are not read)
      if (up8(M) > a.ld_dl) fault("no room for the padding columns");
      write_slots(a.dl, a.dl_where, a.planes, N * a.ld_dl * 2);
      break;
  }
}

}  // namespace

// ---- what dense_api.cpp calls
namespace moe {
int api_fail(int code, const char *msg) {
  g_error = msg;
  return code;
}
int dense_ctx(moe_ctx *c, DenseCtx *d) {
  if (!c) return api_fail(MOE_ERR_INVALID, "null context");
  *d = c->d;
  return MOE_OK;
}

hipError_t launch_dense(const DenseShape &s, const DenseArgs &a0, hipStream_t) {
  DenseArgs a = a0;
  if (g_plant == "slot" && a.b_planes > 1) a.pb = 0x210;
  if (g_plant == "behind" && s.epi == DENSE_STORE) a.ldo += 8;
  const hipError_t e = dense_prepare(s, a);
  if (e != hipSuccess) return fault("a product that is refused"), e;
  note(s, a);
  std::ostringstream o;
  const char *out = s.epi != DENSE_STORE ? "" : a.out_mode == 0 ? ".bf16" : a.out_mode == 1 ? ".f32" : ".add";
  const char *rows = a.stack > 1 ? ".stacked" : a.b_planes > 1 ? ".planes" : "";
  if (const int few = dense_few_rows(s, a)) {
    o << "few" << few << "." << epi_name(s.epi) << out << rows;
  } else {
    const DenseTileDims &d = kDenseTiles[dense_tile(s, a)];
    grid((size_t)((a.M + d.bm - 1) / d.bm) * (((size_t)a.N * a.stack + d.bn - 1) / d.bn), d);
    o << epi_name(s.epi) << (s.at ? (s.bt ? ".tt" : ".tn") : ".nt") << "." << d.bm << "x" << d.bn << out << rows << (a.splits > 1 ? ".parts" : "");
  }
  form(o.str());
  launched();
  return hipSuccess;
}
hipError_t launch_dense_pair(const DenseArgs &a0, const DenseArgs &b0, hipStream_t) {
  DenseArgs a = a0, b = b0;
  const hipError_t e = dense_prepare_pair(a, b);
  if (e != hipSuccess) return fault("a pair that is refused"), e;
  const DenseShape s{true, true, DENSE_STORE};
  note(s, a);
  note(s, b);
  double us;
  const DenseTileDims &d = kDenseTiles[dense_pair_tile(a, b, us)];
  size_t tiles = 0;
  for (const DenseArgs *x : {&a, &b}) tiles += (size_t)((x->M + d.bm - 1) / d.bm) * ((x->N + d.bn - 1) / d.bn);
  grid(tiles, d);
  form("pair." + std::to_string(d.bm) + "x" + std::to_string(d.bn) + (a.out_mode ? ".f32" : ".bf16"));
  launched();
  return hipSuccess;
}
hipError_t launch_dgate(const DgateArgs &a, hipStream_t) {
  const size_t n = (size_t)a.T * a.I;
  read(a.gu, n * 2 * a.gu_parts * 4), read(a.dh, n * a.dh_parts * 4);
  if (a.bias) read(a.bias, (size_t)2 * a.I * 4);
  write_slots(a.h, a.h_where, a.planes, n * 2);
  write_slots(a.dgu, a.dgu_where, a.planes, n * 4);
  if (a.db_part) write(a.db_part, (size_t)dense_dgate_parts(a.T) * 2 * a.I * 4);
  form(std::string("joined") + (a.planes > 1 ? ".planes" : ""));
  launched();
  return hipSuccess;
}
static void note_scale(const DlossScale &d) { read(d.dloss, d.T * 4), read(d.targets, d.T * 4), write(d.scale, 4); }
hipError_t launch_dloss_scale(const DlossScale &d, hipStream_t) {
  note_scale(d);
  form("scale");
  launched();
  return hipSuccess;
}
hipError_t launch_rows(DenseRowJobs a, hipStream_t) {
  const char *names[] = {"planes", "copy", "pack8", "unpack8", "sum_bf16", "sum_f32", "scale"};
  a.ends();
  if (a.count > (int)(sizeof(a.d) / sizeof(a.d[0]))) fault("more jobs than a launch has room for");
  for (int i = 0; i < a.count; i++) {
    const DenseRows &d = a.d[i];
    form(std::string("rows.") + names[d.what] + (d.targets ? ".masked" : ""));
    if (d.targets) read(d.targets, d.n / d.cols * 4);
    switch (d.what) {
      case ROWS_PLANES: read(d.x, d.n * 4), write_slots(d.out, d.where, kPlanes, d.n * 2); break;
      case ROWS_COPY: read(d.x, d.n * 2), write_slots(d.out, kWhereOne, 1, d.n * 2); break;
      case ROWS_PACK8: read(d.x, d.n * 4), write(d.out, d.n + d.n / 32); break;
      case ROWS_UNPACK8:
        read(d.x, d.n + d.n / 32);
        for (int c = 0; c < d.copies; c++) write_slots((uint16_t *)d.out + c * d.n, kWhereOne, 1, d.n * 2);
        break;
      case ROWS_SUM_BF16: read(d.x, d.n * d.cols * 2), write(d.out, d.cols * 4); break;
      case ROWS_SUM_F32: read(d.x, d.n * d.cols * 4), write(d.out, d.cols * 4); break;
      case ROWS_DLOSS_SCALE: note_scale(a.scale); break;
    }
  }
  launched();
  return hipSuccess;
}
hipError_t launch_sums(DenseSums a, hipStream_t) {
  a.ends();
  if (a.count > (int)(sizeof(a.d) / sizeof(a.d[0]))) fault("more sums than a launch has room for");
  for (int i = 0; i < a.count; i++) {
    const DenseSum &d = a.d[i];
    form(std::string("sums") + (d.bf16 ? ".bf16" : ".f32") + (d.few ? ".few" : "") + (d.bias ? ".bias" : ""));
    for (int p = 0; p < d.parts; p++) read(d.part + (size_t)p * d.stride, d.n * 4);
    if (d.bias) read(d.bias, d.n_bias * 4);
    write(d.out, d.n * (d.bf16 ? 2 : 4));
  }
  launched();
  return hipSuccess;
}
hipError_t launch_colsum(const void *x, bool bf16, size_t T, size_t H, float *part, hipStream_t) {
  read(x, T * H * (bf16 ? 2 : 4));
  write(part, dense_colsum_parts(T) * H * 4);
  form(bf16 ? "colsum.bf16" : "colsum.f32");
  launched();
  return hipSuccess;
}
hipError_t launch_loss(const float2 *stats, int parts, const float *picked, const int32_t *targets, size_t T, int, float *loss, float *lse, hipStream_t) {
  read(stats, (size_t)parts * T * 8), read(picked, T * 4), read(targets, T * 4), write(loss, T * 4), write(lse, T * 4);
  form(T >= 1024 ? "loss.16" : T >= 64 ? "loss.4" : "loss.1");
  launched();
  return hipSuccess;
}
hipError_t launch_act8_pack(const void *x, bool bf16, size_t n, size_t cols, uint8_t *packed, hipStream_t) {
  read(x, n * cols * (bf16 ? 2 : 4)), write(packed, n * cols + n * cols / 32);
  launched();
  return hipSuccess;
}
hipError_t launch_act8_unpack(const uint8_t *, size_t, size_t, void *, bool, hipStream_t) { return hipSuccess; }
hipError_t launch_zero(void *p, size_t bytes, hipStream_t) {
  write(p, bytes);
  launched();
  return hipSuccess;
}
}  // namespace moe

static bool g_capturing;
static size_t g_allocations, g_frees, g_most = ~(size_t)0, g_memory = ~(size_t)0;
extern "C" {
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
  *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t bytes) {
  if (bytes > g_memory) return hipErrorOutOfMemory;
  if (bytes > g_most) fault("a workspace above the bound");
  *p = (void *)buffer(g_plant == "short" ? bytes - 4096 : bytes, true);
  g_allocations++;
  return hipSuccess;
}
hipError_t hipFree(void *p) {
  g_frees++;
  for (auto b = g_buffers.begin(); b != g_buffers.end(); ++b)
    if (b->at == (uintptr_t)p) return g_buffers.erase(b), hipSuccess;
  fault("a free of what is not allocated");
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "error"; }
}

namespace {

struct Call {
  std::string op;
  size_t T, H, X;  // X: vocabulary or inner size
  int dtype, a, b;
  std::string text() const {
    std::ostringstream o;
    o << op << " " << T << " " << H << " " << X << " " << dtype;
    if (op == "lossgrad" || op == "ffngrad")
      o << " " << a << " " << b;
    else if (op == "ffn")
      o << " " << a;
    return o.str();
  }
  // about what it costs to check against 64 bits
  double cost() const { return 1e4 + (double)T * H * X + 30.0 * ((double)T * X + (double)H * X + (double)T * H); }
};

bool run(const Call &c) {
  g_buffers.clear(), g_written.clear(), g_slots.clear(), g_reads.clear(), g_writes.clear();
  g_next = (uintptr_t)1 << 40;
  DenseWork work;
  moe_ctx ctx{};
  const size_t el = c.dtype == MOE_F32 ? 4 : 2, T = c.T, H = c.H, X = c.X;
  ctx.d = DenseCtx{nullptr, H, 7.0f, nullptr, 0, &work};
  auto b = [](size_t bytes) { return (char *)buffer(bytes); };
  int rc;
  if (c.op == "loss" || c.op == "lossgrad") {
    ctx.d.lm_w = (const uint16_t *)b(X * H * 2);
    ctx.d.lm_vocab = X;
    void *x = b(T * H * el);
    int32_t *targets = (int32_t *)b(T * 4);
    float *loss = (float *)b(T * 4), *lse = (float *)b(T * 4);
    if (c.op == "loss")
      rc = moe_lm_head_loss_device(&ctx, x, c.dtype, targets, T, X, loss, lse, nullptr);
    else
      rc = moe_lm_head_loss_backward_device(&ctx, x, c.dtype, targets, lse, loss, T, X, c.a ? b(T * H * el) : nullptr, c.b ? b(X * H * el) : nullptr, nullptr);
  } else {
    const size_t kept = T * H + T * H / 32;
    moe_ffn block{X, (uint16_t *)b(2 * X * H * 2), (float *)b(2 * X * 4), (uint16_t *)b(X * H * 2), (float *)b(H * 4)};
    if (c.op == "ffn") {
      void *x = b(T * H * el), *y = b(T * H * el);
      rc = moe_ffn_forward_device(&ctx, &block, x, c.dtype, T, y, c.a ? (uint8_t *)b(kept) : nullptr, nullptr);
    } else {
      void *x = b(c.a ? kept : T * H * el), *dy = b(T * H * el);
      const int m = c.b;
      moe_ffn_grads g{m & 1 ? b(T * H * el) : nullptr, m & 2 ? b(2 * X * H * el) : nullptr, m & 4 ? (float *)b(2 * X * 4) : nullptr,
                      m & 8 ? b(X * H * el) : nullptr, m & 16 ? (float *)b(H * 4) : nullptr};
      rc = moe_ffn_backward_device(&ctx, &block, x, c.a ? (int)MOE_MXFP8 : c.dtype, dy, c.dtype, T, &g, nullptr);
    }
  }
  if (rc != MOE_OK) printf("refused: %s\n", g_error.c_str());
  return rc == MOE_OK;
}

bool parse(const std::string &line, Call &c) {
  std::istringstream in(line);
  c.a = c.b = 0;
  if (!(in >> c.op >> c.T >> c.H >> c.X >> c.dtype)) return false;
  in >> c.a >> c.b;
  return true;
}

}  // namespace

int main(int argc, char **argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  if (what == "calls" || what == "plant") {
    if (what == "calls" && argc > 2) g_most = strtoull(argv[2], nullptr, 10);
    if (what == "plant") g_plant = argv[2];
    std::string line;
    Call c;
    bool fine = true;
    while (std::getline(std::cin, line)) {
      if (!parse(line, c)) continue;
      g_forms.clear();
      const long before = g_faults;
      fine = run(c) && fine;
      printf("%s :", c.text().c_str());
      for (auto &f : g_forms) printf(" %s", f.c_str());
      printf(g_faults > before ? " FAULTS\n" : "\n");
    }
    printf("faults %ld\n", g_faults);
    return g_faults ? 3 : fine ? 0 : 4;
  }
  if (what == "checks") {
    // a product that is taken, and what makes it one that is not
    auto product = [](DenseEpi epi, size_t M) {
      DenseArgs a{};
      a.M = (int)M, a.N = 40, a.K = 64, a.lda = up8(M) + 64, a.ldb = 64;
      a.splits = a.stack = a.stack_step = a.b_planes = a.planes = 1;
      a.ldo = a.ldh = a.ld_dl = up8(M);
      if (epi == DENSE_GATE) a.ldh = up8(M / 2);
      return a;
    };
    int wrong = 0, n = 0;
    auto expect = [&](const char *what, DenseEpi epi, DenseArgs a, bool taken) {
      n++;
      if ((dense_prepare(DenseShape{false, false, epi}, a) == hipSuccess) != taken) wrong++, printf("%s: %s\n", what, taken ? "refused" : "taken");
    };
    for (size_t M : {4, 8, 12, 16, 20, 24, 32, 36, 60, 64}) {
      DenseArgs a = product(DENSE_STORE, M);
      expect("bf16 results in pieces of 8", DENSE_STORE, a, M % 8 == 0);
      a.ldo = M + 4;
      expect("bf16 rows that are not 16 bytes apart", DENSE_STORE, a, M % 8 == 0 && a.ldo % 8 == 0);
      for (int mode : {1, 2}) {
        a = product(DENSE_STORE, M);
        a.out_mode = mode;
        expect("f32 results in pieces of 4", DENSE_STORE, a, true);
        a.M += 2;
        expect("f32 results of 2 more", DENSE_STORE, a, false);
        a.M -= 2, a.ldo += 2;
        expect("f32 rows that are not 16 bytes apart", DENSE_STORE, a, false);
      }
      expect("h in pieces of 8", DENSE_GATE, product(DENSE_GATE, M), M % 16 == 0);
      a = product(DENSE_GATE, 32);
      a.ldh += 4;
      expect("rows of h that are not 16 bytes apart", DENSE_GATE, a, false);
      expect("d(gate, up) in pieces of 4", DENSE_DGATE, product(DENSE_DGATE, M), true);
      expect("d(gate, up) of 1 more", DENSE_DGATE, product(DENSE_DGATE, M + 1), false);
      expect("dlogits", DENSE_DLOGITS, product(DENSE_DLOGITS, M + 1), true);
      a = product(DENSE_DLOGITS, M);
      a.ld_dl += 4;
      expect("rows of dlogits that are not 16 bytes apart", DENSE_DLOGITS, a, false);
      a = product(DENSE_DLOGITS, M);
      a.ld_dl -= 8;
      expect("rows of dlogits without room for the padding", DENSE_DLOGITS, a, false);
      expect("logits", DENSE_STATS, product(DENSE_STATS, M + 1), true);
      DenseArgs x = product(DENSE_STORE, M), y = product(DENSE_STORE, 64);
      n++;
      if ((dense_prepare_pair(x, y) == hipSuccess) != (M % 8 == 0)) wrong++, printf("a pair of %zu rows\n", M);
      x = product(DENSE_STORE, 64), y = product(DENSE_STORE, M);
      if ((dense_prepare_pair(x, y) == hipSuccess) != (M % 8 == 0)) wrong++, printf("a pair of %zu rows\n", M);
    }
    printf("checks %d wrong %d\n", n, wrong);
    return wrong ? 3 : 0;
  }
  if (what == "refusals") {
    DenseWork work;
    moe_ctx ctx{};
    const size_t T = 4, H = 64, V = 40, I = 24;
    ctx.d = DenseCtx{nullptr, H, 7.0f, (const uint16_t *)buffer(V * H * 2), V, &work};
    char *x = (char *)buffer(4096), *y = (char *)buffer(4096), *t = (char *)buffer(64), *a = (char *)buffer(64), *b = (char *)buffer(64),
         *dw = (char *)buffer(V * H * 4), *w = (char *)buffer(1 << 16);
    int wrong = 0, n = 0;
    auto expect = [&](const char *what, int rc, int code = MOE_ERR_INVALID) {
      n++;
      if (rc != code || g_launches) wrong++, printf("%s: %d, %ld launches\n", what, rc, g_launches);
      g_launches = 0;
    };
    auto loss = [&](void *x, void *t, void *a, void *b, size_t V = 40) {
      return moe_lm_head_loss_device(&ctx, x, MOE_F32, (const int32_t *)t, T, V, (float *)a, (float *)b, nullptr);
    };
    auto grad = [&](void *x, void *t, void *lse, void *dloss, void *dx, void *dw, size_t V = 40) {
      return moe_lm_head_loss_backward_device(&ctx, x, MOE_F32, (const int32_t *)t, (const float *)lse, (const float *)dloss, T, V, dx, dw, nullptr);
    };
    for (int off : {1, 2, 3}) {
      expect("targets off", loss(x, t + off, a, b));
      expect("loss off", loss(x, t, a + off, b));
      expect("lse off", loss(x, t, a, b + off));
      expect("targets off", grad(x, t + off, a, b, y, dw));
      expect("lse off", grad(x, t, a + off, b, y, dw));
      expect("dloss off", grad(x, t, a, b + off, y, dw));
    }
    for (int off : {2, 4, 8}) {
      expect("x off", loss(x + off, t, a, b));
      expect("x off", grad(x + off, t, a, b, y, dw));
      expect("dx off", grad(x, t, a, b, y + off, dw));
      expect("dw off", grad(x, t, a, b, y, dw + off));
    }
    ctx.d.lm_vocab = (size_t)1 << 29;
    expect("a head of 2^28 rows and one", loss(x, t, a, b, ((size_t)1 << 28) + 1));
    expect("a head of 2^28 rows and one", grad(x, t, a, b, y, dw, ((size_t)1 << 28) + 1));
    ctx.d.lm_vocab = V;
    expect("twice an output", loss(x, t, a, a));
    expect("an output that is an input", grad(x, t, a, b, x, dw));
    moe_ffn block{I, (uint16_t *)w, nullptr, (uint16_t *)(w + 8192), nullptr};
    moe_ffn_grads g{};
    for (int off : {2, 4, 8}) {
      moe_ffn off_block = block;
      off_block.down += off / 2;
      expect("down off", moe_ffn_forward_device(&ctx, &off_block, x, MOE_F32, T, y, nullptr, nullptr));
      expect("y off", moe_ffn_forward_device(&ctx, &block, x, MOE_F32, T, y + off, nullptr, nullptr));
      g.gate_up_bias = (float *)(dw + off);
      expect("bias gradient off", moe_ffn_backward_device(&ctx, &block, x, MOE_F32, y, MOE_F32, T, &g, nullptr));
    }
    // under capture the workspace cannot grow, and is as it was
    g_capturing = true;
    expect("a workspace that capture needs", loss(x, t, a, b), MOE_ERR_STATE);
    if (work.p || work.captured) wrong++, printf("a refused call changed the workspace\n");
    printf("refusals %d wrong %d\n", n, wrong);
    return wrong || g_faults ? 3 : 0;
  }
  if (what == "growth") {
    DenseWork work;
    moe_ctx ctx{};
    const size_t H = 256, V = 4096, most = 4000;
    ctx.d = DenseCtx{nullptr, H, 7.0f, (const uint16_t *)buffer(V * H * 2), V, &work};
    void *x = (void *)buffer(most * H * 4);
    int32_t *t = (int32_t *)buffer(most * 4);
    float *loss = (float *)buffer(most * 4), *lse = (float *)buffer(most * 4);
    int wrong = 0;
    auto call = [&](size_t T, int code = MOE_OK) {
      g_written.clear();
      if (moe_lm_head_loss_device(&ctx, x, MOE_F32, t, T, V, loss, lse, nullptr) != code) wrong++, printf("%zu tokens: not %d\n", T, code);
    };
    auto check = [&](const char *what, bool holds) {
      if (!holds) wrong++, printf("%s: %zu allocations, %zu frees, %zu bytes\n", what, g_allocations, g_frees, work.cap);
    };
    call(1000);
    const size_t exact = work.cap;
    check("the first workspace", g_allocations == 1 && g_frees == 0);
    for (size_t T = 1001; T <= 1200; T++) call(T);
    check("200 lengths that rise by one", g_allocations <= 3 && g_frees == g_allocations - 1 && work.cap < 2 * exact);
    const size_t allocations = g_allocations, frees = g_frees, room = work.cap;
    g_capturing = true;  // within the room a longer call is captured, past it it is refused and nothing changes
    call(1201);
    void *held = work.p;
    call(most, MOE_ERR_STATE);
    check("under capture", g_allocations == allocations && g_frees == frees && work.p == held && work.captured);
    g_capturing = false;
    g_memory = room + room / 8;  // no memory for the room above a length: the length alone
    for (size_t T = 1210; work.cap == room && T < most; T += 10) call(T);
    check("little memory", g_allocations == allocations + 1 && g_frees == frees && work.kept.size() == 1 && work.kept[0] == held && work.cap <= g_memory);
    g_memory = 0;
    const size_t cap = work.cap;
    call(most, MOE_ERR_OOM);
    check("no memory", work.cap == cap && g_frees == frees);
    call(1200);
    printf("wrong %d\n", wrong);
    return wrong || g_faults ? 3 : 0;
  }
  if (what == "draw") {
    std::mt19937_64 rng(strtoull(argv[3], nullptr, 10));
    auto uniform = [&](double lo, double hi) { return lo + (hi - lo) * (double)(rng() >> 11) / 9007199254740992.0; };
    auto log_int = [&](double lo, double hi) { return (size_t)std::min(hi, std::max(lo, std::round(std::exp(uniform(std::log(lo), std::log(hi)))))); };
    std::map<std::string, std::pair<double, Call>> best;
    for (long i = 0, n = strtol(argv[2], nullptr, 10); i < n; i++) {
      Call c;
      const char *ops[] = {"loss", "lossgrad", "ffn", "ffngrad", "ffngrad"};
      c.op = ops[rng() % 5];
      c.dtype = rng() % 2 ? MOE_F32 : MOE_BF16;
      c.T = log_int(1, 16384);
      c.H = rng() % 4 == 0 ? 2880 : 32 * log_int(1, 90);
      c.a = c.b = 0;
      if (c.op == "loss" || c.op == "lossgrad") {
        c.X = log_int(1, 262144);
        c.a = 1, c.b = rng() % 3 != 0;
      } else {
        c.X = 8 * log_int(1, 1000);
        c.a = rng() % 3 == 0;
        c.b = 31;
      }
      g_forms.clear();
      if (!run(c)) continue;
      for (auto &f : g_forms) {
        auto it = best.find(f);
        if (it == best.end() || c.cost() < it->second.first) best[f] = {c.cost(), c};
      }
    }
    for (auto &f : best) printf("%s : %s\n", f.first.c_str(), f.second.second.text().c_str());
    printf("faults %ld\n", g_faults);
    return g_faults ? 3 : 0;
  }
  return 2;
}
