// C ABI of the dense operators (include/moe_dense.h): checks, workspace, and the order of launches.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/moe_dense.h"
#include "call.hpp"
#include "dense.hpp"
#include "kernels.hpp"

using namespace moe;

namespace {

// Rows [n][cols] as the products take them: their values, or their planes in slots.
struct Rows {
  const uint16_t *p = nullptr;
  size_t n = 0, cols = 0, ld = 0;
  int slots = 1;
  uint32_t where = kWhereOne;
  uint16_t *out() const { return const_cast<uint16_t *>(p); }
  size_t slot() const { return n * ld; }
  size_t size() const { return slots * slot(); }
};
Rows rows_of(int dtype, uint32_t where, size_t n, size_t cols, size_t ld) {
  if (dtype == MOE_BF16) return Rows{nullptr, n, cols, ld};
  return Rows{nullptr, n, cols, ld, where == kWhereThree ? kPlanes : kPairs6, where};
}
// rows in the workspace; of a caller's matrix only if it is f32
Rows place(Carve &w, Rows r) {
  r.p = w.take<uint16_t>(r.size());
  return r;
}
Rows place(Carve &w, Rows r, const void *x, int dtype) {
  if (dtype != MOE_BF16) return place(w, r);
  r.p = (const uint16_t *)x;
  return r;
}
void fill(DenseRowJobs &jobs, const Rows &r, const void *x, int dtype) {
  if (dtype == MOE_F32) jobs.planes((const float *)x, r.out(), r.where, r.slot());
}

// Weights times rows: D[m][n] = sum W[m][k] rows[n][k] (W [M][K], or [K][M] for a launch with A transposed),
// the rows' lower planes first; of few rows, all planes as rows. (Before the rows have a place, for the plan alone.)
DenseArgs product(const uint16_t *W, size_t ldw, const Rows &b, size_t M) {
  DenseArgs a{};
  a.A = W;
  a.lda = ldw;
  a.B = b.p;
  a.ldb = b.ld;
  a.b_slot = b.slot();
  a.M = (int)M;
  a.N = (int)b.n;
  a.K = (int)b.cols;
  a.splits = a.stack = a.stack_step = a.b_planes = 1;
  if (b.where != kWhereOne) {
    if (b.n * kPlanes <= 64) {
      a.stack = kPlanes;  // the last slots of the planes: three in a row, of a right operand every other one
      a.stack_step = b.where == kWhereRight ? 2 : 1;
      if (a.B) a.B += (dense_last_slot(b.where, 0) - (kPlanes - 1) * a.stack_step) * a.b_slot;
    } else {
      a.b_planes = kPlanes;
      for (int i = 0; i < kPlanes; i++) a.pb |= (uint32_t)dense_last_slot(b.where, kPlanes - 1 - i) << 4 * i;
    }
  }
  return a;
}
// Rows times rows over their rows: D[m][n] = sum_t a[t][m] b[t][n]; of copies of a's values and b's three planes,
// or of both's planes in pairs.
DenseArgs gradient(const Rows &x, const Rows &y) {
  DenseArgs a{};
  a.A = x.p;
  a.lda = x.ld;
  a.B = y.p;
  a.ldb = y.ld;
  a.M = (int)x.cols;
  a.N = (int)y.cols;
  a.K = (int)(std::min(x.slots, y.slots) * x.n);
  a.splits = a.stack = a.stack_step = a.b_planes = 1;
  return a;
}

// out [N][M] (+ bias) of a product, K split where that fills the device; part: [splits][N][M] f32 then, whose
// sum is left to `sums`.
int store(DenseArgs a, bool at, bool bt, int splits, float *part, const float *bias, void *out, int dtype, DenseSums &sums, hipStream_t s) {
  const DenseShape shape{at, bt, DENSE_STORE};
  a.ldo = (size_t)a.M;
  if (splits > 1) {
    a.splits = splits;
    a.split_stride = (size_t)a.M * a.N;
    a.out = part;
    a.out_mode = 1;
    HIP_TRY(launch_dense(shape, a, s));
    sums.add(part, a.split_stride, dense_split_count(a), a.split_stride, bias, (size_t)a.M, out, dtype == MOE_BF16);
    return MOE_OK;
  }
  a.out = out;
  a.out_mode = dtype == MOE_BF16 ? 0 : 1;
  a.bias = bias;
  HIP_TRY(launch_dense(shape, a, s));
  return MOE_OK;
}

int zero(void *p, size_t bytes, hipStream_t s) {
  if (p) HIP_TRY(launch_zero(p, bytes, s));
  return MOE_OK;
}

// ------------------------------------------------------------------ loss

int check_loss(const DenseCtx &c, const void *x, int dtype, const int32_t *targets, size_t T, size_t vocab) {
  RETURN_IF(check_dtype(dtype));
  if (!c.lm_vocab) return fail(MOE_ERR_STATE, "call init_lm_head_bf16 first");
  if (!c.lm_w) return fail(MOE_ERR_STATE, "the loss reads the bf16 LM head; the context holds the f32 one");
  if (!vocab || vocab > c.lm_vocab)
    return fail(MOE_ERR_INVALID, "vocab %zu outside [1, %zu]", vocab, c.lm_vocab);
  if (vocab > kMaxVocab) return fail(MOE_ERR_INVALID, "vocab %zu above %zu", vocab, kMaxVocab);
  RETURN_IF(check_tokens(T));
  if (T && (!x || !targets)) return fail(MOE_ERR_INVALID, "null x or targets");
  RETURN_IF(check_aligned({targets}, 4));
  return check_aligned({x});
}

// tokens whose statistics are kept at once: up to 16384, and of wide heads (2^18 rows and more) so many that their
// statistics, a maximum and a sum per 64 to 128 rows, stay below 512 MB and a launch's threads below 2^32, 256 at least
size_t loss_tokens(size_t vocab) {
  size_t n = 16384;
  while (n > 256 && n * (vocab / 64) * 8 > (size_t)512 << 20) n /= 2;
  return n;
}
constexpr size_t kGradTokens = 8192;                  // tokens and bytes of the logits' gradient at once
constexpr size_t kGradBytes = (size_t)512 << 20;

// ------------------------------------------------------------------ gated block

int check_block(const moe_ffn *b, const void *x, const void *other, size_t T) {
  if (!b || !b->gate_up || !b->down) return fail(MOE_ERR_INVALID, "null block or weights");
  if (!b->inter || b->inter % 8 || b->inter > kMaxInter)
    return fail(MOE_ERR_INVALID, "inter %zu must be a positive multiple of 8, at most %zu", b->inter, kMaxInter);
  RETURN_IF(check_tokens(T));
  if (T && (!x || !other)) return fail(MOE_ERR_INVALID, "null rows");
  return check_aligned({b->gate_up, b->gate_up_bias, b->down, b->down_bias, x, other});
}

}  // namespace

extern "C" {

int moe_lm_head_loss_device(moe_ctx *ctx, const void *x, int dtype, const int32_t *targets, size_t T, size_t vocab,
                            float *loss, float *lse, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_loss(c, x, dtype, targets, T, vocab));
  if (!T) return MOE_OK;
  if (!loss || !lse) return fail(MOE_ERR_INVALID, "null loss or lse");
  RETURN_IF(check_aligned({loss, lse}, 4));
  RETURN_IF(check_distinct({loss, lse}, {x, targets, c.lm_w}));
  const hipStream_t s = stream ? (hipStream_t)stream : c.stream;
  const size_t H = c.H, Tc = std::min(T, loss_tokens(vocab));
  const DenseShape shape{false, false, DENSE_STATS};
  Carve w;
  Rows r;
  float2 *stats = nullptr;
  float *picked = nullptr;
  for (int placed = 0; placed < 2; placed++) {
    r = rows_of(dtype, kWhereThree, Tc, H, H);
    size_t most = 0;  // (the last piece of tokens may take another tile)
    for (size_t t0 = 0; t0 < T; t0 += Tc) {
      r.n = std::min(Tc, T - t0);
      most = std::max(most, r.n * (size_t)dense_parts(shape, product(c.lm_w, H, r, vocab)));
    }
    r.n = Tc;
    r = place(w, r, x, dtype);
    stats = w.take<float2>(most);
    picked = w.take<float>(Tc);
    if (!placed) {
      RETURN_IF(ensure(c, w.off, s));
      w = Carve{(char *)c.work->p};
    }
  }
  for (size_t t0 = 0; t0 < T; t0 += Tc) {
    const size_t n = std::min(Tc, T - t0);
    Rows piece = r;
    piece.n = n;
    if (dtype == MOE_BF16) piece.p += t0 * H;
    DenseRowJobs jobs;
    fill(jobs, piece, (const char *)x + t0 * H * elem(dtype), dtype);
    HIP_TRY(launch_rows(jobs, s));
    DenseArgs a = product(c.lm_w, H, piece, vocab);
    a.targets = targets + t0;
    a.stats = stats;
    a.picked = picked;
    HIP_TRY(launch_dense(shape, a, s));
    HIP_TRY(launch_loss(stats, dense_parts(shape, a), picked, targets + t0, n, (int)vocab, loss + t0, lse + t0, s));
  }
  return MOE_OK;
}

int moe_lm_head_loss_backward_device(moe_ctx *ctx, const void *x, int dtype, const int32_t *targets, const float *lse,
                                     const float *dloss, size_t T, size_t vocab, void *dx, void *dw, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_loss(c, x, dtype, targets, T, vocab));
  RETURN_IF(check_aligned({dx, dw}));
  const hipStream_t s = stream ? (hipStream_t)stream : c.stream;
  const size_t H = c.H;
  RETURN_IF(check_distinct({dx, dw}, {x, targets, lse, dloss, c.lm_w}));
  if (!T) return zero(dw, vocab * H * elem(dtype), s);
  if (!lse || !dloss) return fail(MOE_ERR_INVALID, "null lse or dloss");
  RETURN_IF(check_aligned({lse, dloss}, 4));
  if (!dx && !dw) return MOE_OK;
  const int P = dtype == MOE_BF16 ? 1 : kPlanes;
  const bool bf = dtype == MOE_BF16;
  // pieces of tokens and of the vocabulary whose gradient of the logits is held at once
  const size_t Tc = std::min(T, kGradTokens), nt = (T + Tc - 1) / Tc;
  const size_t most = std::max<size_t>(256, kGradBytes / (2 * (bf ? 1 : kPairs6) * Tc) / 256 * 256), nv = (vocab + most - 1) / most;
  const size_t Vc = std::min(vocab, ((vocab + nv - 1) / nv + 255) / 256 * 256), ld = (Vc + 7) / 8 * 8;
  const DenseShape sx{true, false, DENSE_STORE}, sw{true, true, DENSE_STORE};
  // few tokens: dx from K splits of every piece of the vocabulary, summed at the end; many: added up
  const int splits = dense_splits(sx, product(c.lm_w, H, rows_of(dtype, kWhereRight, Tc, Vc, ld), H));
  const bool parts = dx && splits > 1 && nt == 1;
  const bool masked = !bf || dw;  // the rows in the workspace, those of ignored tokens as zeros
  Carve w;
  Rows r, dl;
  float *dx_acc = nullptr, *dw_acc = nullptr, *scale = nullptr;
  for (int placed = 0; placed < 2; placed++) {
    r = rows_of(dtype, kWhereLeft, T, H, H);
    r = masked ? place(w, r) : place(w, r, x, dtype);  // (f32: the slots of each piece of tokens together)
    scale = w.take<float>(1);
    dl = place(w, rows_of(dtype, kWhereRight, Tc, Vc, ld));
    if (parts)
      dx_acc = w.take<float>(nv * splits * T * H);
    else if (dx)
      dx_acc = bf && nv > 1 ? w.take<float>(T * H) : bf ? nullptr : (float *)dx;
    if (dw) dw_acc = bf && nt > 1 ? w.take<float>(Vc * H) : nullptr;
    if (!placed) {
      RETURN_IF(ensure(c, w.off, s));
      w = Carve{(char *)c.work->p};
    }
  }
  auto piece = [&](size_t t0, size_t n) {
    Rows q = r;
    q.p += r.slots * t0 * H;
    q.n = n;
    return q;
  };
  // The gradient of the logits is held over the largest |dloss| and the results multiplied by it: for the
  // mean's constant dloss the entries of the targets, which weigh most, then lie next to -1 and are rounded
  // by their p alone, where bf16(1 / n) would put one error into all of them.
  const DlossScale largest{dloss, targets, T, (int)vocab, scale};
  const bool beside = masked && T <= 1024;  // in the launch that prepares the rows
  if (!beside) HIP_TRY(launch_dloss_scale(largest, s));
  for (size_t t0 = 0; t0 < T && masked; t0 += Tc) {
    const size_t n = std::min(Tc, T - t0);
    const Rows p = piece(t0, n);
    DenseRowJobs jobs;
    if (bf)
      jobs.copy((const uint16_t *)x + t0 * H, p.out(), n * H, targets + t0, H);
    else
      jobs.planes((const float *)x + t0 * H, p.out(), p.where, n * H, targets + t0, H);
    if (beside) jobs.dloss_scale(largest);
    HIP_TRY(launch_rows(jobs, s));
  }
  int written = 0;  // parts of dx
  for (size_t v0 = 0; v0 < vocab; v0 += Vc) {
    const size_t nvoc = std::min(Vc, vocab - v0);
    const uint16_t *wv = c.lm_w + v0 * H;
    for (size_t t0 = 0; t0 < T; t0 += Tc) {
      const size_t n = std::min(Tc, T - t0);
      const Rows rows = piece(t0, n);
      Rows d = dl;
      d.n = n;
      d.cols = nvoc;
      DenseArgs a = product(wv, H, rows, nvoc);
      a.targets = targets + t0;
      a.lse = lse + t0;
      a.dloss = dloss + t0;
      a.scale = scale;
      a.v0 = (int)v0;
      a.vocab = (int)vocab;
      a.dl = d.out();
      a.dl_slot = d.slot();
      a.dl_where = d.where;
      a.ld_dl = ld;
      a.planes = P;
      HIP_TRY(launch_dense(DenseShape{false, false, DENSE_DLOGITS}, a, s));
      if (dx) {
        DenseArgs g = product(wv, H, d, H);
        g.ldo = H;
        g.scale = scale;
        if (parts) {
          g.splits = splits;
          g.split_stride = T * H;
          g.out = dx_acc + (size_t)written * T * H;
          g.out_mode = 1;
          written += dense_split_count(g);
        } else if (dx_acc) {
          g.out = dx_acc + t0 * H;
          g.out_mode = v0 ? 2 : 1;
        } else {
          g.out = (uint16_t *)dx + t0 * H;
        }
        HIP_TRY(launch_dense(sx, g, s));
      }
      if (dw) {
        DenseArgs g = gradient(rows, d);
        g.ldo = H;
        g.scale = scale;
        if (!bf || dw_acc) {
          g.out = bf ? dw_acc : (float *)dw + v0 * H;
          g.out_mode = t0 ? 2 : 1;
        } else {
          g.out = (uint16_t *)dw + v0 * H;
        }
        HIP_TRY(launch_dense(sw, g, s));
      }
    }
    if (dw && dw_acc) {
      DenseSums sums;
      sums.add(dw_acc, 0, 1, nvoc * H, nullptr, 1, (uint16_t *)dw + v0 * H, true);
      HIP_TRY(launch_sums(sums, s));
    }
  }
  DenseSums sums;
  if (parts)
    sums.add(dx_acc, T * H, written, T * H, nullptr, 1, dx, bf);
  else if (dx && dx_acc && bf)
    sums.add(dx_acc, 0, 1, T * H, nullptr, 1, dx, true);
  HIP_TRY(launch_sums(sums, s));
  return MOE_OK;
}

int moe_ffn_forward_device(moe_ctx *ctx, const moe_ffn *b, const void *x, int dtype, size_t T, void *y, uint8_t *x8,
                           void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_dtype(dtype));
  RETURN_IF(check_block(b, x, y, T));
  RETURN_IF(check_aligned({x8}));
  if (!T) return MOE_OK;
  RETURN_IF(check_distinct({y, x8}, {x, b->gate_up, b->gate_up_bias, b->down, b->down_bias}));
  const hipStream_t s = stream ? (hipStream_t)stream : c.stream;
  const size_t H = c.H, I = b->inter;
  const int P = dtype == MOE_BF16 ? 1 : kPlanes;
  Carve w;
  Rows r, h;
  float *part = nullptr;
  int splits = 1;
  for (int placed = 0; placed < 2; placed++) {
    r = place(w, rows_of(dtype, kWhereThree, T, H, H), x, dtype);
    h = place(w, rows_of(dtype, kWhereThree, T, I, I));
    splits = dense_splits(DenseShape{false, false, DENSE_STORE}, product(b->down, I, h, H));
    part = splits > 1 ? w.take<float>(splits * T * H) : nullptr;
    if (!placed) {
      RETURN_IF(ensure(c, w.off, s));
      w = Carve{(char *)c.work->p};
    }
  }
  DenseRowJobs jobs;
  fill(jobs, r, x, dtype);
  if (x8 && dtype == MOE_F32) jobs.pack8((const float *)x, T * H, x8);
  if (x8 && dtype == MOE_BF16) HIP_TRY(launch_act8_pack(x, true, T, H, x8, s));
  HIP_TRY(launch_rows(jobs, s));
  DenseArgs g = product(b->gate_up, H, r, 2 * I);
  g.bias = b->gate_up_bias;
  g.limit = c.clamp;
  g.h = h.out();
  g.h_slot = h.slot();
  g.h_where = h.where;
  g.ldh = I;
  g.planes = P;
  HIP_TRY(launch_dense(DenseShape{false, false, DENSE_GATE}, g, s));
  DenseSums sums;
  RETURN_IF(store(product(b->down, I, h, H), false, false, splits, part, b->down_bias, y, dtype, sums, s));
  HIP_TRY(launch_sums(sums, s));
  return MOE_OK;
}

int moe_ffn_backward_device(moe_ctx *ctx, const moe_ffn *b, const void *x, int x_type, const void *dy, int dtype, size_t T,
                            const moe_ffn_grads *out, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_dtype(dtype));
  if (x_type != dtype && x_type != MOE_MXFP8)
    return fail(MOE_ERR_INVALID, "x_type %d is neither dtype %d nor MOE_MXFP8", x_type, dtype);
  if (!out) return fail(MOE_ERR_INVALID, "null gradients");
  RETURN_IF(check_block(b, x, dy, T));
  RETURN_IF(check_aligned({out->x, out->gate_up, out->gate_up_bias, out->down, out->down_bias}));
  RETURN_IF(check_distinct({out->x, out->gate_up, out->gate_up_bias, out->down, out->down_bias},
                           {x, dy, b->gate_up, b->gate_up_bias, b->down, b->down_bias}));
  const hipStream_t s = stream ? (hipStream_t)stream : c.stream;
  const size_t H = c.H, I = b->inter, el = elem(dtype);
  if (!T) {
    RETURN_IF(zero(out->gate_up, 2 * I * H * el, s));
    RETURN_IF(zero(out->gate_up_bias, 2 * I * 4, s));
    RETURN_IF(zero(out->down, H * I * el, s));
    return zero(out->down_bias, H * 4, s);
  }
  const int P = dtype == MOE_BF16 ? 1 : kPlanes;
  const bool bf = dtype == MOE_BF16;
  const bool inner = out->x || out->gate_up || out->gate_up_bias || out->down;
  const DenseShape ss{false, false, DENSE_STORE}, sg{true, false, DENSE_DGATE}, sx{true, false, DENSE_STORE}, sw{true, true, DENSE_STORE};
  const uint32_t to_x = x_type == MOE_MXFP8 ? kWhereThree : kWhereRight;  // d(gate, up): a checkpoint's copies meet its planes one by one
  Carve w;
  Rows r, d, h, dgu;
  float *gu = nullptr, *dh = nullptr, *db = nullptr, *col = nullptr, *px = nullptr, *pgu = nullptr, *pd = nullptr;
  int nx = 1, ngu = 1, nd = 1, db_parts = 0, n_raw = 1, n_dh = 1;
  bool apart = false;  // d(gate, up) in a kernel of its own, from K parts of gate, up and dh
  for (int placed = 0; placed < 2; placed++) {
    if (inner) {
      if (x_type == MOE_MXFP8) {  // exact in bf16: one plane, a copy of it for each of the planes it meets
        r = Rows{nullptr, T, H, H, bf ? 1 : kPlanes};
        r = place(w, r);
      } else {
        r = place(w, rows_of(dtype, kWhereLeft, T, H, H), x, dtype);
      }
      d = place(w, rows_of(dtype, kWhereRight, T, H, H), dy, dtype);
      // Few rows leave most of the device idle in products that are not split: then gate, up and dh come in K
      // parts, which a kernel of its own joins (333 f32 rows, 2048 x 1536: 20 + 13.6 + 10 us; DENSE_DGATE, with
      // gate and up before it, 24 + 25)
      DenseArgs raw = product(b->gate_up, H, r, 2 * I);
      DenseArgs in = product(b->down, I, d, I);
      raw.out_mode = in.out_mode = 1;
      const double one = dense_estimate(ss, raw) + dense_estimate(sg, in);
      raw.joined = in.joined = true;
      raw.splits = n_raw = dense_splits(ss, raw);
      in.splits = n_dh = dense_splits(sx, in);
      // (that kernel's bytes at 5 TB/s; what its parts cost is in the estimates)
      const double bytes = ((n_raw > 1 ? 0.0 : 8.0) + (n_dh > 1 ? 0.0 : 4.0) + 2.0 * rows_of(dtype, kWhereLeft, T, I, I).slots +
                            4.0 * rows_of(dtype, to_x, T, I, I).slots) * T * I;
      apart = dense_estimate(ss, raw) + dense_estimate(sx, in) + 1.0 + bytes / 5e6 < one && T <= 65536;
      if (!apart) n_raw = n_dh = 1;
      gu = w.take<float>(n_raw * T * 2 * I);
      dh = apart ? w.take<float>(n_dh * T * I) : nullptr;
      h = place(w, rows_of(dtype, kWhereLeft, T, I, I));
      dgu = place(w, rows_of(dtype, to_x, T, 2 * I, 2 * I));
      db_parts = apart ? dense_dgate_parts((int)T) : dense_parts(sg, product(b->down, I, d, I));
      // (one part is the result)
      db = !out->gate_up_bias ? nullptr : db_parts > 1 ? w.take<float>((size_t)db_parts * 2 * I) : out->gate_up_bias;
      auto splits = [&](const DenseShape &shape, DenseArgs a) {
        a.joined = db_parts > 1 && out->gate_up_bias;
        return dense_splits(shape, a);
      };
      nx = splits(sx, product(b->gate_up, H, dgu, H));
      ngu = splits(sw, gradient(r, dgu));
      nd = splits(sw, gradient(h, d));
      px = out->x && nx > 1 ? w.take<float>(nx * T * H) : nullptr;
      pgu = out->gate_up && ngu > 1 ? w.take<float>(ngu * 2 * I * H) : nullptr;
      pd = out->down && nd > 1 ? w.take<float>(nd * I * H) : nullptr;
    }
    col = !out->down_bias ? nullptr : dense_colsum_parts(T) > 1 ? w.take<float>(dense_colsum_parts(T) * H) : out->down_bias;
    if (!placed) {
      RETURN_IF(ensure(c, w.off, s));
      w = Carve{(char *)c.work->p};
    }
  }
  DenseSums sums;  // in one launch at the end
  DenseRowJobs jobs;
  if (out->down_bias && col == out->down_bias) {
    jobs.column_sums(dy, bf, T, H, col);
  } else if (out->down_bias) {
    HIP_TRY(launch_colsum(dy, bf, T, H, col, s));
    sums.add(col, H, dense_colsum_parts(T), H, nullptr, 1, out->down_bias, false);
  }
  if (inner) {
    if (x_type == MOE_MXFP8) jobs.unpack8((const uint8_t *)x, T * H, r.out(), r.slots);
    if (dtype == MOE_F32) jobs.planes((const float *)dy, d.out(), d.where, T * H);
    if (x_type == MOE_F32) jobs.planes((const float *)x, r.out(), r.where, T * H);
  }
  HIP_TRY(launch_rows(jobs, s));
  if (!inner) {
    HIP_TRY(launch_sums(sums, s));
    return MOE_OK;
  }
  // gate and up as f32, their K parts side by side
  auto parts = [&](const DenseShape &shape, DenseArgs g, int splits, const float *bias, float *out) -> int {
    g.ldo = (size_t)g.M;
    g.out = out;
    g.out_mode = 1;
    g.splits = splits;
    g.split_stride = (size_t)g.M * g.N;
    g.bias = bias;
    HIP_TRY(launch_dense(shape, g, s));
    return MOE_OK;
  };
  RETURN_IF(parts(ss, product(b->gate_up, H, r, 2 * I), n_raw, apart ? nullptr : b->gate_up_bias, gu));
  DenseArgs g = product(b->down, I, d, I);
  if (apart) {
    RETURN_IF(parts(sx, g, n_dh, nullptr, dh));
    HIP_TRY(launch_dgate(DgateArgs{gu, b->gate_up_bias, dh, n_raw, n_dh, (int)T, (int)I, P, c.clamp, h.out(), dgu.out(), h.where, dgu.where, db}, s));
  } else {
    g.limit = c.clamp;
    g.gu = gu;
    g.h = h.out();
    g.h_slot = h.slot();
    g.h_where = h.where;
    g.ldh = I;
    g.dgu = dgu.out();
    g.dgu_slot = dgu.slot();
    g.dgu_where = dgu.where;
    g.db_part = db;
    g.planes = P;
    HIP_TRY(launch_dense(sg, g, s));
  }
  if (db && db_parts > 1) sums.add(db, 2 * I, db_parts, 2 * I, nullptr, 1, out->gate_up_bias, false);
  if (out->x) RETURN_IF(store(product(b->gate_up, H, dgu, H), true, false, nx, px, nullptr, out->x, dtype, sums, s));
  DenseArgs wd = gradient(h, d), wgu = gradient(r, dgu);  // (of a checkpoint's x, wgu has the fewer rows)
  wd.out_mode = wgu.out_mode = bf ? 0 : 1;
  if (out->gate_up && out->down && ngu == 1 && nd == 1 && dense_pair_pays(wd, wgu)) {
    wd.ldo = I;
    wd.out = out->down;
    wgu.ldo = H;
    wgu.out = out->gate_up;
    HIP_TRY(launch_dense_pair(wd, wgu, s));
  } else {
    if (out->gate_up) RETURN_IF(store(wgu, true, true, ngu, pgu, nullptr, out->gate_up, dtype, sums, s));
    if (out->down) RETURN_IF(store(wd, true, true, nd, pd, nullptr, out->down, dtype, sums, s));
  }
  HIP_TRY(launch_sums(sums, s));
  return MOE_OK;
}

size_t moe_act8_bytes(size_t n, size_t cols) { return cols % 32 ? 0 : n * cols + n * (cols / 32); }

static int check_act8(const void *from, const void *to, int dtype, size_t n, size_t cols) {
  RETURN_IF(check_dtype(dtype));
  if (!cols || cols % 32 || cols > kMaxInter) return fail(MOE_ERR_INVALID, "cols %zu must be a positive multiple of 32, at most %zu", cols, kMaxInter);
  RETURN_IF(check_tokens(n));
  if (n && (!from || !to)) return fail(MOE_ERR_INVALID, "null argument");
  RETURN_IF(check_aligned({from, to}));
  return n ? check_distinct({to}, {from}) : MOE_OK;
}

int moe_act8_pack_device(moe_ctx *ctx, const void *x, int dtype, size_t n, size_t cols, uint8_t *packed, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_act8(x, packed, dtype, n, cols));
  HIP_TRY(launch_act8_pack(x, dtype == MOE_BF16, n, cols, packed, stream ? (hipStream_t)stream : c.stream));
  return MOE_OK;
}

int moe_act8_unpack_device(moe_ctx *ctx, const uint8_t *packed, size_t n, size_t cols, void *out, int dtype, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_act8(packed, out, dtype, n, cols));
  HIP_TRY(launch_act8_unpack(packed, n, cols, out, dtype == MOE_BF16, stream ? (hipStream_t)stream : c.stream));
  return MOE_OK;
}

}  // extern "C"
