// Plan of the dense products: tile, K parts, the checks before a launch, and the jobs of the launches around the
// products. Host code.
#include "dense_plan.hpp"

#include <algorithm>
#include <cmath>

namespace moe {

namespace {

// k values of each split, a multiple of the step
int split_k(const DenseArgs &a) {
  const long steps = ((long)a.K + kDenseStep - 1) / kDenseStep, n = a.splits < 1 ? 1 : a.splits;
  return (int)((steps + n - 1) / n * kDenseStep);
}

constexpr int kCus = 256;  // of an MI355X: the plan is for the whole device

// Estimated us of a product on one tile shape with its K in `splits` parts. A workgroup's step takes the
// largest of the time that its products take at the tile's full rate, that its loads of A take where A is
// read once, from memory (both shared by the workgroups of its CU), and that its loads wait, spread over
// the steps that its slots hold ahead; each workgroup has a prologue and an epilogue that stores its
// results; parts are summed in another launch. `others`: tiles of the same shape in the launch, as many as do the same steps. Whole rounds of workgroups and what is left for the last one count apart.
double dense_us(const DenseShape &s, const DenseTileDims &d, const DenseArgs &a, int splits, long others = 0) {
  const long tiles_n = ((long)a.N * a.stack + d.bn - 1) / d.bn, tiles = (long)((a.M + d.bm - 1) / d.bm) * tiles_n * splits + others;
  const long steps = (((long)a.K + kDenseStep - 1) / kDenseStep + splits - 1) / splits;
  // bytes that a result costs, about: of rows in planes, results in planes (GATE 3 slots, the gradients 6)
  const bool planes = a.b_planes > 1 || a.stack > 1;
  const double result = s.epi == DENSE_STATS ? 0.0 : s.epi == DENSE_GATE ? (planes ? 3.0 : 1.0)
                        : s.epi == DENSE_DGATE ? (planes ? 44.0 : 14.0) : s.epi == DENSE_DLOGITS ? (planes ? 12.0 : 2.0)
                        : a.out_mode || splits > 1 ? 4.0 : 2.0;
  // a transposed A's rows of k are read in pieces of a tile's rows: below 128 bytes the slower for it
  const double memory = s.at && d.bm < 64 ? 23.0 * d.bm / 64 : 23.0;  // GB/s a CU; 5.9 TB/s in all
  auto round = [&](double on_cu) {
    double step = std::max(0.52 / (d.ns - 1) + 0.12, on_cu * d.bm * d.bn * 2.0 * kDenseStep * d.planes * kCus / (d.rate * 1e6));
    if (tiles_n == 1) step = std::max(step, on_cu * d.bm * 128e-3 / memory);
    const double stores = on_cu * d.bm * d.bn * result * kCus / 4.5e6;  // us at 4.5 TB/s
    // f32 weight gradients of few rows, bound by their stores: of two workgroups a CU one stores while the other
    // starts (19 rows, 32003 x 1024: 128 x 128 31.7 us, 256 x 256 34.3; bf16 rows of such tiles, 256 bytes, went slower)
    if (s.bt && a.out_mode && d.bn == 128 && on_cu == d.wgs && stores > 2.0 * steps * step) return std::max(steps * step + 2.5, stores);
    return steps * step + 2.5 + stores;
  };
  const long whole = tiles / (kCus * d.wgs), rest = tiles - whole * kCus * d.wgs;
  const double on = (double)rest / kCus;  // of the last round: between the busiest CU's and the mean
  double us = whole * round(d.wgs) + (rest ? round(std::max(1.0, 0.5 * (on + std::ceil(on)))) : 0.0);
  if (splits > 1) us += (a.joined ? 0.5 : 4.5) + 4.0 * splits * a.M * a.N / 5e6;
  return us;
}

bool tile_fits(const DenseShape &s, const DenseTileDims &d, const DenseArgs &a) {
  if (d.planes != a.b_planes) return false;
  if (a.stack > 1 && (d.bn > 64 || a.N * a.stack > d.bn)) return false;  // stacked planes lie in one tile
  // 288 rows: K-contiguous they keep too much in registers (620 TFLOP/s)
  return d.bm <= 256 || (s.at && s.epi == DENSE_STORE && a.K >= 1024);
}

constexpr DenseShape kGradient{true, true, DENSE_STORE};

}  // namespace

int dense_pair_tile(const DenseArgs &a, const DenseArgs &b, double &us) {
  int best = -1;
  for (int t = 0; t < kDenseTileCount; t++) {
    const DenseTileDims &d = kDenseTiles[t];
    if (!tile_fits(kGradient, d, a)) continue;
    const double tiles = (double)((b.M + d.bm - 1) / d.bm) * ((b.N + d.bn - 1) / d.bn);
    const double u = dense_us(kGradient, d, a, 1, (long)std::ceil(tiles * b.K / a.K));
    if (best < 0 || u < us) best = t, us = u;
  }
  return best;
}

int dense_tile(const DenseShape &s, const DenseArgs &a) {
  int best = -1;
  double us = 0.0;
  for (int t = 0; t < kDenseTileCount; t++) {
    const DenseTileDims &d = kDenseTiles[t];
    if (!tile_fits(s, d, a)) continue;
    const double u = dense_us(s, d, a, dense_split_count(a));
    if (best < 0 || u < us) best = t, us = u;
  }
  return best;
}

int dense_parts(const DenseShape &s, const DenseArgs &a) {
  const DenseTileDims &d = kDenseTiles[dense_tile(s, a)];
  if (s.epi == DENSE_STATS) return (a.M + d.bm - 1) / d.bm * d.wm;
  if (s.epi == DENSE_DGATE) return (a.N * a.stack + d.bn - 1) / d.bn * d.wn;
  return 0;
}

int dense_split_count(const DenseArgs &a) {
  const long k = split_k(a);
  return (int)((a.K + k - 1) / k);
}

double dense_estimate(const DenseShape &s, const DenseArgs &a) {
  return dense_us(s, kDenseTiles[dense_tile(s, a)], a, dense_split_count(a));
}

int dense_splits(const DenseShape &s, const DenseArgs &a0) {
  if (dense_few_rows(s, a0)) return 1;
  const long steps = ((long)a0.K + kDenseStep - 1) / kDenseStep;
  int best = 1;
  double us = 0.0;
  for (int n : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    if (n > 1 && steps / n < 4) break;
    DenseArgs a = a0;
    a.splits = n;
    a.splits = dense_split_count(a);
    const double u = dense_estimate(s, a);
    if (n == 1 || u < us) best = a.splits, us = u;
  }
  return best;
}

bool dense_pair_pays(const DenseArgs &a, const DenseArgs &b) {
  if (a.splits > 1 || b.splits > 1 || a.K < b.K) return false;
  double us = 0.0;
  dense_pair_tile(a, b, us);
  return us < dense_estimate(kGradient, a) + dense_estimate(kGradient, b);
}

// (more rows of A than 4 tiles a CU keep the rings' larger tiles full, and 16 rows of B took 21.6 us in the
// 2880 x 2880 block against 20.9 through the rings)
int dense_few_rows(const DenseShape &s, const DenseArgs &a) {
  if (s.at || s.bt || (s.epi != DENSE_GATE && s.epi != DENSE_STORE) || a.b_planes != 1 || a.N * a.stack > 8 || a.M % 16 || a.K % 8 ||
      a.M > 16 * 1024 || a.splits > 1 || a.scale || a.out_mode == 2)
    return 0;
  // the fewest rows that fit the CUs once: where some CUs take two workgroups they are waited for (5760 rows of
  // weights by 16: 10.1 us, by 24: 9.4), and where many take none the others have the more to read
  const int rows = (a.M + kCus - 1) / kCus;
  return rows <= 8 ? 8 : rows <= 12 ? 12 : rows <= 16 || rows > 24 ? 16 : 24;
}

namespace {
// Results leave in pieces of 16 bytes (dense_rows; d(gate, up) 4 rows at a time): whole ones, in rows that lie so.
bool stores_fit(DenseEpi epi, const DenseArgs &a) {
  const size_t M = (size_t)a.M;
  switch (epi) {
    case DENSE_STORE: return a.out_mode == 0 ? M % 8 == 0 && a.ldo % 8 == 0 && a.ldo >= M : M % 4 == 0 && a.ldo % 4 == 0 && a.ldo >= M;
    case DENSE_GATE: return M % 16 == 0 && a.ldh % 8 == 0 && a.ldh >= M / 2;
    case DENSE_DGATE: return M % 4 == 0 && a.ldh % 4 == 0 && a.ldh >= M;
    case DENSE_DLOGITS: return a.ld_dl % 8 == 0 && a.ld_dl >= M;
    case DENSE_STATS: return true;
  }
  return false;
}
}  // namespace

hipError_t dense_prepare(const DenseShape &s, DenseArgs &a) {
  if (a.M <= 0 || a.N <= 0 || a.K <= 0 || (a.b_planes != 1 && a.b_planes != kPlanes) || a.stack < 1 || a.lda % 8 || a.ldb % 8)
    return hipErrorInvalidValue;
  if (!stores_fit(s.epi, a)) return hipErrorInvalidValue;
  a.k_split = split_k(a);
  a.splits = dense_split_count(a);
  if (a.splits > 1 && (s.epi != DENSE_STORE || a.out_mode != 1)) return hipErrorInvalidValue;
  return hipSuccess;
}

hipError_t dense_prepare_pair(DenseArgs &a, DenseArgs &b) {
  for (DenseArgs *x : {&a, &b}) {
    if (x->M <= 0 || x->N <= 0 || x->K <= 0 || x->b_planes != 1 || x->stack != 1 || x->lda % 8 || x->ldb % 8 || x->splits > 1 || x->K > a.K ||
        !stores_fit(DENSE_STORE, *x))
      return hipErrorInvalidValue;
    x->k_split = split_k(*x);
  }
  return hipSuccess;
}

int dense_dgate_parts(int T) { return (T + kDgateRows - 1) / kDgateRows; }
int dense_colsum_parts(size_t T) { return (int)((T + kColRows - 1) / kColRows); }

namespace {
unsigned blocks_for(size_t n) { return (unsigned)std::min<size_t>((n + 255) / 256, 65536); }
// where the blocks of each job end; their number
template <class J>
size_t dense_ends(J &a) {
  size_t blocks = 0;
  for (int i = 0; i < (int)(sizeof(a.d) / sizeof(a.d[0])); i++) {
    if (i < a.count) blocks += a.d[i].blocks;
    a.end[i] = (unsigned)blocks;
  }
  return blocks;
}
}  // namespace

size_t DenseRowJobs::ends() { return dense_ends(*this); }
size_t DenseSums::ends() { return dense_ends(*this); }
void DenseRowJobs::planes(const float *x, uint16_t *out, uint32_t where, size_t n, const int32_t *targets, size_t cols) {
  if (n) d[count++] = DenseRows{ROWS_PLANES, x, out, n, cols, where, 0, blocks_for(n / 4), targets};
}
void DenseRowJobs::copy(const uint16_t *x, uint16_t *out, size_t n, const int32_t *targets, size_t cols) {
  if (n) d[count++] = DenseRows{ROWS_COPY, x, out, n, cols, 0, 0, blocks_for(n / 8), targets};
}
void DenseRowJobs::pack8(const float *x, size_t n, uint8_t *packed) {
  if (n) d[count++] = DenseRows{ROWS_PACK8, x, packed, n, 0, 0, 0, blocks_for(n / 8), nullptr};
}
void DenseRowJobs::unpack8(const uint8_t *packed, size_t n, uint16_t *out, int copies) {
  if (n) d[count++] = DenseRows{ROWS_UNPACK8, packed, out, n, 0, 0, copies, blocks_for(n / 8), nullptr};
}
void DenseRowJobs::column_sums(const void *x, bool bf16, size_t T, size_t H, float *out) {
  d[count++] = DenseRows{bf16 ? ROWS_SUM_BF16 : ROWS_SUM_F32, x, out, T, H, 0, 0, (unsigned)((H + 63) / 64), nullptr};
}
void DenseRowJobs::dloss_scale(const DlossScale &s) {
  scale = s;
  d[count++] = DenseRows{ROWS_DLOSS_SCALE, nullptr, nullptr, 0, 0, 0, 0, 1, nullptr};
}

void DenseSums::add(const float *part, size_t stride, int parts, size_t n, const float *bias, size_t n_bias, void *out, bool bf16) {
  const bool few = !bf16 && !bias && n <= 65536 && parts > 8;
  d[count++] = DenseSum{part, stride, n, n_bias, bias, out, parts, few ? (unsigned)((n + 31) / 32) : blocks_for(n), bf16, few};
}

}  // namespace moe
