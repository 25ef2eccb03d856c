// Host interface of the dense operators' kernels (dense_gemm.hpp, dense.hip, act8.hip): bf16 matrix
// products with the epilogues of the LM-head loss and of the gated feed-forward block.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

namespace moe {

// f32 values enter the bf16 MFMA as the sum of kPlanes bf16 values (8 significant bits each: the 24
// of an f32 exactly, short of the subnormal range); bf16 values as one. A matrix of such values lies in
// the workspace as slots [slot][rows][cols], each a plane: `where` holds in byte p the slots of plane p.
// The product of two such matrices over their rows (a weight gradient) leaves out the planes' products
// below 2^-24 of the largest and takes the other six as one product over 6 times the rows: its left
// operand's slots hold the planes 0 0 1 1 2 0, its right one's 1 2 0 1 0 0. (As six passes over K, each with
// a K tail of its own, the gradient of the LM head for 19 rows took 54 us.)
// A value that is not finite (or is not as bf16) is plane 0 alone, and in the last slot of that plane alone, 0 in
// the others: met with the other operand's lower planes, which may be 0 or of the other sign, an infinity would
// become NaN. So the last slots of plane 0 meet each other, and the products that read one slot of each plane
// take the last ones: 5 3 4 (left) and 5 3 1 (right), of three slots 2 1 0.
constexpr int kPlanes = 3;
constexpr int kPairs6 = 6;
constexpr uint32_t kWhereOne = 0x01, kWhereThree = 0x010204, kWhereLeft = 0x100C23, kWhereRight = 0x020934;
constexpr int dense_last_slot(uint32_t where, int plane) { return 31 - __builtin_clz(where >> 8 * plane & 255); }

// Epilogues. What they leave for the next product (h, d(gate, up), the logits' gradient) is in the activations'
// type, as the products take it: f32 in three planes, bf16 rounded once more, 2^-8. A second plane of bf16 rows would
// double the time of the product that reads it; without the rounding a block's results were 0.0017 off (relative, 4096
// rows), with it 0.0023 to 0.0024.
enum DenseEpi {
  DENSE_STORE = 0,   // out (+ bias) as f32 or bf16, or added to f32
  DENSE_GATE = 1,    // rows of D are interleaved gate and up: h = act(gate, up) as bf16 planes
  DENSE_DGATE = 2,   // D = dh: with the gate and up of gu they give h, d(gate, up) and bias sums
  DENSE_STATS = 3,   // D = logits: running maximum and sum of exponentials of each column's tile
  DENSE_DLOGITS = 4  // D = logits: their gradient as bf16 planes
};

// D[m][n] = sum over B's planes and k of A[m][k] B_p[n][k], stored as [n][m] (m contiguous).
// Layouts of an operand: K-contiguous ([rows][k], the fast case) or transposed ([k][rows]).
// A K-contiguous operand is readable up to K rounded up to 8; a transposed one's rows up to M (N)
// rounded up to 8.
struct DenseArgs {
  const uint16_t *A, *B;
  size_t b_slot;            // elements between slots of B
  size_t lda, ldb;          // elements between rows of the stored matrix
  int M, N, K;
  int stack;                // slots of B that are taken as rows [slot][N] (N * stack <= 64), else 1
  int stack_step;           // from one of these slots to the next: 1 or 2
  int b_planes;             // slots of B that meet A's values in turn: 1, or kPlanes
  uint32_t pb;              // those slots, 4 bits each, in the order of their products
  int splits;               // K split (DENSE_STORE with f32 only): out + split * split_stride
  int k_split;              // K per split, a multiple of the step
  bool joined;              // for the plan: a launch that comes anyway sums the splits
  // DENSE_STORE
  void *out;
  size_t ldo, split_stride;
  int out_mode;             // 0 bf16, 1 f32, 2 f32 added to
  const float *bias;        // [M] or NULL
  const float *scale;       // factor of the result (one value) or NULL; of the loss: what dloss is divided by
  // gated block
  float limit;
  uint16_t *h;              // [slots][N][ldh] bf16
  size_t h_slot, ldh;
  uint32_t h_where;
  const float *gu;          // [N][2 M]
  uint16_t *dgu;            // [slots][N][2 M]
  size_t dgu_slot;
  uint32_t dgu_where;
  float *db_part;           // [parts][2 M] or NULL
  int planes;
  // loss
  const int32_t *targets;   // [N], in the whole vocabulary
  int v0;                   // first vocabulary row of D
  float2 *stats;            // [parts][N]: maximum, sum of exp(l - maximum)
  float *picked;            // [N] target logits
  const float *lse, *dloss; // [N]
  int vocab;                // rows of the whole vocabulary: targets at or above it are invalid
  uint16_t *dl;             // [slots][N][ld_dl]
  size_t dl_slot, ld_dl;
  uint32_t dl_where;
};

struct DenseShape {
  bool at, bt;   // A / B transposed
  DenseEpi epi;
};
int dense_parts(const DenseShape &s, const DenseArgs &a);  // parts of db_part / stats that a launch writes
// K splits worth taking (none of them empty)
int dense_splits(const DenseShape &s, const DenseArgs &a);
int dense_split_count(const DenseArgs &a);  // the splits that a launch with a.splits makes (none of them empty)
double dense_estimate(const DenseShape &s, const DenseArgs &a);  // us of a launch, about
hipError_t launch_dense(const DenseShape &s, const DenseArgs &a, hipStream_t st);
// Two weight gradients (both operands transposed, DENSE_STORE) in one launch, the one with more rows first;
// whether the plan takes that for faster than two.
hipError_t launch_dense_pair(const DenseArgs &a, const DenseArgs &b, hipStream_t st);
bool dense_pair_pays(const DenseArgs &a, const DenseArgs &b);

// DENSE_DGATE's epilogue as a kernel of its own, for gate, up and dh that come in K parts: gu [gu_parts][T][2 I]
// (+ bias), dh [dh_parts][T][I]; db_part [dense_dgate_parts(T)][2 I] or NULL.
struct DgateArgs {
  const float *gu, *bias, *dh;
  int gu_parts, dh_parts, T, I, planes;
  float limit;
  uint16_t *h, *dgu;  // [slots][T][I], [slots][T][2 I]
  uint32_t h_where, dgu_where;
  float *db_part;
};
constexpr int kDgateRows = 16;  // rows of a part
int dense_dgate_parts(int T);
hipError_t launch_dgate(const DgateArgs &a, hipStream_t s);

// scale: the largest magnitude of dloss [T] at tokens whose target lies in the vocabulary (the others' may
// be anything), 1 where that is 0 or not finite.
struct DlossScale {
  const float *dloss;
  const int32_t *targets;
  size_t T;
  int vocab;
  float *scale;
};
hipError_t launch_dloss_scale(const DlossScale &d, hipStream_t s);

// Work on rows in one launch.
enum DenseRowsWhat { ROWS_PLANES, ROWS_COPY, ROWS_PACK8, ROWS_UNPACK8, ROWS_SUM_BF16, ROWS_SUM_F32, ROWS_DLOSS_SCALE };
struct DenseRows {
  DenseRowsWhat what;
  const void *x;
  void *out;
  size_t n, cols;
  uint32_t where;
  int copies;
  unsigned blocks;
  const int32_t *targets;  // of rows of `cols`, or NULL: rows of negative ones as zeros
};
struct DenseRowJobs {
  unsigned end[4];  // set by the launch
  DenseRows d[4];
  DlossScale scale{};
  int count = 0;
  // x [n] f32 as kPlanes bf16 planes in the slots (n elements each) of `where`
  void planes(const float *x, uint16_t *out, uint32_t where, size_t n, const int32_t *targets = nullptr, size_t cols = 0);
  // bf16 values
  void copy(const uint16_t *x, uint16_t *out, size_t n, const int32_t *targets, size_t cols);
  // f32 values as a checkpoint; one as bf16 values, `copies` of them one behind the other (act8.hip's forms)
  void pack8(const float *x, size_t n, uint8_t *packed);
  void unpack8(const uint8_t *packed, size_t n, uint16_t *out, int copies);
  void column_sums(const void *x, bool bf16, size_t T, size_t H, float *out);  // dense_colsum_parts(T) == 1
  void dloss_scale(const DlossScale &s);  // few tokens
  size_t ends();  // sets `end`; the blocks of all
};
hipError_t launch_rows(DenseRowJobs a, hipStream_t s);

// out[i] = sum over parts of part[p * stride + i] (+ bias[i % n_bias]) for i < n, in order; bf16 or f32.
struct DenseSum {
  const float *part;
  size_t stride, n, n_bias;
  const float *bias;
  void *out;
  int parts;
  unsigned blocks;
  bool bf16, few;
};
// Up to 5 of them in one launch (those that a backward pass of the gated block can need).
struct DenseSums {
  unsigned end[5];  // set by the launch
  DenseSum d[5];
  int count = 0;
  void add(const float *part, size_t stride, int parts, size_t n, const float *bias, size_t n_bias, void *out, bool bf16);
  size_t ends();
};
hipError_t launch_sums(DenseSums a, hipStream_t s);
// Column sums of x [T][H] (f32 or bf16) into parts [dense_colsum_parts(T)][H].
constexpr size_t kColRows = 512;  // of a part
int dense_colsum_parts(size_t T);
hipError_t launch_colsum(const void *x, bool bf16, size_t T, size_t H, float *part, hipStream_t s);
// loss and log-sum-exp of each token from the parts of DENSE_STATS.
hipError_t launch_loss(const float2 *stats, int parts, const float *picked, const int32_t *targets, size_t T,
                       int vocab, float *loss, float *lse, hipStream_t s);

// MXFP8 activation checkpoints (act8.hip): codes [n][cols], then scales [n][cols / 32].
hipError_t launch_act8_pack(const void *x, bool bf16, size_t n, size_t cols, uint8_t *packed, hipStream_t s);
hipError_t launch_act8_unpack(const uint8_t *packed, size_t n, size_t cols, void *out, bool bf16, hipStream_t s);

// Device workspace of the dense operators: grows at need; a buffer that a captured graph may hold is
// kept until the context goes.
struct DenseWork {
  void *p = nullptr;
  size_t cap = 0;
  bool captured = false;  // used by a call under capture since it was allocated
  std::vector<void *> kept;
};

// What the dense operators need of a context (moe_api.cpp).
struct DenseCtx {
  hipStream_t stream;  // the context's
  size_t H;
  float clamp;
  const uint16_t *lm_w;  // bf16 LM head rows, NULL if none or f32
  size_t lm_vocab;
  DenseWork *work;
};

}  // namespace moe
