// Tile shapes of the dense products and the rules that pick one, their K parts and what a launch accepts: host code
// that needs no device (dense_plan.cpp).
#pragma once
#include "dense.hpp"

namespace moe {

constexpr int kDenseStep = 64;  // k values per step
constexpr int kDenseHalf = 32;  // and per half, an MFMA's

// X(rows, columns, wavefronts along each, LDS slots, B's planes, workgroups of a CU, TFLOP/s of the device
// full of them, planes counted). The rates are those of 2880 k values (loss over 201088 rows, 512 tokens and
// more), with planes those of 2048 (loss of 100 and 333 rows over 50257).
#define MOE_DENSE_TILES(X)            \
  X(288, 256, 2, 4, 2, 1, 1, 1180.0)  \
  X(256, 256, 2, 4, 2, 1, 1, 1290.0)  \
  X(192, 256, 2, 4, 2, 1, 1, 1190.0)  \
  X(128, 128, 2, 2, 2, 1, 2, 1000.0)  \
  X(128, 64, 2, 2, 3, 1, 2, 800.0)    \
  X(64, 64, 2, 2, 4, 1, 2, 600.0)     \
  X(32, 64, 2, 2, 6, 1, 2, 430.0)     \
  X(32, 32, 2, 2, 8, 1, 2, 300.0)     \
  X(32, 16, 2, 1, 8, 1, 3, 220.0)     \
  X(128, 16, 4, 1, 4, 1, 2, 220.0)    \
  X(64, 16, 4, 1, 8, 1, 2, 210.0)     \
  X(16, 16, 1, 1, 16, 1, 2, 110.0)    \
  X(256, 128, 4, 2, 2, 3, 1, 1280.0)  \
  X(128, 64, 2, 2, 2, 3, 2, 1200.0)   \
  X(64, 64, 2, 2, 2, 3, 2, 980.0)     \
  X(64, 32, 2, 2, 4, 3, 2, 780.0)     \
  X(32, 32, 2, 2, 5, 3, 2, 480.0)

struct DenseTileDims {
  int bm, bn, wm, wn, ns, planes, wgs;
  double rate;
};
constexpr DenseTileDims kDenseTiles[] = {
#define X(bm, bn, wm, wn, ns, planes, wgs, rate) {bm, bn, wm, wn, ns, planes, wgs, rate},
    MOE_DENSE_TILES(X)
#undef X
};
constexpr int kDenseTileCount = sizeof(kDenseTiles) / sizeof(kDenseTiles[0]);

int dense_tile(const DenseShape &s, const DenseArgs &a);  // index of the tile that the plan takes
// tile of two weight gradients in one launch, and its estimated us
int dense_pair_tile(const DenseArgs &a, const DenseArgs &b, double &us);
// rows of A that a workgroup of the register kernel takes (dense_few.hip), 0 where it does not take the product
int dense_few_rows(const DenseShape &s, const DenseArgs &a);
// Checks what the kernels assume of a product and sets its K parts.
hipError_t dense_prepare(const DenseShape &s, DenseArgs &a);
hipError_t dense_prepare_pair(DenseArgs &a, DenseArgs &b);

}  // namespace moe
