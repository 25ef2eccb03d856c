// Activation checkpoints in 8 bits (MXFP8): e4m3 codes with one power-of-two scale per 32 values.
//
// e: the smallest exponent (at least -127) with max |x| <= 448 * 2^e, so that nothing saturates and
// every code is within half a step of its value: 2^-4 relative in e4m3's normal range, 2^(e - 10)
// below it. Scale byte e + 127. A block that holds a value that is not finite has scale byte 255 and
// reads back as NaN. A code times its scale has 4 significant bits: exact in bf16.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "act8.hpp"
#include "dense.hpp"
#include "kernels.hpp"

namespace moe {
namespace {

// Four lanes a block of 32 values (which leave together); bound by the bytes read and written: 4096 x 2880 f32 packed in 10.6 us
// (5.6 TB/s) and unpacked in 12.8 (4.6).
template <class S>
__global__ __launch_bounds__(256) void k_act8_pack(const S *x, size_t blocks, uint8_t *codes, uint8_t *scales) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i / 4 < blocks; i += (size_t)gridDim.x * 256) act8_pack8(x, i, codes, scales);
}

template <class D>
__global__ __launch_bounds__(256) void k_act8_unpack(const uint8_t *codes, const uint8_t *scales, size_t blocks, D *out) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i / 4 < blocks; i += (size_t)gridDim.x * 256) act8_unpack8(codes, scales, i, blocks, out, 1);
}

// (a launch has less than 2^32 threads: of 2^34 values and more each takes several)
unsigned grid_for(size_t blocks) { return (unsigned)std::min<size_t>((blocks * 4 + 255) / 256, (size_t)1 << 23); }

}  // namespace

hipError_t launch_act8_pack(const void *x, bool bf16, size_t n, size_t cols, uint8_t *packed, hipStream_t s) {
  const size_t blocks = n * cols / 32;
  if (!blocks) return hipSuccess;
  if (cols % 32) return hipErrorInvalidValue;
  uint8_t *scales = packed + n * cols;
  return bf16 ? launch_own(k_act8_pack<uint16_t>, grid_for(blocks), 256, 0, s, (const uint16_t *)x, blocks, packed, scales)
              : launch_own(k_act8_pack<float>, grid_for(blocks), 256, 0, s, (const float *)x, blocks, packed, scales);
}

hipError_t launch_act8_unpack(const uint8_t *packed, size_t n, size_t cols, void *out, bool bf16, hipStream_t s) {
  const size_t blocks = n * cols / 32;
  if (!blocks) return hipSuccess;
  if (cols % 32) return hipErrorInvalidValue;
  const uint8_t *scales = packed + n * cols;
  return bf16 ? launch_own(k_act8_unpack<uint16_t>, grid_for(blocks), 256, 0, s, packed, scales, blocks, (uint16_t *)out)
              : launch_own(k_act8_unpack<float>, grid_for(blocks), 256, 0, s, packed, scales, blocks, (float *)out);
}

}  // namespace moe
