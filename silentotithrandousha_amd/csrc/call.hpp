// What the host sources of the operators beside the path (dense_api.cpp, serve_api.cpp) share: failures, checks of
// arguments, and the context's workspace.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "../../include/moe_dense.h"
#include "dense.hpp"

namespace moe {

int api_fail(int code, const char *msg);
int dense_ctx(moe_ctx *c, DenseCtx *d);

inline int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return api_fail(code, buf);
}

// (a reported error is not left for the next launch, which would report it again as its own)
#define HIP_TRY(call)                                                                          \
  do {                                                                                         \
    hipError_t e_ = (call);                                                                    \
    if (e_ != hipSuccess) {                                                                    \
      (void)hipGetLastError();                                                                 \
      return fail(e_ == hipErrorOutOfMemory ? MOE_ERR_OOM : MOE_ERR_HIP, "%s: %s (%s:%d)",     \
                  #call, hipGetErrorString(e_), __FILE__, __LINE__);                           \
    }                                                                                          \
  } while (0)

#define RETURN_IF(rc)  \
  do {                 \
    int r_ = (rc);     \
    if (r_) return r_; \
  } while (0)

constexpr size_t kMaxTokens = (size_t)1 << 20;  // tokens per call, as the path-level calls
constexpr size_t kMaxInter = (size_t)1 << 20;   // columns
constexpr size_t kMaxVocab = (size_t)1 << 28;

inline size_t al(size_t v) { return (v + 255) / 256 * 256; }

// Parts of the workspace: sized first (base NULL), then placed.
struct Carve {
  char *base = nullptr;
  size_t off = 0;
  template <class T>
  T *take(size_t n) {
    T *p = base ? (T *)(base + off) : nullptr;
    off += al(n * sizeof(T));
    return p;
  }
};

// Grows the context's workspace to `bytes`, a second time and later with room above them (a quarter, at most 256 MB): the
// old one's release waits for the device, which lengths that rise by one would make every call do. A call under capture
// marks it: a graph may hold it.
inline int ensure(const DenseCtx &c, size_t bytes, hipStream_t s) {
  DenseWork &w = *c.work;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  HIP_TRY(hipStreamIsCapturing(s, &cap));
  const bool capturing = cap != hipStreamCaptureStatusNone;
  if (bytes > w.cap) {
    try {  // (room to keep the old one, before there is anything to undo)
      w.kept.reserve(w.kept.size() + 1);
    } catch (...) {
      return fail(MOE_ERR_OOM, "out of host memory");
    }
    if (capturing)
      return fail(MOE_ERR_STATE, "workspace too small for this call during graph capture; run it once uncaptured first");
    void *q = nullptr;
    size_t want = bytes + (w.p ? std::min(bytes / 4, (size_t)256 << 20) : 0);
    hipError_t e = hipMalloc(&q, want);
    if (e != hipSuccess && want > bytes) {
      (void)hipGetLastError();
      e = hipMalloc(&q, want = bytes);
    }
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return fail(MOE_ERR_OOM, "hipMalloc(%zu): %s", bytes, hipGetErrorString(e));
    }
    if (w.p && w.captured)
      w.kept.push_back(w.p);
    else if (w.p)
      (void)hipFree(w.p);  // waits for the launches that use it
    w.p = q;
    w.cap = want;
    w.captured = false;
  }
  w.captured |= capturing;
  return MOE_OK;
}

inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline size_t elem(int dtype) { return dtype == MOE_F32 ? 4 : 2; }

inline int check_dtype(int dtype) {
  if (dtype != MOE_F32 && dtype != MOE_BF16) return fail(MOE_ERR_INVALID, "dtype %d is neither MOE_F32 nor MOE_BF16", dtype);
  return MOE_OK;
}
// Pointers that matrix loads and stores of 16 bytes go through, or values one by one (4 bytes).
inline int check_aligned(std::initializer_list<const void *> ps, size_t bytes = 16) {
  for (const void *p : ps)
    if (!aligned(p, bytes)) return fail(MOE_ERR_INVALID, "device pointer %p is not %zu-byte aligned", p, bytes);
  return MOE_OK;
}
inline int check_tokens(size_t T) {
  if (T > kMaxTokens) return fail(MOE_ERR_INVALID, "n_tokens %zu above %zu", T, kMaxTokens);
  return MOE_OK;
}
// An output that is also an input, or twice an output.
inline int check_distinct(std::initializer_list<const void *> outs, std::initializer_list<const void *> ins) {
  for (auto o = outs.begin(); o != outs.end(); ++o) {
    if (!*o) continue;
    for (auto p = outs.begin(); p != o; ++p)
      if (*p == *o) return fail(MOE_ERR_INVALID, "two outputs at %p", *o);
    for (const void *i : ins)
      if (i == *o) return fail(MOE_ERR_INVALID, "an output is also an input (%p)", *o);
  }
  return MOE_OK;
}

}  // namespace moe
