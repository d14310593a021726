// Checks and failures of the C entry points of the dense and of the grouped operators.
#pragma once

#include <stdarg.h>
#include <stdio.h>

#include "mmoe_dense.cuh"

namespace {

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return mmoe::record_failure(code, buf);
}

inline int cuda_fail(cudaError_t e, const char* what) { return fail(MMOE_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e)); }

// row and column indexes, rounded up to a tile, are 32-bit numbers
constexpr int32_t kMostTokens = 1 << 30, kMostChannels = 1 << 29;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
