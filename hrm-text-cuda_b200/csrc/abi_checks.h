// Argument checks shared by the extern "C" entry points.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/hrm_ops.h"

namespace {

inline int cuda_status(cudaError_t e) { return e == cudaSuccess ? HRM_OK : HRM_ERR_CUDA + (int)e; }

// n * m for non-negative operands, or -1 when it would exceed limit.
inline int64_t mul_checked(int64_t n, int64_t m, int64_t limit = INT64_MAX / 8) {
  if (n < 0 || m < 0) return -1;
  if (n != 0 && m > limit / n) return -1;
  return n * m;
}

// True when [a, a + abytes) and [b, b + bbytes) share a byte.
inline bool overlap(const void* a, int64_t abytes, const void* b, int64_t bbytes) {
  if (a == nullptr || b == nullptr || abytes <= 0 || bbytes <= 0) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  return pa < pb + (uintptr_t)bbytes && pb < pa + (uintptr_t)abytes;
}

// Partial overlap (anything but identical ranges) of two equal-sized buffers.
inline bool partial_overlap(const void* a, const void* b, int64_t bytes) { return a != b && overlap(a, bytes, b, bytes); }

inline cudaStream_t as_cuda(hrm_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace
