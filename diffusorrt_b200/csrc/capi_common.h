// Errors of the C ABI, shared by its translation units: a failing call records its text for
// drt_last_error() of the calling thread and returns its status.
#pragma once
#include <cuda_runtime.h>

#include "../../include/diffusorrt_b200.h"

namespace drt {
int set_error(int code, const char* fmt, ...) __attribute__((visibility("hidden")));
}  // namespace drt

#define CK(expr)                                                                                         \
  do {                                                                                                   \
    cudaError_t _e = (expr);                                                                             \
    if (_e != cudaSuccess)                                                                               \
      return set_error(DRT_INTERNAL_ERROR, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(_e), __FILE__, \
                       __LINE__);                                                                        \
  } while (0)
#define TRY(expr)                 \
  do {                            \
    int _r = (expr);              \
    if (_r != DRT_OK) return _r;  \
  } while (0)
#define REQUIRE(cond, ...)                                     \
  do {                                                         \
    if (!(cond)) return set_error(DRT_INVALID_ARGUMENT, __VA_ARGS__); \
  } while (0)
