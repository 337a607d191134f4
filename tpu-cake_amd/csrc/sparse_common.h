// Shared by the kernels of librpa_sparse: the device's error word, wave reductions, host errors.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "rpa_sparse.h"

namespace rpa_sparse {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// One word per device, set by kernels and read by rpa_sparse_read_error_word.  It is the library's
// own so that no call needs a workspace that two captured graphs could share.
__device__ int32_t g_error_word;

__device__ __forceinline__ void flag_error(int bits) { atomicOr(&g_error_word, bits); }

__device__ __forceinline__ int ceil_div(int a, int b) { return a / b + (a % b > 0); }

// ---- host side ----
// The message of the thread's last failure: a fixed buffer, so that reporting one cannot throw.
thread_local char g_last_error[256];

__attribute__((format(printf, 2, 3))) int fail(int code, const char* format, ...) {
  va_list args;
  va_start(args, format);
  vsnprintf(g_last_error, sizeof g_last_error, format, args);
  va_end(args);
  return code;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(RPA_E_HIP, "%s: %s", what, hipGetErrorString(e));
  return RPA_OK;
}

}  // namespace
}  // namespace rpa_sparse
