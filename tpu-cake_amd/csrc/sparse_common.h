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

// Takes back the bits that a caller has read; other streams' kernels may set others meanwhile.
__global__ void clear_error_kernel(int bits) { atomicAnd(&g_error_word, ~bits); }

__device__ __forceinline__ int ceil_div(int a, int b) { return a / b + (a % b > 0); }

constexpr uint32_t kSumCap = 1u << 30;  // sums saturate here: limits (pages, tokens) are below this

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;  // a, b <= 2^30
  return s < kSumCap ? s : kSumCap;
}

struct Pair {
  uint32_t a, b;
};

// Exclusive sums of a pair over the workgroup's threads, and the workgroup's totals.  Saturating
// addition of non-negative numbers is associative, so any order gives the same.
template <int WAVES>
__device__ __forceinline__ Pair scan_pairs(Pair v, Pair& total, Pair (*lds)) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  Pair inc = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t a = __shfl_up(inc.a, d), b = __shfl_up(inc.b, d);
    if (lane >= d) inc = {sat_add(inc.a, a), sat_add(inc.b, b)};
  }
  __syncthreads();  // the last use of lds
  if (lane == 63) lds[wave] = inc;
  __syncthreads();
  Pair before = {0, 0};
  total = {0, 0};
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const Pair t = lds[w];
    if (w == wave) before = total;
    total = {sat_add(total.a, t.a), sat_add(total.b, t.b)};
  }
  Pair up = {__shfl_up(inc.a, 1), __shfl_up(inc.b, 1)};
  if (lane == 0) up = {0, 0};
  return {sat_add(before.a, up.a), sat_add(before.b, up.b)};
}

// A wave's LDS accesses execute in order; this keeps the compiler from reordering them.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float swap_max(float v) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float swap_sum(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The largest of a value over the wave.
__device__ __forceinline__ float wave_max(float v) {
  const auto step = [&](auto dpp) {
    v = fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(v), __float_as_uint(v), dpp(), 0xf, 0xf, false)));
  };
  step([] { return 0xB1; });   // quad_perm 1 0 3 2
  step([] { return 0x4E; });   // quad_perm 2 3 0 1
  step([] { return 0x141; });  // row_half_mirror
  step([] { return 0x140; });  // row_mirror
  return swap_max(v);
}

// ---- host side ----
// The most entries of what a kernel's loop walks in 32 bits: an index steps by less than 2^16.
constexpr int kMostIndex = 0x7fffffff - 0x10000;

// The message of the thread's last failure: a fixed buffer, so that reporting one cannot throw.
thread_local char g_last_error[256];

__attribute__((format(printf, 2, 3))) int fail(int code, const char* format, ...) {
  va_list args;
  va_start(args, format);
  vsnprintf(g_last_error, sizeof g_last_error, format, args);
  va_end(args);
  return code;
}

// HIP launches fewer than 2^32 threads along a dimension.
constexpr long long kMostThreads = (1ll << 32) - 1;

int check_launch(long long groups, int threads) {
  if (groups > kMostThreads / threads) return fail(RPA_E_UNSUPPORTED, "more rows than one launch takes");
  return RPA_OK;
}

// Memory of a call: `outer` blocks, `step` bytes apart, of `bytes` each.
struct Memory {
  const char* name;
  const void* at;
  long long bytes, outer = 1, step = 0;
};

// Rows [tokens, heads, dim] of 16 bits; strides in values.  Blocks are what lies within the larger stride.
Memory rows_of(const char* name, const void* at, long long tokens, long long heads, long long dim, long long token, long long head) {
  const bool by_token = token >= head;
  const long long inner = by_token ? (heads - 1) * head : (tokens - 1) * token;
  return {name, at, 2 * (inner + dim), by_token ? tokens : heads, 2 * (by_token ? token : head)};
}

bool meets(const Memory& a, const Memory& out) {  // out: one block
  if (!a.at || !out.at || a.bytes <= 0 || out.bytes <= 0) return false;
  const long long from = (long long)((uintptr_t)out.at - (uintptr_t)a.at);  // of out, from a's first byte on
  // the first block that ends behind out's first byte
  const long long k = from < a.bytes ? 0 : a.step > 0 ? (from - a.bytes) / a.step + 1 : a.outer;
  return k < a.outer && k * a.step < from + out.bytes;
}

// Workgroups run in no order: what a call writes must not lie in what it reads, nor in another output.
template <int N>
int check_separate(const Memory& out, const Memory (&others)[N]) {
  for (const Memory& m : others)
    if (meets(m, out)) return fail(RPA_E_INVALID, "%s overlaps %s: outputs need memory of their own", out.name, m.name);
  return RPA_OK;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(RPA_E_HIP, "%s: %s", what, hipGetErrorString(e));
  return RPA_OK;
}

}  // namespace
}  // namespace rpa_sparse
