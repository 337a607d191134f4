// The page index: what it holds, and the append that keeps it with the K/V rows.
//
// For each (page, kv head) the index holds, over the page's keys, the largest and the smallest value
// of every dimension as int8 on a grid 2^e, e the smallest whole number in [-100, 100] with
// 127 * 2^e >= the largest magnitude; the largest are rounded up and the smallest down, so they stay
// bounds.  Powers of two are exact: floor and ceil onto a fine grid and then onto a coarser one give
// what they give onto the coarser one at once, so widening a page's bounds token by token gives the
// same bytes as computing them from all of its keys, in any order.
#pragma once

#include "sparse_common.h"

namespace rpa_sparse {
namespace {

constexpr int kExpMin = -100, kExpMax = 100;
constexpr float kFp8Max = 448.f;

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ void unpack8(u32x4 w, float x[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // e in [-126, 127]

// The smallest e in [kExpMin, kExpMax] with 127 * 2^e >= amax >= 0: 127 = 1.984375 * 2^6.
__device__ __forceinline__ int grid_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 6 + ((u & 0x7fffffu) > 0x7e0000u);
  return min(max(e, kExpMin), kExpMax);
}

// x on the grid 2^e, rounded up or down.  Products that underflow to zero keep their direction.
__device__ __forceinline__ int grid_up(float x, float inv) {
  const float y = ceilf(x * inv);
  const int r = (int)fminf(fmaxf(y, -127.f), 127.f);
  return x > 0.f && r < 1 ? 1 : r;
}
__device__ __forceinline__ int grid_down(float x, float inv) {
  const float y = floorf(x * inv);
  const int r = (int)fminf(fmaxf(y, -127.f), 127.f);
  return x < 0.f && r > -1 ? -1 : r;
}

// A pool value's fp8 code: x / scale, saturated (NaN stays NaN), to nearest even.
__device__ __forceinline__ float fp8_operand(float x, float scale) {
  const float y = x / scale;
  return y < -kFp8Max ? -kFp8Max : (y > kFp8Max ? kFp8Max : y);
}
__device__ __forceinline__ u32x2 fp8_codes(const float x[8], float scale) {
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int c = 0;
    c = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_operand(x[4 * i], scale), fp8_operand(x[4 * i + 1], scale), c, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_operand(x[4 * i + 2], scale), fp8_operand(x[4 * i + 3], scale), c, true);
    w[i] = (uint32_t)c;
  }
  return w;
}
__device__ __forceinline__ void fp8_values(u32x2 w, float scale, float x[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    x[4 * i] = a[0] * scale, x[4 * i + 1] = a[1] * scale, x[4 * i + 2] = b[0] * scale, x[4 * i + 3] = b[1] * scale;
  }
}

struct AppendParams {
  const uint16_t *k, *v;
  const int32_t* slots;
  uint8_t* kv;
  const float* scales;  // fp32 [P, Hkv, 2], or nullptr: the two below
  float k_scale, v_scale;
  int8_t *bounds, *exps;  // nullptr: no index
  long long k_token, k_head, v_token, v_head;  // strides, in values
  long long rows;                              // P * S
  int T, Hkv, D, S;
};

// One workgroup per token, one wave per kv head (each wave takes heads wave, wave + W, ...): the rows
// are copied (or quantised) 16 bytes a lane.  A token that is the first of its page's new rows -- row 0
// of a page, or a slot that does not follow the previous token's -- also widens the page's bounds by
// the whole run of consecutive slots, reading their keys once more (L2) with 64 / (D / 8) rows in
// flight per wave; decode rows are runs of one.  Runs of one page are the work of one wave, so no
// atomics and no order decide the result.
template <bool FP8>
__global__ __launch_bounds__(512) void append_kernel(AppendParams p) {
  const int lane = threadIdx.x % 64, t = blockIdx.x;
  const int slot = p.slots[t];
  if (slot == -1) return;
  if (slot < 0 || slot >= p.rows) {
    if (threadIdx.x == 0) flag_error(RPA_SPARSE_ERR_SLOT);
    return;
  }
  const int page = slot / p.S, row = slot % p.S;
  const int chunks = p.D / 8;
  int run = 0;  // new rows of this page from here on, 0: they belong to an earlier token's run
  if (p.bounds && (row == 0 || t == 0 || p.slots[t - 1] != slot - 1)) {
    const int most = min(p.S - row, p.T - t);
    run = most;
    for (int base = 1; base < most; base += 64) {
      const int i = base + lane;
      const unsigned long long end = __ballot(i >= most || p.slots[t + i] != slot + i);
      if (end) {
        run = base + __builtin_ctzll(end);
        break;
      }
    }
  }
  for (int h = threadIdx.x / 64; h < p.Hkv; h += blockDim.x / 64) {
    float scale[2] = {p.k_scale, p.v_scale};
    if (FP8 && p.scales) {
      const float* s = p.scales + ((size_t)page * p.Hkv + h) * 2;
      scale[0] = s[0], scale[1] = s[1];
    }
    for (int i = lane; i < 2 * chunks; i += 64) {
      const int part = i >= chunks, c = i - part * chunks;
      const uint16_t* src = part ? p.v + t * p.v_token + h * p.v_head : p.k + t * p.k_token + h * p.k_head;
      const u32x4 w = *(const u32x4*)(src + 8 * c);
      const size_t at = ((size_t)slot * (2 * p.Hkv) + 2 * h + part) * p.D + 8 * c;
      if (FP8) {
        float x[8];
        unpack8(w, x);
        *(u32x2*)(p.kv + at) = fp8_codes(x, part ? scale[1] : scale[0]);
      } else {
        *(u32x4*)(p.kv + 2 * at) = w;
      }
    }
    if (run == 0) continue;
    const int teams = 64 / chunks, team = lane / chunks, c = lane % chunks;
    float hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) hi[i] = -__builtin_inff(), lo[i] = __builtin_inff();
    if (team < teams) {
      const uint16_t* src = p.k + (t + team) * p.k_token + h * p.k_head + 8 * c;
#pragma unroll 4
      for (int r = team; r < run; r += teams, src += teams * p.k_token) {
        float x[8];
        unpack8(*(const u32x4*)src, x);
        if (FP8) fp8_values(fp8_codes(x, scale[0]), scale[0], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = x[i] == x[i] ? x[i] : 0.f;  // NaN counts as 0
          hi[i] = fmaxf(hi[i], y);
          lo[i] = fminf(lo[i], y);
        }
      }
    }
    float amax = 0.f;
    if (team < min(teams, run))
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
#pragma unroll
    for (int d = 32; d; d /= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
    for (int g = 1; g < min(teams, run); ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = fmaxf(hi[i], __shfl(hi[i], g * chunks + c));
        lo[i] = fminf(lo[i], __shfl(lo[i], g * chunks + c));
      }
    const size_t at = (size_t)page * p.Hkv + h;
    int e = grid_exponent(amax);
    const int old = row == 0 ? kExpMin : min(max((int)p.exps[at], kExpMin), kExpMax);
    e = max(e, old);
    if (lane < chunks) {
      int8_t* const up = p.bounds + at * 2 * p.D + 8 * c;
      int8_t* const down = up + p.D;
      u32x2 was_up = {0, 0}, was_down = {0, 0}, now_up, now_down;
      if (row) was_up = *(const u32x2*)up, was_down = *(const u32x2*)down;
      const float inv = pow2(-e);
      const int shift = min(e - old, 31);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int u = grid_up(hi[i], inv), d = grid_down(lo[i], inv);
        if (row) {
          const int pu = (int8_t)(was_up[i / 4] >> (8 * (i % 4))), pd = (int8_t)(was_down[i / 4] >> (8 * (i % 4)));
          u = max(u, -(-pu >> shift));
          d = min(d, pd >> shift);
        }
        const uint32_t ub = (uint32_t)(u & 255) << (8 * (i % 4)), db = (uint32_t)(d & 255) << (8 * (i % 4));
        if (i % 4 == 0) now_up[i / 4] = ub, now_down[i / 4] = db;
        else now_up[i / 4] |= ub, now_down[i / 4] |= db;
      }
      *(u32x2*)up = now_up;
      *(u32x2*)down = now_down;
    }
    if (lane == 0) p.exps[at] = (int8_t)e;
  }
}

int check_heads(int hkv, int d, int kv_dtype) {
  if (hkv <= 0) return fail(RPA_E_INVALID, "non-positive dimension in shape");
  if (kv_dtype != RPA_KV_BF16 && kv_dtype != RPA_KV_FP8_E4M3)
    return fail(RPA_E_INVALID, "kv_dtype must be RPA_KV_BF16 or RPA_KV_FP8_E4M3");
  const bool fp8 = kv_dtype == RPA_KV_FP8_E4M3;
  if (d != 256 && (d > 128 || d < (fp8 ? 64 : 32) || d % (fp8 ? 16 : 8)))
    return fail(RPA_E_UNSUPPORTED, "head_dim %d is not built (256, or a multiple of %d in [%d, 128])", d, fp8 ? 16 : 8,
                fp8 ? 64 : 32);
  return RPA_OK;
}

int check_pool(int pages, int page_size) {
  if (pages <= 0 || page_size <= 0) return fail(RPA_E_INVALID, "non-positive dimension in shape");
  if ((long long)pages * page_size > 0x7fffffffll) return fail(RPA_E_INVALID, "total_pages * page_size overflows int32");
  return RPA_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_strides(const char* name, const void* p, long long token, long long head) {
  if (!aligned16(p) || token % 8 || head % 8)
    return fail(RPA_E_INVALID, "%s must be 16-byte aligned with strides of a multiple of 8 values", name);
  return RPA_OK;
}

int check_append(const rpa_append_shape_t* s) {
  if (!s) return fail(RPA_E_INVALID, "shape is NULL");
  if (s->num_tokens < 0) return fail(RPA_E_INVALID, "negative num_tokens");
  const int rc = check_heads(s->num_kv_heads, s->head_dim, s->kv_dtype);
  return rc ? rc : check_pool(s->total_pages, s->page_size);
}

}  // namespace
}  // namespace rpa_sparse
