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

constexpr int kAppendTokens = 8, kAppendLong = 2048;  // tokens of a workgroup, in batches longer than that
constexpr int kAppendRounds = 4;

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
  int wide;  // workgroups that widen bounds
  uint32_t chunk_magic, row_magic;  // ceil(2^32 / n) for n = D / 8 and 2 D / 8: i / n for i < 2^26
};

// Copies, or quantises, the rows of TOKENS tokens, a wave one kv head of them at a time (heads wave, wave + W,
// ...), 16 bytes a lane with four loads in flight.  K and V do not wait for the slots.
template <bool FP8, int TOKENS>
__device__ __forceinline__ void copy_rows(const AppendParams& p, int t0) {
  const int lane = threadIdx.x % 64;
  const int chunks = p.D / 8, row_chunks = 2 * chunks;
  const int items = min(TOKENS, p.T - t0) * row_chunks;
  const int wave = threadIdx.x / 64, waves = blockDim.x / 64;
  constexpr int kHold = 4;
  u32x4 w[kHold];
  const auto load = [&](int h, int base) {
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      const int idx = min(base + 64 * u + lane, items - 1);
      const int i = __umulhi((uint32_t)idx, p.row_magic), c = idx - i * row_chunks, part = c >= chunks;
      const uint16_t* src = part ? p.v + (t0 + i) * p.v_token + h * p.v_head : p.k + (t0 + i) * p.k_token + h * p.k_head;
      w[u] = *(const u32x4*)(src + 8 * (c - part * chunks));
    }
  };
  load(wave, 0);
  const int mine = lane < TOKENS && t0 + lane < p.T ? p.slots[t0 + lane] : -1;
  if (wave == 0 && mine != -1 && (mine < 0 || mine >= p.rows)) flag_error(RPA_SPARSE_ERR_SLOT);
#pragma unroll 1
  for (int h = wave; h < p.Hkv; h += waves) {
#pragma unroll 1
    for (int base = 0; base < items; base += 64 * kHold) {
      if (h != wave || base) load(h, base);
      int slot[kHold];
      float scale[kHold];
#pragma unroll
      for (int u = 0; u < kHold; ++u) {
        const int idx = min(base + 64 * u + lane, items - 1);
        const int i = __umulhi((uint32_t)idx, p.row_magic), part = idx - i * row_chunks >= chunks;
        slot[u] = __shfl(mine, i);
        if (slot[u] < 0 || slot[u] >= p.rows || base + 64 * u + lane >= items) slot[u] = -1;
        scale[u] = part ? p.v_scale : p.k_scale;
        if (FP8 && p.scales) scale[u] = p.scales[((size_t)(max(slot[u], 0) / p.S) * p.Hkv + h) * 2 + part];
      }
#pragma unroll
      for (int u = 0; u < kHold; ++u) {
        if (slot[u] < 0) continue;
        const int idx = base + 64 * u + lane;
        const int i = __umulhi((uint32_t)idx, p.row_magic), c = idx - i * row_chunks, part = c >= chunks;
        const size_t at = ((size_t)slot[u] * (2 * p.Hkv) + 2 * h + part) * p.D + 8 * (c - part * chunks);
        if (FP8) {
          float x[8];
          unpack8(w[u], x);
          *(u32x2*)(p.kv + at) = fp8_codes(x, scale[u]);
        } else {
          *(u32x4*)(p.kv + 2 * at) = w[u];
        }
      }
    }
  }
}

// One run of new rows -- `run` tokens from t on, from `row` of `page` on -- for all teams of a wave (alone: the
// same one, each a share of its rows), or one a team (run 0: none).
template <bool FP8>
__device__ __forceinline__ void widen_runs(const AppendParams& p, int t, int page, int row, int run, bool alone, int team,
                                           int teams, int c) {
  const int chunks = p.D / 8;
  const int step = alone ? min(teams, run) : min(run, 1), from = alone ? team : 0;
  const bool merges = run > 0 && (!alone || team == 0);
  for (int h = threadIdx.x / 64; h < p.Hkv; h += blockDim.x / 64) {
    const size_t at = (size_t)(run ? page : 0) * p.Hkv + h;  // without a run the page may be any number
    int8_t* const up = p.bounds + at * 2 * p.D + 8 * c;
    int8_t* const down = up + p.D;
    u32x2 was_up = {0, 0}, was_down = {0, 0};
    int old = kExpMin;
    if (merges && row) {  // a page begun earlier
      old = min(max((int)p.exps[at], kExpMin), kExpMax);
      was_up = *(const u32x2*)up, was_down = *(const u32x2*)down;
    }
    const float scale = FP8 ? (p.scales ? p.scales[2 * at] : p.k_scale) : 1.f;
    float hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) hi[i] = -__builtin_inff(), lo[i] = __builtin_inff();
    if (from < step) {
      const uint16_t* src = p.k + (t + from) * p.k_token + h * p.k_head + 8 * c;
#pragma unroll 2  // four rows in flight take 17 registers more, and 26 us where two take 25
      for (int r = from; r < run; r += step, src += step * p.k_token) {
        float x[8];
        unpack8(*(const u32x4*)src, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = x[i] == x[i] ? x[i] : 0.f;  // NaN counts as 0
          hi[i] = fmaxf(hi[i], y);
          lo[i] = fminf(lo[i], y);
        }
      }
    }
    if (alone)
      for (int g = 1; g < step; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          hi[i] = fmaxf(hi[i], __shfl(hi[i], g * chunks + c));
          lo[i] = fminf(lo[i], __shfl(lo[i], g * chunks + c));
        }
    if (FP8) {
      fp8_values(fp8_codes(hi, scale), scale, hi);
      fp8_values(fp8_codes(lo, scale), scale, lo);
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // a scale of 0 or none that is a number: 0, as other NaN
        hi[i] = hi[i] == hi[i] ? hi[i] : 0.f;
        lo[i] = lo[i] == lo[i] ? lo[i] : 0.f;
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
    float most = amax;
    for (int i = 1; i < chunks; ++i) most = fmaxf(most, __shfl(amax, min(team * chunks + (c + i < chunks ? c + i : c + i - chunks), 63)));
    const int e = max(grid_exponent(most), old);
    if (merges) {
      const float inv = pow2(-e);
      const int shift = min(e - old, 31);
      u32x2 now_up = {0, 0}, now_down = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int u = grid_up(hi[i], inv), d = grid_down(lo[i], inv);
        const int pu = (int8_t)(was_up[i / 4] >> (8 * (i % 4))), pd = (int8_t)(was_down[i / 4] >> (8 * (i % 4)));
        u = row ? max(u, -(-pu >> shift)) : u;
        d = row ? min(d, pd >> shift) : d;
        now_up[i / 4] |= (uint32_t)(u & 255) << (8 * (i % 4));
        now_down[i / 4] |= (uint32_t)(d & 255) << (8 * (i % 4));
      }
      *(u32x2*)up = now_up;
      *(u32x2*)down = now_down;
      if (c == 0) p.exps[at] = (int8_t)e;
    }
  }
}

// Widens the bounds of the pages that `count` tokens from t0 on are the first new rows of: row 0 of a page, or
// a slot that does not follow the previous token's.  Such a token stands for its whole run of consecutive slots
// in the page, and a run is the work of one wave, so no atomics and no order decide the result.  A wave takes a
// kv head; its teams of D / 8 lanes take a run each, or, where there is one only (prompts), every so manieth of
// its rows.  Quantising is monotone: the bounds of an fp8 page come from the largest and smallest inputs,
// quantised.
template <bool FP8>
__device__ __forceinline__ void widen_bounds(const AppendParams& p, int t0, int count) {
  const int lane = threadIdx.x % 64, chunks = p.D / 8;
  const int team = __umulhi((uint32_t)lane, p.chunk_magic), c = lane - team * chunks;
  const int teams = __umulhi(64u, p.chunk_magic);
  // the slots from here on, a lane each
  const int mine = t0 + lane < p.T ? p.slots[t0 + lane] : -2;
  const int left = t0 > 0 ? p.slots[t0 - 1] : -2;
  const int before = __shfl_up(mine, 1), prev = lane ? before : left;
  const unsigned long long leads =
      __ballot(lane < count && mine >= 0 && mine < p.rows && (mine % p.S == 0 || prev != mine - 1));
  if (leads == 0) return;
  // each slot's run as far as the slots at hand go: rows of its page at consecutive slots
  const int after = __shfl_down(mine, 1);
  const bool joins = lane < 63 && after == mine + 1 && after % p.S != 0;
  const unsigned long long breaks = ~__ballot(joins) >> lane;  // bit i: slot lane + i is the last of its run
  const int length = breaks ? 1 + __builtin_ctzll(breaks) : 64;
  const bool is_lead = leads >> lane & 1;
  // short runs: a team each; long ones: one after another, all teams on each
  const bool apart = __ballot(is_lead && (length > 16 || lane + length > 63)) == 0 && (leads & (leads - 1));
  for (unsigned long long todo = leads; todo; todo = apart ? 0 : todo & (todo - 1)) {
    const int first = apart ? min(team, count - 1) : __builtin_ctzll(todo), t = t0 + first;
    const bool lead = team < teams && (!apart || (team < count && (leads >> first & 1)));
    const int slot = max(__shfl(mine, first), 0), row = slot % p.S, most = min(p.S - row, p.T - t);
    int run = __shfl(length, first);
    if (!apart && first + run > 63)  // further than the slots at hand
      for (run = 64 - first; run < most; run += 64) {
        const int i = run + lane;
        const unsigned long long end = __ballot(i >= most || p.slots[t + i] != slot + i);
        if (end) {
          run += __builtin_ctzll(end);
          break;
        }
      }
    widen_runs<FP8>(p, t, slot / p.S, row, lead ? min(run, most) : 0, !apart, team, teams, c);
  }
}

// One launch: the first `wide` workgroups (with an index) widen bounds, the others copy rows beside them.  Decode
// batches are bound by latency: a token a workgroup, or a team.  Long batches are bound by the turnover of
// workgroups and by runs that start late: eight tokens, and four rounds of teams first.  64 decode tokens of 8 heads
// of 128 take 5.3 us (launch and two round trips); 9 000 prompt tokens into an fp8 pool, 55 MB, 24.6 us or 2.2 TB/s, into
// a bf16 pool, 74 MB, 21.3 us or 3.5 TB/s.  K is read twice, by the workgroups that copy and by those that widen: 54 MB are
// fetched where 37 would do.
template <bool FP8, int TOKENS>
__global__ __launch_bounds__(512) void append_kernel(AppendParams p) {
  const int block = blockIdx.x, teams = __umulhi(64u, p.chunk_magic);
  if (block < p.wide) {
    constexpr int kRounds = TOKENS > 1 ? kAppendRounds : 1;
    for (int r = 0; r < kRounds; ++r) {
      const int t0 = (block * kRounds + r) * teams;
      if (t0 < p.T) widen_bounds<FP8>(p, t0, min(teams, p.T - t0));
    }
  } else {
    copy_rows<FP8, TOKENS>(p, (block - p.wide) * TOKENS);
  }
}


int check_heads(int hkv, int d, int kv_dtype) {
  if (hkv <= 0) return fail(RPA_E_INVALID, "non-positive dimension in shape");
  if (hkv > 65535) return fail(RPA_E_UNSUPPORTED, "more than 65535 kv heads");  // a launch's y dimension, 32-bit rows
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
  if (s->num_tokens >= 1 << 30) return fail(RPA_E_INVALID, "num_tokens must be below 2^30");
  const int rc = check_heads(s->num_kv_heads, s->head_dim, s->kv_dtype);
  return rc ? rc : check_pool(s->total_pages, s->page_size);
}

}  // namespace
}  // namespace rpa_sparse
