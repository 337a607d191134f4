// Eviction: which rows of a sequence each kv head keeps, and the moves that bring them together.
//
// Mathematics: a row's key is its weight as an unsigned whole number of the same order (0 for NaN), the largest of all for
// rows that stay in any case.  The budget-th largest key of a (sequence, head) is found digit by digit: counts of the
// next eight bits over the rows that share the bits so far, four times.  Rows above it stay, and of the rows at it
// the lowest ones, as many as fit.  Kept rows at or past `budget` and rows below it that go are equally many: the i-th of the
// one take the places of the i-th of the other.  Counts are whole numbers, so nothing depends on an order.
//
// A cache's rows are in no order for attention, so only what lies past the budget is moved, not everything behind the
// first gap; the ledger's positions tell the recent rows.  Moves read past the budget and write before it: they
// do not meet, and a list that is applied twice gives the same.
#pragma once

#include "attend_kernels.h"

namespace rpa_sparse {
namespace {

struct ChooseParams {
  const float* weights;
  const int32_t *positions, *kv_lens, *table, *num_seqs, *dropped;
  int32_t* moves;
  int N, PPS, Hkv, P, S, budget, limit, sinks, recent, M;
};

// The order of weights as whole numbers, 0 for NaN; zeros of both signs are equal.
__device__ __forceinline__ uint32_t weight_key(float w) { return w == w ? ordered(w + 0.f) : 0u; }

constexpr int kChooseThreads = 1024;

// One workgroup a (kv head, sequence).
__global__ __launch_bounds__(kChooseThreads) void choose_rows_kernel(ChooseParams p) {
  constexpr int kWaves = kChooseThreads / 64;
  __shared__ uint32_t s_count[256];
  __shared__ Pair s_scan[kWaves];
  __shared__ uint32_t s_found[2];
  const int tid = threadIdx.x;
  const int h = blockIdx.x % p.Hkv, seq = blockIdx.x / p.Hkv;
  int32_t* const list = p.moves + ((size_t)seq * p.Hkv + h) * p.M * 2;
  const long long capacity = (long long)p.PPS * p.S;
  int n = seq < *p.num_seqs ? p.kv_lens[seq] : 0;
  const long long end = (long long)n + (p.dropped ? p.dropped[seq] : 0);
  if (n > capacity) {
    if (tid == 0) flag_error(RPA_SPARSE_ERR_LEN);
    n = (int)capacity;
  }
  int done = 0;  // entries of the list
  if (n > p.limit && n > p.budget) {  // uniform
    const int32_t* const table = p.table + (size_t)seq * p.PPS;
    const auto slot_of = [&](int row) {  // -1: no such page
      const int page = table[row / p.S];
      return page >= 0 && page < p.P ? page * p.S + row % p.S : -1;
    };
    const auto key_of = [&](int row) {
      const int slot = slot_of(row);
      if (slot < 0) {
        flag_error(RPA_SPARSE_ERR_PAGE);
        return 0u;
      }
      const size_t at = ((size_t)(slot / p.S) * p.Hkv + h) * p.S + slot % p.S;
      const int position = p.positions[at];
      return position < p.sinks || position >= end - p.recent ? 0xffffffffu : weight_key(p.weights[at]);
    };
    uint32_t prefix = 0, rank = p.budget;  // the rank-th largest of the keys that begin with prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kChooseThreads) s_count[i] = 0;
      __syncthreads();
      for (int row = tid; row < n; row += kChooseThreads) {
        const uint32_t key = key_of(row);
        if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&s_count[key >> shift & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t above = 0;
        int d = 255;
        while (d > 0 && above + s_count[d] < rank) above += s_count[d--];
        s_found[0] = prefix << 8 | d, s_found[1] = rank - above;
      }
      __syncthreads();
      prefix = s_found[0], rank = s_found[1];
    }
    // rank: how many of the rows at this very key stay
    uint32_t equal = 0, late = 0, holes = 0;
    for (int base = 0; base < n; base += kChooseThreads) {
      const int row = base + tid;
      const uint32_t key = row < n ? key_of(row) : 0u;
      const bool same = row < n && key == prefix;
      Pair total;
      Pair before = scan_pairs<kWaves>({same, 0}, total, s_scan);
      const bool kept = row < n && (key > prefix || (same && equal + before.a < rank));
      equal += total.a;
      const bool comes = kept && row >= p.budget, goes = row < n && !kept && row < p.budget;
      before = scan_pairs<kWaves>({comes, goes}, total, s_scan);
      if (comes && late + before.a < (uint32_t)p.M) list[2 * (late + before.a) + 1] = slot_of(row);
      if (goes && holes + before.b < (uint32_t)p.M) list[2 * (holes + before.b)] = slot_of(row);
      late += total.a, holes += total.b;
    }
    if (late > (uint32_t)p.M && tid == 0) flag_error(RPA_SPARSE_ERR_LEN);
    done = (int)min(late, (uint32_t)p.M);
  }
  for (long long i = 2ll * done + tid; i < 2ll * p.M; i += kChooseThreads) list[i] = -1;
}

struct MoveParams {
  const int32_t* moves;
  const float* scales;
  uint8_t* kv;
  float* weights;
  int32_t* positions;
  long long entries, rows;  // of all lists; P * S
  int M, Hkv, D, S, chunks;  // chunks: 16 bytes each, of a head's key and value row
};

// A wave takes entries of the lists, its lanes 16 bytes of a head's key and value row, which lie together.
template <bool FP8>
__global__ __launch_bounds__(256) void move_kernel(MoveParams p) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const long long entry = (long long)blockIdx.x * 4 + wave;
  if (entry >= p.entries) return;
  const int h = (int)(entry / p.M % p.Hkv);
  const int to = p.moves[2 * entry], from = p.moves[2 * entry + 1];
  if (to < 0 || from < 0) return;
  if (to >= p.rows || from >= p.rows) {
    if (lane == 0) flag_error(RPA_SPARSE_ERR_SLOT);
    return;
  }
  const size_t row_bytes = 16ull * p.chunks;
  const uint8_t* const src = p.kv + ((size_t)from * p.Hkv + h) * row_bytes;
  uint8_t* const dst = p.kv + ((size_t)to * p.Hkv + h) * row_bytes;
  const size_t head_from = (size_t)(from / p.S) * p.Hkv + h, head_to = (size_t)(to / p.S) * p.Hkv + h;
  for (int c = lane; c < p.chunks; c += 64) {
    u32x4 w = *(const u32x4*)(src + 16 * c);
    if (FP8 && p.scales) {
      const int part = 2 * c >= p.chunks;
      const float there = p.scales[2 * head_from + part], here = p.scales[2 * head_to + part];
      if (there != here) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          fp8_values(u32x2{w[2 * i], w[2 * i + 1]}, there, x);
          const u32x2 codes = fp8_codes(x, here);
          w[2 * i] = codes[0], w[2 * i + 1] = codes[1];
        }
      }
    }
    *(u32x4*)(dst + 16 * c) = w;
  }
  if (lane == 0) {
    const size_t a = head_from * p.S + from % p.S, b = head_to * p.S + to % p.S;
    p.weights[b] = p.weights[a];
    p.positions[b] = p.positions[a];
  }
}

// ---- host side ----
int check_choose(const rpa_choose_shape_t* s) {
  if (!s) return fail(RPA_E_INVALID, "shape is NULL");
  if (s->max_num_seqs <= 0 || s->pages_per_seq <= 0 || s->num_kv_heads <= 0 || s->max_moves <= 0)
    return fail(RPA_E_INVALID, "non-positive dimension in shape");
  if (s->num_kv_heads > 65535) return fail(RPA_E_UNSUPPORTED, "more than 65535 kv heads");
  int rc = check_pool(s->total_pages, s->page_size);
  if (rc) return rc;
  if ((long long)s->pages_per_seq * s->page_size > kMostIndex)
    return fail(RPA_E_INVALID, "pages_per_seq * page_size must be at most 2^31 - 2^16 - 1");
  if (s->budget < 1 || s->limit < s->budget) return fail(RPA_E_INVALID, "budget must be positive and limit at least budget");
  if (s->sinks < 0 || s->recent < 0 || (long long)s->sinks + s->recent > s->budget)
    return fail(RPA_E_INVALID, "sinks and recent must not be negative nor more than the budget together");
  if (s->max_moves >= 1 << 30) return fail(RPA_E_INVALID, "max_moves must be below 2^30");
  return check_launch((long long)s->max_num_seqs * s->num_kv_heads, kChooseThreads);
}

int check_move(const rpa_move_shape_t* s) {
  if (!s) return fail(RPA_E_INVALID, "shape is NULL");
  if (s->num_lists < 0 || s->max_moves <= 0) return fail(RPA_E_INVALID, "non-positive dimension in shape");
  int rc = check_heads(s->num_kv_heads, s->head_dim, s->kv_dtype);
  if (rc || (rc = check_pool(s->total_pages, s->page_size))) return rc;
  const __int128 entries = (__int128)s->num_lists * s->num_kv_heads * s->max_moves;
  if (entries > 4 * (kMostThreads / 256)) return fail(RPA_E_UNSUPPORTED, "more rows than one launch takes");
  return RPA_OK;
}

}  // namespace
}  // namespace rpa_sparse
