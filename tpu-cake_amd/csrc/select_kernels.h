// The choice of pages: for each (token, kv head) the pages whose keys can score highest.
//
// Mathematics: the group's queries are rounded to int8 on a grid 2^f they share (f as the index's
// exponents), qh.  A key x of page p has q . x <= sum_d max(q_d hi_d, q_d lo_d), so with the index's
// int8 bounds the score is
//     s(p) = 2^e(p) max_g sum_d max(qh_gd hi_d, qh_gd lo_d) = 2^e(p) max_g ([qh+ ; qh-] . [hi ; lo])_g,
// qh+ = max(qh, 0), qh- = min(qh, 0): one int8 product of length 2 D a page and head, on
// v_mfma_i32_16x16x64_i8.  |sum| <= 127^2 D < 2^24, so it is exact in int32 and as fp32, and the
// product with 2^e too: which pages win never depends on the order of summation.  (2^f is common to a
// row's pages and is left out.)  Scores become unsigned keys of the same order, 0 for pages the token
// does not see, the largest for forced pages (the first `sink`, the last `recent`); the num_pages-th
// largest key is found two bits a step by counting (v_cmp and s_bcnt1 over keys held in registers),
// and pages of that very key fill up in ascending order.
//
// The index is read once for a row: (2 D + 1) bytes a page and head, 1/32 of a 16-key bf16 page of
// 128-dim heads; it bounds long contexts.  Short ones are bound by latency (metadata, page ids, index
// rows, then the counting steps: four dependent round trips).
#pragma once

#include "page_index.h"

namespace rpa_sparse {
namespace {

constexpr uint32_t kForced = 0xffffffffu;  // no finite float maps to it, nor to 0

struct SelectParams {
  const uint16_t* q;
  const int8_t *bounds, *exps;
  const int32_t *kv_lens, *table, *cu, *num_seqs;
  int32_t* out;
  uint32_t* keys;  // the split form's keys
  long long q_token, q_head;  // strides, in values
  int T, Hkv, G, D, P, S, N, PPS, K, sink, recent;
  int gp;      // columns a token takes: G rounded up to a power of two (tiles), or to a multiple of 16
  int tokens;  // tokens a workgroup scores together
  long long stride;  // keys of a token's row: PPS rounded up to 16
  int first;   // the split form's first token
};

// A token's sequence and its newest page (-1: no key is visible, or no such token).
struct Place {
  int seq, pos;
};

// The sequence of token t, by a 64-ary search of cu (non-decreasing; anything else stays in range):
// one round trip for up to 64 sequences, two for 4096.
__device__ __forceinline__ Place place_of(const int32_t* cu, const int32_t* num_seqs, const int32_t* kv_lens, int N, int t) {
  const int lane = threadIdx.x % 64;
  const int ends = lane < N ? cu[lane + 1] : 0x7fffffff;  // beside num_seqs, not after it
  const int n = min(max(*num_seqs, 0), N);
  int lo = 0;
  if (n <= 64) {
    lo = __popcll(__ballot(lane < n && ends <= t));
  } else {
    int len = n;  // the answer is in [lo, lo + len]
    while (len > 0) {
      const int step = (len + 63) / 64;
      const int at = lo + (lane + 1) * step - 1;  // ends of the lane's part
      const bool below = at < lo + len && cu[at + 1] <= t;
      const int parts = __popcll(__ballot(below));
      const int base = lo + parts * step;
      len = min(step - 1, max(lo + len - base, 0));
      lo = min(base, n);
    }
  }
  if (lo >= n) return {-1, -1};
  const int begin = cu[lo], end = cu[lo + 1];
  if (t < begin || t >= end) return {-1, -1};
  return {lo, kv_lens[lo] - (end - t)};
}

__device__ __forceinline__ int newest_page(const Place& at, int S, int PPS) {
  if (at.pos < 0) return -1;
  const int page = at.pos / S;
  if (page >= PPS) {
    flag_error(RPA_SPARSE_ERR_LEN);
    return PPS - 1;
  }
  return page;
}

// A monotone map of finite floats to unsigned whole numbers.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Rounds one token's group of queries to int8: positive parts in columns' first D bytes, negative parts
// in the next D, zeros up to the row's end.  The columns past G repeat head 0, which leaves a maximum.
template <int STEPS>
__device__ void round_queries(const SelectParams& p, int t, int h, int8_t* rows, int row_bytes) {
  const int lane = threadIdx.x % 64, chunks = p.D / 8;
  const uint16_t* q = p.q + t * p.q_token + (long long)h * p.G * p.q_head;
  float amax = 0.f;
  for (int i = lane; i < p.G * chunks; i += 64) {
    float x[8];
    unpack8(*(const u32x4*)(q + i / chunks * p.q_head + 8 * (i % chunks)), x);
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[k]));  // fmaxf drops NaN
  }
#pragma unroll
  for (int d = 32; d; d /= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
  const float inv = pow2(-grid_exponent(amax));
  for (int i = lane; i < p.gp * chunks; i += 64) {
    const int col = i / chunks, c = i % chunks;
    float x[8];
    unpack8(*(const u32x4*)(q + (col < p.G ? col : 0) * p.q_head + 8 * c), x);
    u32x2 pos, neg;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = x[k] == x[k] ? (int)fminf(fmaxf(rintf(x[k] * inv), -127.f), 127.f) : 0;
      const uint32_t a = (uint32_t)(max(r, 0) & 255) << (8 * (k % 4)), b = (uint32_t)(min(r, 0) & 255) << (8 * (k % 4));
      if (k % 4 == 0) pos[k / 4] = a, neg[k / 4] = b;
      else pos[k / 4] |= a, neg[k / 4] |= b;
    }
    int8_t* row = rows + col * row_bytes;
    *(u32x2*)(row + 8 * c) = pos;
    *(u32x2*)(row + p.D + 8 * c) = neg;
  }
  const int tail = (STEPS * 64 - 2 * p.D) / 8;
  for (int i = lane; i < p.gp * tail; i += 64) *(u32x2*)(rows + i / tail * row_bytes + 2 * p.D + 8 * (i % tail)) = u32x2{0, 0};
}

// The largest of a lane's value over its group of `width` (1, 2, 4, 8 or 16) neighbouring lanes.
__device__ __forceinline__ int max_over(int v, int width) {
  if (width > 1) v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xf, 0xf, false));   // quad_perm 1 0 3 2
  if (width > 2) v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xf, 0xf, false));   // quad_perm 2 3 0 1
  if (width > 4) v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, false));  // row_half_mirror
  if (width > 8) v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, false));  // row_mirror
  return v;
}

// The keys of pages [begin, end) of one sequence (begin a multiple of 16; the last 16 may pass end) for
// the tokens of `rows`, 16 pages a wave and turn.  last[i]: the newest page of local token i, negative
// where it is of another sequence.  keys: token i's row at i * p.stride (LDS or global).
template <int STEPS, int WAVES>
__device__ __forceinline__ void score_pages(const SelectParams& p, int seq, int h, const int8_t* rows, const int* last,
                                            int begin, int end, uint32_t* keys) {
  constexpr int kRow = STEPS * 64 + 16;
  constexpr int kTurn = 2;  // page tiles a wave holds at once
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, n = lane % 16, j = lane / 16;
  const int width = min(p.gp, 16), tiles = p.tokens * p.gp / 16;  // column tiles
  const int32_t* table = p.table + (size_t)seq * p.PPS;
  for (int base = begin + wave * 16; base < end; base += WAVES * 16 * kTurn) {
    int phys[kTurn];
#pragma unroll
    for (int u = 0; u < kTurn; ++u) {
      const int page = min(base + u * WAVES * 16 + n, end - 1);
      phys[u] = table[page];
    }
    i32x4 a[kTurn][STEPS];
    int e[kTurn];
#pragma unroll
    for (int u = 0; u < kTurn; ++u) {
      if (phys[u] < 0 || phys[u] >= p.P) {
        flag_error(RPA_SPARSE_ERR_PAGE);
        phys[u] = 0;
      }
      const size_t at = (size_t)phys[u] * p.Hkv + h;
      const int8_t* row = p.bounds + at * 2 * p.D;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int off = 64 * s + 16 * j;
        a[u][s] = off < 2 * p.D ? *(const i32x4*)(row + off) : i32x4{0, 0, 0, 0};
      }
      e[u] = p.exps[at];
    }
#pragma unroll
    for (int u = 0; u < kTurn; ++u) {
      const int first = base + u * WAVES * 16;
      if (first >= end) break;
      float grid[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) grid[i] = pow2(min(max(__shfl(e[u], 4 * j + i), kExpMin), kExpMax));
      int best[4];
      for (int c = 0; c < tiles; ++c) {
        i32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const i32x4 b = *(const i32x4*)(rows + (16 * c + n) * kRow + 64 * s + 16 * j);
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][s], b, acc, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int m = max_over(acc[i], width);
          best[i] = p.gp > 16 && c > 0 ? max(best[i], m) : m;
        }
        if (p.gp > 16 && c + 1 < tiles) continue;  // one token over several tiles
        const int token = p.gp > 16 ? 0 : (16 * c + n) / width;
        const int newest = last[token];
        if (n % width == 0 && newest >= 0) {
          u32x4 key;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int page = first + 4 * j + i;
            key[i] = page > newest                                      ? 0
                     : page < p.sink || page > newest - p.recent        ? kForced
                                                                        : ordered((float)best[i] * grid[i]);
          }
          *(u32x4*)(keys + (size_t)token * p.stride + first + 4 * j) = key;
        }
      }
    }
  }
}

// Writes the chosen pages of one row, ascending, from its n keys; run by a team of THREADS threads (one
// wave, or the whole workgroup).  KPT: keys a thread holds in registers, consecutive ones; 0: any
// number, read again in every step.  s_count: 16 x 4 zeroed ints and s_scan: THREADS / 64 pairs, of
// the team's own; unused by teams of one wave.
template <int THREADS, int KPT>
__device__ __forceinline__ void choose(const uint32_t* keys, int n, int K, int32_t* out, int* s_count, Pair* s_scan) {
  const int tid = threadIdx.x % THREADS, lane = threadIdx.x % 64;
  if (n <= K) {  // all of them
    for (int i = tid; i < K; i += THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int per = KPT ? KPT : (n + THREADS - 1) / THREADS;
  const int own = tid * per;
  uint32_t held[KPT ? KPT : 1];
  if (KPT) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) held[i] = own + i < n ? keys[own + i] : 0;
  }
  const auto key = [&](int i) { return KPT ? held[KPT ? i : 0] : own + i < n ? keys[own + i] : 0u; };
  uint32_t threshold = 0;  // at least K keys reach it; n > K, so it ends above 0
  for (int step = 0; step < 16; ++step) {
    const int shift = 30 - 2 * step;
    const uint32_t t1 = threshold | 1u << shift, t2 = threshold | 2u << shift, t3 = threshold | 3u << shift;
    int c1 = 0, c2 = 0, c3 = 0;
    if (KPT) {
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        c1 += __popcll(__ballot(held[i] >= t1));
        c2 += __popcll(__ballot(held[i] >= t2));
        c3 += __popcll(__ballot(held[i] >= t3));
      }
    } else {
      for (int i = 0; i < per; ++i) {
        const uint32_t k = key(i);
        c1 += __popcll(__ballot(k >= t1));
        c2 += __popcll(__ballot(k >= t2));
        c3 += __popcll(__ballot(k >= t3));
      }
    }
    if (THREADS > 64) {
      if (lane == 0) {
        atomicAdd(s_count + 4 * step, c1);
        atomicAdd(s_count + 4 * step + 1, c2);
        atomicAdd(s_count + 4 * step + 2, c3);
      }
      __syncthreads();
      c1 = s_count[4 * step], c2 = s_count[4 * step + 1], c3 = s_count[4 * step + 2];
    }
    const int most = c3 >= K ? c3 : c2 >= K ? c2 : c1 >= K ? c1 : -1;
    threshold = c3 >= K ? t3 : c2 >= K ? t2 : c1 >= K ? t1 : threshold;
    if (most == K) break;  // exactly these
  }
  uint32_t above = 0, equal = 0;
#pragma unroll
  for (int i = 0; i < per; ++i) above += key(i) > threshold, equal += key(i) == threshold;
  Pair before, total;
  if (THREADS > 64) {
    before = scan_pairs<THREADS / 64>({above, equal}, total, s_scan);
  } else {
    Pair inc = {above, equal};
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t a = __shfl_up(inc.a, d), b = __shfl_up(inc.b, d);
      inc = lane >= d ? Pair{inc.a + a, inc.b + b} : inc;
    }
    total = {(uint32_t)__shfl((int)inc.a, 63), (uint32_t)__shfl((int)inc.b, 63)};
    before = {inc.a - above, inc.b - equal};
  }
  const uint32_t ties = (uint32_t)K - total.a;  // of the threshold's key, the first ones
  uint32_t a = before.a, b = before.b;
#pragma unroll
  for (int i = 0; i < per; ++i) {
    const uint32_t k = key(i);
    const bool gt = k > threshold, eq = k == threshold;
    if (gt || (eq && b < ties)) out[a + min(b, ties)] = own + i;
    a += gt, b += eq;
  }
}

// One launch for rows whose keys fit the LDS.  TILE: p.tokens consecutive tokens share each page's
// index row (prompt chunks), and a wave chooses for a token at a time; otherwise one token, and the
// workgroup chooses together.
template <int STEPS, int KPT, bool TILE>
__global__ __launch_bounds__(512) void select_kernel(SelectParams p) {
  constexpr int kThreads = 512, kWaves = kThreads / 64, kRow = STEPS * 64 + 16;
  extern __shared__ __align__(16) uint8_t lds[];
  uint32_t* const keys = (uint32_t*)lds;
  int8_t* const rows = (int8_t*)(lds + (size_t)p.tokens * p.stride * 4);
  __shared__ int s_seq[16], s_last[16], s_seen[16];
  __shared__ int s_count[64];
  __shared__ Pair s_scan[kWaves];
  const int tid = threadIdx.x, wave = tid / 64;
  const int h = blockIdx.x % p.Hkv, t0 = blockIdx.x / p.Hkv * p.tokens;
  if (tid < 64) s_count[tid] = 0;
  for (int i = wave; i < p.tokens; i += kWaves) {
    const int t = t0 + i;
    const Place at = t < p.T ? place_of(p.cu, p.num_seqs, p.kv_lens, p.N, t) : Place{-1, -1};
    const int newest = newest_page(at, p.S, p.PPS);
    if (tid % 64 == 0) s_seq[i] = newest < 0 ? -1 : at.seq, s_last[i] = newest;
    if (t < p.T) round_queries<STEPS>(p, t, h, rows + (size_t)i * p.gp * kRow, kRow);
    else
      for (int b = tid % 64; b < p.gp * kRow / 8; b += 64) ((u32x2*)(rows + (size_t)i * p.gp * kRow))[b] = u32x2{0, 0};
  }
  __syncthreads();
  for (int i = 0; i < p.tokens;) {  // a sequence's tokens together
    const int seq = s_seq[i];
    int next = i + 1;
    while (next < p.tokens && s_seq[next] == seq) ++next;
    const int visible = seq < 0 ? 0 : s_last[next - 1] + 1;
    if (visible > p.K) {
      if (TILE) {
        __syncthreads();
        if (tid < p.tokens) s_seen[tid] = tid >= i && tid < next ? s_last[tid] : -1;
        __syncthreads();
      }
      score_pages<STEPS, kWaves>(p, seq, h, rows, TILE ? s_seen : s_last, 0, visible, keys);
    }
    i = next;
  }
  __syncthreads();
  if (TILE) {
    for (int i = wave; i < p.tokens && t0 + i < p.T; i += kWaves)
      choose<64, KPT>(keys + (size_t)i * p.stride, s_last[i] + 1, p.K, p.out + ((size_t)(t0 + i) * p.Hkv + h) * p.K, nullptr,
                      nullptr);
  } else {
    choose<kThreads, KPT>(keys, s_last[0] + 1, p.K, p.out + ((size_t)t0 * p.Hkv + h) * p.K, s_count, s_scan);
  }
}

constexpr int kSplitPages = 512;  // pages a workgroup of the split form scores

// The split form, for few rows or rows past the LDS: keys to global memory, then a launch that chooses.
template <int STEPS>
__global__ __launch_bounds__(256) void score_kernel(SelectParams p) {
  constexpr int kThreads = 256, kWaves = kThreads / 64, kRow = STEPS * 64 + 16;
  extern __shared__ __align__(16) uint8_t lds[];
  int8_t* const rows = (int8_t*)lds;
  __shared__ int s_seq[16], s_last[16], s_seen[16];
  const int tid = threadIdx.x, wave = tid / 64;
  const int h = blockIdx.y, local = blockIdx.z * p.tokens, t0 = p.first + local;
  const int begin = blockIdx.x * kSplitPages;
  for (int i = wave; i < p.tokens; i += kWaves) {
    const int t = t0 + i;
    const Place at = t < p.T ? place_of(p.cu, p.num_seqs, p.kv_lens, p.N, t) : Place{-1, -1};
    const int newest = newest_page(at, p.S, p.PPS);
    if (tid % 64 == 0) s_seq[i] = newest < 0 ? -1 : at.seq, s_last[i] = newest;
  }
  __syncthreads();
  int most = -1;
  for (int i = 0; i < p.tokens; ++i) most = max(most, s_last[i]);
  if (most < begin) return;  // uniform
  for (int i = wave; i < p.tokens; i += kWaves) {
    if (t0 + i < p.T) round_queries<STEPS>(p, t0 + i, h, rows + (size_t)i * p.gp * kRow, kRow);
    else
      for (int b = tid % 64; b < p.gp * kRow / 8; b += 64) ((u32x2*)(rows + (size_t)i * p.gp * kRow))[b] = u32x2{0, 0};
  }
  __syncthreads();
  for (int i = 0; i < p.tokens;) {
    const int seq = s_seq[i];
    int next = i + 1;
    while (next < p.tokens && s_seq[next] == seq) ++next;
    const int visible = seq < 0 ? 0 : s_last[next - 1] + 1;
    if (visible > p.K && visible > begin) {
      __syncthreads();
      if (tid < p.tokens) s_seen[tid] = tid >= i && tid < next ? s_last[tid] : -1;
      __syncthreads();
      // token i's row of head h is p.keys + ((local + i) * Hkv + h) * stride: score_pages steps by p.stride
      SelectParams q = p;
      q.stride = p.stride * p.Hkv;
      score_pages<STEPS, kWaves>(q, seq, h, rows, s_seen, begin, min(visible, begin + kSplitPages),
                                 p.keys + ((size_t)local * p.Hkv + h) * p.stride);
    }
    i = next;
  }
}

template <int KPT>
__global__ __launch_bounds__(1024) void choose_kernel(SelectParams p) {
  constexpr int kThreads = 1024;
  __shared__ int s_count[64];
  __shared__ Pair s_scan[kThreads / 64];
  const int h = blockIdx.x % p.Hkv, local = blockIdx.x / p.Hkv, t = p.first + local;
  if (threadIdx.x < 64) s_count[threadIdx.x] = 0;
  const Place at = place_of(p.cu, p.num_seqs, p.kv_lens, p.N, t);
  const int newest = newest_page(at, p.S, p.PPS);
  __syncthreads();
  choose<kThreads, KPT>(p.keys + ((size_t)local * p.Hkv + h) * p.stride, newest + 1, p.K,
                        p.out + ((size_t)t * p.Hkv + h) * p.K, s_count, s_scan);
}

// ---- host side ----
int check_sparse(const rpa_sparse_shape_t* s) {
  if (!s) return fail(RPA_E_INVALID, "shape is NULL");
  if (s->num_tokens < 0) return fail(RPA_E_INVALID, "negative num_tokens");
  int rc = check_heads(s->num_kv_heads, s->head_dim, s->kv_dtype);
  if (rc) return rc;
  if ((rc = check_pool(s->total_pages, s->page_size))) return rc;
  if (s->num_q_heads <= 0 || s->max_num_seqs <= 0 || s->pages_per_seq <= 0 || s->num_pages <= 0)
    return fail(RPA_E_INVALID, "non-positive dimension in shape");
  if (s->num_q_heads % s->num_kv_heads)
    return fail(RPA_E_INVALID, "num_q_heads=%d must be divisible by num_kv_heads=%d", s->num_q_heads, s->num_kv_heads);
  if ((long long)s->pages_per_seq * s->page_size > 0x7fffffffll)
    return fail(RPA_E_INVALID, "pages_per_seq * page_size overflows int32");
  if ((long long)s->num_tokens * s->num_kv_heads > 0x7fffffffll)
    return fail(RPA_E_INVALID, "num_tokens * num_kv_heads overflows int32");
  if (s->num_q_heads / s->num_kv_heads > 256) return fail(RPA_E_UNSUPPORTED, "more than 256 query heads per kv head");
  return RPA_OK;
}

// How a call is laid out, from its sizes alone.
struct SelectPlan {
  int gp, tokens, steps;
  long long stride;
  bool tile, split;
  size_t lds;       // dynamic, of the scoring kernel
  long long batch;  // split: tokens scored before their pages are chosen
  size_t bytes;     // split: workspace
};

constexpr size_t kSelectLds = 60 * 1024;
constexpr size_t kSelectWorkspace = 256u << 20;  // the split form works through more rows in turns

SelectPlan plan_select(const rpa_sparse_shape_t& s) {
  SelectPlan r = {};
  const int G = s.num_q_heads / s.num_kv_heads;
  r.stride = ((long long)s.pages_per_seq + 15) / 16 * 16;
  const int need = (2 * s.head_dim + 63) / 64;
  r.steps = need <= 2 ? 2 : need <= 4 ? 4 : 8;
  const size_t row = r.steps * 64 + 16, keys = (size_t)r.stride * 4;
  const long long rows = (long long)s.num_tokens * s.num_kv_heads;
  r.tile = s.num_tokens > 2 * s.max_num_seqs && G <= 16;
  if (r.tile) {
    for (r.gp = 1; r.gp < G; r.gp *= 2) {
    }
    const int least = 16 / r.gp;  // the tokens of one column tile
    const size_t token = r.gp * row;
    for (r.tokens = 16; r.tokens > least && r.tokens * (token + keys) > kSelectLds; r.tokens /= 2) {
    }
    r.split = r.tokens * (token + keys) > kSelectLds || r.stride > 2048;
    for (r.tokens = r.split ? 16 : r.tokens; r.tokens > least && r.tokens * token > kSelectLds; r.tokens /= 2) {
    }
    r.lds = r.tokens * (token + (r.split ? 0 : keys));
  } else {
    r.gp = (G + 15) / 16 * 16;
    r.tokens = 1;
    r.split = r.gp * row + keys > kSelectLds || (rows < 256 && r.stride > 1024);
    r.lds = r.gp * row + (r.split ? 0 : keys);
  }
  if (r.split) {
    const long long token = (long long)s.num_kv_heads * keys, most = (long long)kSelectWorkspace / token;
    r.batch = most < r.tokens ? r.tokens : most / r.tokens * r.tokens;
    if (r.batch > 65535ll * r.tokens) r.batch = 65535ll * r.tokens;
    const long long all = ((long long)s.num_tokens + r.tokens - 1) / r.tokens * r.tokens;
    if (r.batch > all) r.batch = all;
    r.bytes = (size_t)(r.batch * token);
  }
  return r;
}

template <int STEPS>
int launch_select(const SelectPlan& plan, SelectParams p, hipStream_t stream) {
  if (!plan.split) {
    const int grid = (p.T + plan.tokens - 1) / plan.tokens * p.Hkv;
    const auto kernel = plan.tile ? (plan.stride <= 512 ? select_kernel<STEPS, 8, true> : select_kernel<STEPS, 32, true>)
                                  : (plan.stride <= 2048   ? select_kernel<STEPS, 4, false>
                                     : plan.stride <= 8192 ? select_kernel<STEPS, 16, false>
                                                           : select_kernel<STEPS, 32, false>);
    kernel<<<grid, 512, plan.lds, stream>>>(p);
    return launched("select_pages");
  }
  for (long long first = 0; first < p.T; first += plan.batch) {
    p.first = (int)first;
    const int tokens = (int)(p.T - first < plan.batch ? p.T - first : plan.batch);
    const dim3 grid((p.PPS + kSplitPages - 1) / kSplitPages, p.Hkv, (tokens + plan.tokens - 1) / plan.tokens);
    score_kernel<STEPS><<<grid, 256, plan.lds, stream>>>(p);
    const auto kernel = plan.stride <= 8192    ? choose_kernel<8>
                        : plan.stride <= 32768 ? choose_kernel<32>
                                               : choose_kernel<0>;
    kernel<<<tokens * p.Hkv, 1024, 0, stream>>>(p);
    const int rc = launched("select_pages");
    if (rc) return rc;
  }
  return RPA_OK;
}

}  // namespace
}  // namespace rpa_sparse
