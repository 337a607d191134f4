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
// largest key is found among the few that a first bound leaves, and pages of that very key fill up in ascending order.
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
  int gp;      // columns a token takes: G rounded up to 4, 8 or a multiple of 16
  int shift;   // log2 of gp, at most 4
  int tokens;  // tokens a workgroup scores together
  long long stride;  // keys of a token's row: PPS rounded up to 16
  int first;   // the split form's first token
  uint32_t chunk_magic;  // ceil(2^32 / (D / 8)): i / (D / 8) for i < 2^27
};

// A token's sequence and its newest page (-1: no key is visible, or no such token).
struct Place {
  int seq, pos;
};

// The sequence of token t and its position there: the number of sequences that end at or before t (cu
// is non-decreasing; anything else stays in range).  One round trip to memory where there are up to 64
// sequences, a lane each, or where token t is all of sequence t (a decode batch): all of that is loaded
// at once.  Otherwise a 64-ary search, two more for up to 4096 sequences and the ends' own.
__device__ __forceinline__ Place place_of(const int32_t* cu, const int32_t* num_seqs, const int32_t* kv_lens, int N, int t) {
  const int lane = threadIdx.x % 64;
  const int own = min(N <= 64 ? lane : t, N - 1);
  const int begin0 = cu[own], end0 = cu[own + 1], len0 = kv_lens[own];
  const int n = min(max(*num_seqs, 0), N);
  if (N <= 64) {
    const int lo = __popcll(__ballot(lane < n && end0 <= t));
    const int begin = __shfl(begin0, lo & 63), end = __shfl(end0, lo & 63), len = __shfl(len0, lo & 63);
    return lo >= n || t < begin || t >= end ? Place{-1, -1} : Place{lo, len - (end - t)};
  }
  if (t < n && begin0 == t && end0 == t + 1) return {t, len0 - 1};  // uniform: the same words in all lanes
  int lo = 0, len = n;  // the answer is in [lo, lo + len]
  while (len > 0) {
    const int step = (len + 63) / 64;
    const int at = lo + (lane + 1) * step - 1;  // the last of the lane's part
    const bool below = at < lo + len && cu[at + 1] <= t;
    const int base = lo + __popcll(__ballot(below)) * step;
    len = min(step - 1, max(lo + len - base, 0));
    lo = min(base, n);
  }
  if (lo >= n) return {-1, -1};
  const int begin = cu[lo], end = cu[lo + 1];
  return t < begin || t >= end ? Place{-1, -1} : Place{lo, kv_lens[lo] - (end - t)};
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
// One wave; w: the group's first values, 16 bytes a lane and 64 lanes a step, loaded beforehand.
constexpr int kHeld = 2;

__device__ __forceinline__ void load_queries(const SelectParams& p, int t, int h, u32x4 w[kHeld]) {
  const int lane = threadIdx.x % 64, chunks = p.D / 8;
  const uint16_t* q = p.q + t * p.q_token + (long long)h * p.G * p.q_head;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const int i = lane + 64 * k, col = __umulhi((uint32_t)i, p.chunk_magic);
    w[k] = u32x4{0, 0, 0, 0};
    if (i < p.G * chunks) w[k] = *(const u32x4*)(q + col * p.q_head + 8 * (i - col * chunks));
  }
}

template <int STEPS>
__device__ __forceinline__ void round_queries(const SelectParams& p, int t, int h, const u32x4 w[kHeld], int8_t* rows) {
  constexpr int kRow = STEPS * 64 + 16;
  const int lane = threadIdx.x % 64, chunks = p.D / 8, total = p.G * chunks;
  const uint16_t* q = p.q + t * p.q_token + (long long)h * p.G * p.q_head;
  const auto at = [&](int i) {
    const int col = __umulhi((uint32_t)i, p.chunk_magic);
    return *(const u32x4*)(q + col * p.q_head + 8 * (i - col * chunks));
  };
  float amax = 0.f;
  const auto widen = [&](u32x4 v) {
    float x[8];
    unpack8(v, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[k]));  // fmaxf drops NaN
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k) widen(w[k]);
  for (int i = lane + 64 * kHeld; i < total; i += 64) widen(at(i));
  const float inv = pow2(-grid_exponent(wave_max(amax)));
  const auto put = [&](int i, u32x4 v) {
    const int col = __umulhi((uint32_t)i, p.chunk_magic), c = i - col * chunks;
    float x[8];
    unpack8(v, x);
    u32x2 pos, neg;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = x[k] == x[k] ? (int)fminf(fmaxf(rintf(x[k] * inv), -127.f), 127.f) : 0;
      const uint32_t a = (uint32_t)(max(r, 0) & 255) << (8 * (k % 4)), b = (uint32_t)(min(r, 0) & 255) << (8 * (k % 4));
      if (k % 4 == 0) pos[k / 4] = a, neg[k / 4] = b;
      else pos[k / 4] |= a, neg[k / 4] |= b;
    }
    for (int to = col; to < p.gp; to = to < p.G && to > 0 ? p.gp : max(to + 1, p.G)) {  // head 0's also past G
      *(u32x2*)(rows + to * kRow + 8 * c) = pos;
      *(u32x2*)(rows + to * kRow + p.D + 8 * c) = neg;
    }
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (lane + 64 * k < total) put(lane + 64 * k, w[k]);
  for (int i = lane + 64 * kHeld; i < total; i += 64) put(i, at(i));
  const int tail = (STEPS * 64 - 2 * p.D) / 8;
  for (int i = lane; i < p.gp * tail; i += 64) *(u32x2*)(rows + i / tail * kRow + 2 * p.D + 8 * (i % tail)) = u32x2{0, 0};
}

template <int STEPS>
__device__ __forceinline__ void zero_queries(const SelectParams& p, int8_t* rows) {
  for (int i = threadIdx.x % 64; i < p.gp * (STEPS * 64 + 16) / 8; i += 64) ((u32x2*)rows)[i] = u32x2{0, 0};
}

// The largest of a lane's value over its group of 4, 8 or 16 neighbouring lanes.
__device__ __forceinline__ int max_over(int v, int width) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xf, 0xf, false));  // quad_perm 1 0 3 2
  v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xf, 0xf, false));  // quad_perm 2 3 0 1
  if (width > 4) v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, false));  // row_half_mirror
  if (width > 8) v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, false));  // row_mirror
  return v;
}

// The keys of pages [begin, end) of one sequence (begin a multiple of 16; the last 16 may pass end) for
// its local tokens [from, to), 16 pages a wave and turn, by wave `rank` of `waves`.  last[i]: local token
// i's newest page.  keys: token i's row at i * p.stride (LDS or global).  The next turn's page ids are
// loaded behind this turn's index rows.  The code is kept short: every workgroup runs it a few times
// only, and at first fetches it line by line.
template <int STEPS>
__device__ __forceinline__ void score_pages(const SelectParams& p, int seq, int h, const int8_t* rows, const int* last,
                                            int from, int to, int begin, int end, int rank, int waves, uint32_t* keys) {
  constexpr int kRow = STEPS * 64 + 16;
  const int lane = threadIdx.x % 64, n = lane % 16, j = lane / 16;
  const int width = 1 << p.shift;
  const int tile0 = from * p.gp / 16, tile1 = (to * p.gp + 15) / 16;  // column tiles of the tokens
  const int32_t* table = p.table + (size_t)seq * p.PPS;
  const int stride = waves * 16;
  int next = table[min(begin + rank * 16 + n, end - 1)];
#pragma unroll 1
  for (int first = begin + rank * 16; first < end; first += stride) {
    int phys = next;
    if (phys < 0 || phys >= p.P) {
      flag_error(RPA_SPARSE_ERR_PAGE);
      phys = 0;
    }
    const size_t at = (size_t)phys * p.Hkv + h;
    const int8_t* row = p.bounds + at * 2 * p.D;
    i32x4 a[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int off = 64 * s + 16 * j;
      a[s] = off < 2 * p.D ? *(const i32x4*)(row + off) : i32x4{0, 0, 0, 0};
    }
    const int e = p.exps[at];
    next = table[min(first + stride + n, end - 1)];
    // a token's columns share its four pages: column i of 4, 8 or 16 writes page i % 4
    const int i = n % 4, page = first + 4 * j + i;
    const float grid = pow2(min(max(__shfl(e, 4 * j + i), kExpMin), kExpMax));
    int best[4];
#pragma unroll 1
    for (int c = tile0; c < tile1; ++c) {
      i32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const i32x4 b = *(const i32x4*)(rows + (16 * c + n) * kRow + 64 * s + 16 * j);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s], b, acc, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int m = max_over(acc[k], width);
        best[k] = p.gp > 16 && c > tile0 ? max(best[k], m) : m;
      }
      if (p.gp > 16 && c + 1 < tile1) continue;  // one token over several tiles
      const int token = p.gp > 16 ? 0 : (16 * c + n) >> p.shift;
      if (token < from || token >= to) continue;
      const int newest = last[token];
      const int value = i & 2 ? (i & 1 ? best[3] : best[2]) : (i & 1 ? best[1] : best[0]);
      const uint32_t k = ordered((float)value * grid);
      keys[(size_t)token * p.stride + page] =
          page > newest ? 0 : page < p.sink || page > newest - p.recent ? kForced : k;
    }
  }
}

// The scores of a workgroup's local tokens over pages [begin, begin + pages): runs of tokens of one
// sequence are scored apart, by waves of their own where there are fewer runs than waves.
template <int STEPS, int WAVES>
__device__ __forceinline__ void score_tokens(const SelectParams& p, int h, const int8_t* rows, const int* seq, const int* last,
                                             int begin, int pages, uint32_t* keys) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  int runs = 0;
  for (int i = 0; i < p.tokens; ++i) runs += i == 0 || seq[i] != seq[i - 1];
  const int teams = min(runs, WAVES);
  int run = -1;
  for (int i = 0; i < p.tokens;) {
    int to = i + 1;
    while (to < p.tokens && seq[to] == seq[i]) ++to;
    ++run;
    const int visible = seq[i] < 0 ? 0 : last[to - 1] + 1;
    if (run % teams == wave % teams && visible > p.K && visible > begin)
      score_pages<STEPS>(p, seq[i], h, rows, last, i, to, begin, min(visible, begin + pages), wave / teams,
                         (WAVES - wave % teams + teams - 1) / teams, keys);
    i = to;
  }
}

constexpr int kFew = 128;  // candidates that one wave ranks

// What one wave shares with itself while it chooses for a row, and a workgroup.
struct WaveTeam {
  alignas(16) uint32_t key[kFew + 4];
  int page[kFew];
};
template <int THREADS>
struct Team {
  static constexpr int kGroups = 256;  // maxima that bound the choice
  int count[64];                       // zeroed before
  Pair scan[THREADS / 64];
  uint32_t bound;                      // zeroed before
  alignas(16) uint32_t top[kGroups];
  alignas(16) uint32_t key[THREADS + 4];
  int page[THREADS];
};

// Of `found` candidates in page order, `need` < found or equal: this thread's (number c) is chosen if
// fewer than `need` are higher, equal ones before it counting as higher.
__device__ __forceinline__ bool ranks_among(const uint32_t* key, int found, int need, int c) {
  const uint32_t k = c < found ? key[c] : 0u;
  int rank = 0;
#pragma unroll 4
  for (int i = 0; i < (found + 3) / 4; ++i) {
    const u32x4 o = ((const u32x4*)key)[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) rank += o[e] + (4 * i + e < c) > k;
  }
  return c < found && rank < need;
}

// A threshold that at least `need` of the team's keys reach, found two bits a step from the top by
// counting; fewer than `need` keys are above the one of 16 steps.  Ends early when at most `enough` keys
// reach it.  key(i), i < per: this thread's keys.
template <int THREADS, int PER, typename Key>
__device__ __forceinline__ uint32_t search(const Key& key, int per, int need, int enough, int steps, int* count) {
  uint32_t threshold = 0;
  for (int step = 0; step < steps; ++step) {
    const int shift = 30 - 2 * step;
    const uint32_t t1 = threshold | 1u << shift, t2 = threshold | 2u << shift, t3 = threshold | 3u << shift;
    int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
    for (int i = 0; i < (PER ? PER : per); ++i) {
      const uint32_t k = key(i);
      c1 += __popcll(__ballot(k >= t1));
      c2 += __popcll(__ballot(k >= t2));
      c3 += __popcll(__ballot(k >= t3));
    }
    if (THREADS > 64) {
      if (threadIdx.x % 64 == 0) {
        atomicAdd(count + 4 * step, c1);
        atomicAdd(count + 4 * step + 1, c2);
        atomicAdd(count + 4 * step + 2, c3);
      }
      __syncthreads();
      c1 = count[4 * step], c2 = count[4 * step + 1], c3 = count[4 * step + 2];
    }
    threshold = c3 >= need ? t3 : c2 >= need ? t2 : c1 >= need ? t1 : threshold;
    const int reach = c3 >= need ? c3 : c2 >= need ? c2 : c1 >= need ? c1 : enough + 1;
    if (reach <= enough) break;
  }
  return threshold;
}

// Writes the `need` highest of the team's keys' pages, ascending, of equal keys the first ones; more
// than `need` keys are not 0.  Threads own consecutive keys; page(i): of this thread's i-th.
template <int THREADS, int PER, typename Key, typename Page>
__device__ __forceinline__ void take(const Key& key, const Page& page, int per, int need, int32_t* out, int* count, Pair* scan) {
  const uint32_t threshold = search<THREADS, PER>(key, per, need, need, 16, count);
  Pair own = {0, 0}, total;
#pragma unroll
  for (int i = 0; i < (PER ? PER : per); ++i) own.a += key(i) > threshold, own.b += key(i) == threshold;
  Pair at = scan_pairs<THREADS / 64>(own, total, scan);
  const uint32_t ties = (uint32_t)need - total.a;  // of the threshold's own key, the first ones
#pragma unroll
  for (int i = 0; i < (PER ? PER : per); ++i) {
    const uint32_t k = key(i);
    const bool above = k > threshold, equal = k == threshold;
    if (above | (equal & (at.b < ties))) out[at.a + min(at.b, ties)] = page(i);
    at.a += above, at.b += equal;
  }
}

// The rows that list every page, and the forced pages of the others: before and behind the rest.
// Returns how many of the others are wanted, 0: nothing is left to do.
template <int THREADS>
__device__ __forceinline__ int choose_forced(const SelectParams& p, int n, int32_t* out) {
  const int tid = threadIdx.x % THREADS;
  if (n <= p.K) {
    for (int i = tid; i < p.K; i += THREADS) out[i] = i < n ? i : -1;
    return 0;
  }
  for (int i = tid; i < p.sink; i += THREADS) out[i] = i;
  for (int i = tid; i < p.recent; i += THREADS) out[p.K - p.recent + i] = n - p.recent + i;
  return p.K - p.sink - p.recent;  // n > K >= sink + recent
}

// One wave writes the chosen pages of one row, ascending, from its n <= 64 * KPT keys.
//
// Few keys survive a cheap bound: where the 64 lanes' maxima hold `need` values of at least x, so do the
// keys, and none below x is chosen.  x is the need-th largest maximum to 16 bits; of n random keys not many
// more than `need` survive.  They are moved together and each is ranked against all of them.
template <int KPT>
__device__ __forceinline__ void choose_wave(const SelectParams& p, const uint32_t* keys, int n, int32_t* out, WaveTeam& team) {
  const int lane = threadIdx.x % 64;
  const int need = choose_forced<64>(p, n, out);
  if (need == 0) return;
  out += p.sink;
  uint32_t held[KPT], top = 0;  // pages lane, lane + 64, ...
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    held[i] = 0;
    if (64 * i < n) held[i] = keys[min(64 * i + lane, n - 1)];
  }
#pragma unroll
  for (int i = 0; i < KPT; ++i) {  // forced pages count as absent
    held[i] = 64 * i + lane < n && held[i] != kForced ? held[i] : 0u;
    top = max(top, held[i]);
  }
  const auto count = [&](uint32_t t) { return __popcll(__ballot(top >= t)); };
  uint32_t bound = 0;
  for (int shift = 30; need <= 64 && shift >= 16; shift -= 2) {
    const uint32_t t1 = bound | 1u << shift, t2 = bound | 2u << shift, t3 = bound | 3u << shift;
    const int c1 = count(t1), c2 = count(t2), c3 = count(t3);
    bound = c3 >= need ? t3 : c2 >= need ? t2 : c1 >= need ? t1 : bound;
    if ((c3 >= need ? c3 : c2 >= need ? c2 : c1) == need) break;
  }
  bound = max(bound, 1u);
  int found = 0;
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    if (64 * i >= n) break;
    const bool is = held[i] >= bound;
    const unsigned long long who = __ballot(is);
    const int to = found + __popcll(who & ((1ull << lane) - 1));
    if (is && to < kFew) team.key[to] = held[i], team.page[to] = 64 * i + lane;
    found += __popcll(who);
  }
  int written = 0;
  if (found <= kFew) {
    if (lane < 4) team.key[found + lane] = 0;  // what the last four-word read passes
    wave_fence();
#pragma unroll 1
    for (int c = lane; c - lane < found; c += 64) {
      const bool chosen = ranks_among(team.key, found, need, c);
      const unsigned long long who = __ballot(chosen);
      if (chosen) out[written + __popcll(who & ((1ull << lane) - 1))] = team.page[c];
      written += __popcll(who);
    }
    wave_fence();
    return;
  }
  // too many: the threshold that `need` of all keys reach, its own key's first pages as far as they go
  const uint32_t threshold = search<64, KPT>([&](int i) { return held[i]; }, KPT, need, need, 16, nullptr);
  int above = 0, ties = 0;
#pragma unroll
  for (int i = 0; i < KPT; ++i) above += __popcll(__ballot(held[i] > threshold));
#pragma unroll
  for (int i = 0; i < KPT; ++i) {
    const unsigned long long equal = __ballot(held[i] == threshold);
    const bool chosen = held[i] > threshold ||
                        (held[i] == threshold && ties + __popcll(equal & ((1ull << lane) - 1)) < need - above);
    const unsigned long long who = __ballot(chosen);
    if (chosen) out[written + __popcll(who & ((1ull << lane) - 1))] = 64 * i + lane;
    written += __popcll(who), ties += __popcll(equal);
  }
}

// The same by a workgroup, for more keys, with barriers between its steps: 64 or 256 maxima bound the
// choice, and each thread ranks one candidate.  KPT: keys a thread holds in registers, consecutive ones, a
// multiple of 4; 0: any number, read again each time.  The row is allocated to a multiple of 16 keys.
template <int THREADS, int KPT>
__device__ __forceinline__ void choose(const SelectParams& p, const uint32_t* keys, int n, int32_t* out, Team<THREADS>& team) {
  const int tid = threadIdx.x, lane = tid % 64;
  const int need = choose_forced<THREADS>(p, n, out);
  if (need == 0) return;
  out += p.sink;
  const int per = KPT ? KPT : (n + THREADS - 1) / THREADS;
  const int own = tid * per;
  uint32_t held[KPT ? KPT : 4];
  if (KPT) {
#pragma unroll
    for (int i = 0; i < KPT; i += 4) {
      const u32x4 w = *(const u32x4*)(keys + (own + i < n ? own + i : 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) held[i + e] = w[e];
    }
#pragma unroll
    for (int i = 0; i < KPT; ++i) held[i] = own + i < n && held[i] != kForced ? held[i] : 0u;  // forced: absent
  }
  const auto key = [&](int i) {
    if (KPT) return held[KPT ? i : 0];
    const uint32_t k = own + i < n ? keys[own + i] : 0u;
    return k == kForced ? 0u : k;
  };
  const auto page = [&](int i) { return own + i; };
  const int groups = need <= 48 ? 64 : Team<THREADS>::kGroups;
  if (need <= groups / 4 * 3) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < (KPT ? KPT : per); ++i) top = max(top, key(i));
    const int wide = THREADS / groups;  // threads of a group, a power of two
    for (int d = 1; d < wide; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if (tid % wide == 0) team.top[tid / wide] = top;
    __syncthreads();
    if (tid < groups) {
      const uint32_t mine = team.top[tid];
      int reach = 0;
#pragma unroll 4
      for (int i = 0; i < groups / 4; ++i) {
        const u32x4 o = ((const u32x4*)team.top)[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) reach += o[k] >= mine;
      }
      if (reach >= need) atomicMax(&team.bound, mine);
    }
    __syncthreads();
    const uint32_t bound = max(1u, team.bound);
    Pair mine = {0, 0}, total;
#pragma unroll
    for (int i = 0; i < (KPT ? KPT : per); ++i) mine.a += key(i) >= bound;
    const Pair at = scan_pairs<THREADS / 64>(mine, total, team.scan);
    const int found = (int)total.a;
    if (found <= THREADS) {
      uint32_t to = at.a;
      if (mine.a) {
#pragma unroll
        for (int i = 0; i < (KPT ? KPT : per); ++i)
          if (key(i) >= bound) team.key[to] = key(i), team.page[to] = own + i, ++to;
      }
      if (tid < 4) team.key[found + tid] = 0;  // what the last four-word read passes
      __syncthreads();
      const bool chosen = tid - lane < found && ranks_among(team.key, found, need, tid);
      const unsigned long long who = __ballot(chosen);
      int written = 0;
      if (found > 64) {
        if (lane == 0) team.top[tid / 64] = __popcll(who);
        __syncthreads();
        for (int w = 0; w < tid / 64; ++w) written += team.top[w];
      }
      if (chosen) out[written + __popcll(who & ((1ull << lane) - 1))] = team.page[tid];
      return;
    }
  }
  __syncthreads();
  take<THREADS, KPT>(key, page, per, need, out, team.count, team.scan);
}

// Places the workgroup's tokens and rounds their queries.
template <int STEPS, int WAVES>
__device__ __forceinline__ void prepare_tokens(const SelectParams& p, int t0, int h, int* seq, int* last, int8_t* rows) {
  const int wave = threadIdx.x / 64;
  for (int i = wave; i < p.tokens; i += WAVES) {
    const int t = t0 + i;
    int8_t* const mine = rows + (size_t)i * p.gp * (STEPS * 64 + 16);
    Place at = {-1, -1};
    if (t < p.T) {
      u32x4 w[kHeld];
      load_queries(p, t, h, w);  // beside the metadata
      at = place_of(p.cu, p.num_seqs, p.kv_lens, p.N, t);
      round_queries<STEPS>(p, t, h, w, mine);
    } else {
      zero_queries<STEPS>(p, mine);
    }
    const int newest = newest_page(at, p.S, p.PPS);
    if (threadIdx.x % 64 == 0) seq[i] = newest < 0 ? -1 : at.seq, last[i] = newest;
  }
}

// One launch for rows whose keys fit the LDS: p.tokens consecutive tokens of a head share each page's index
// row (one token a sequence in decode batches).  WAVE: rows of up to 64 * KPT keys, chosen by a wave each;
// otherwise by the whole workgroup.
template <int STEPS, int KPT, bool WAVE>
__global__ __launch_bounds__(512) void select_kernel(SelectParams p) {
  constexpr int kThreads = 512, kWaves = kThreads / 64;
  extern __shared__ __align__(16) uint8_t lds[];
  uint32_t* const keys = (uint32_t*)lds;
  int8_t* const rows = (int8_t*)(lds + (size_t)p.tokens * p.stride * 4);
  __shared__ int s_seq[16], s_last[16];
  __shared__ typename std::conditional<WAVE, WaveTeam, Team<kThreads>>::type s_team[WAVE ? kWaves : 1];
  const int tid = threadIdx.x, wave = tid / 64;
  const int h = blockIdx.x % p.Hkv, t0 = blockIdx.x / p.Hkv * p.tokens;
  if constexpr (!WAVE)
    if (tid < 64) s_team[0].count[tid] = 0, s_team[0].bound = 0;
  prepare_tokens<STEPS, kWaves>(p, t0, h, s_seq, s_last, rows);
  __syncthreads();
  score_tokens<STEPS, kWaves>(p, h, rows, s_seq, s_last, 0, p.PPS, keys);
  __syncthreads();
  int32_t* const out = p.out + ((size_t)t0 * p.Hkv + h) * p.K;
  if constexpr (WAVE) {
    for (int i = wave; i < p.tokens && t0 + i < p.T; i += kWaves)
      choose_wave<KPT>(p, keys + (size_t)i * p.stride, s_last[i] + 1, out + (size_t)i * p.Hkv * p.K, s_team[wave]);
  } else {
    choose<kThreads, KPT>(p, keys, s_last[0] + 1, out, s_team[0]);  // one token
  }
}

constexpr int kSplitPages = 512;  // pages a workgroup of the split form scores

// The split form, for few rows or rows past the LDS: keys to global memory, then a launch that chooses.
template <int STEPS>
__global__ __launch_bounds__(256) void score_kernel(SelectParams p) {
  constexpr int kWaves = 4;
  extern __shared__ __align__(16) uint8_t lds[];
  int8_t* const rows = (int8_t*)lds;
  __shared__ int s_seq[16], s_last[16];
  const int h = blockIdx.y, local = blockIdx.z * p.tokens, begin = blockIdx.x * kSplitPages;
  prepare_tokens<STEPS, kWaves>(p, p.first + local, h, s_seq, s_last, rows);
  __syncthreads();
  // token i's row of head h is row (local + i) * Hkv + h of the keys
  uint32_t* const keys = p.keys + ((size_t)local * p.Hkv + h) * p.stride;
  p.stride *= p.Hkv;
  score_tokens<STEPS, kWaves>(p, h, rows, s_seq, s_last, begin, kSplitPages, keys);
}

template <int KPT>
__global__ __launch_bounds__(1024) void choose_kernel(SelectParams p) {
  constexpr int kThreads = 1024;
  __shared__ Team<kThreads> s_team;
  const int h = blockIdx.x % p.Hkv, local = blockIdx.x / p.Hkv, t = p.first + local;
  if (threadIdx.x < 64) s_team.count[threadIdx.x] = 0, s_team.bound = 0;
  const Place at = place_of(p.cu, p.num_seqs, p.kv_lens, p.N, t);
  const int newest = newest_page(at, p.S, p.PPS);
  __syncthreads();
  choose<kThreads, KPT>(p, p.keys + ((size_t)local * p.Hkv + h) * p.stride, newest + 1,
                        p.out + ((size_t)t * p.Hkv + h) * p.K, s_team);
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
    r.gp = G <= 4 ? 4 : G <= 8 ? 8 : 16;
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
    const auto kernel = plan.stride <= 512    ? select_kernel<STEPS, 8, true>
                        : plan.stride <= 2048 ? select_kernel<STEPS, 32, true>
                        : plan.stride <= 8192 ? select_kernel<STEPS, 16, false>
                                              : select_kernel<STEPS, 32, false>;
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
