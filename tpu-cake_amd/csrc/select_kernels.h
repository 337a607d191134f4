// The choice of pages: for each (token, kv head) the pages whose keys can score highest.
//
// Mathematics: the group's queries are rounded to int8 on a grid 2^f they share (f as the index's
// exponents), qh.  A key x of page p has q . x <= sum_d max(q_d hi_d, q_d lo_d); the score estimates that bound from qh,
// so a query below half a step of the group's grid counts as 0 and the head with the largest scores decides:
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
//
// Measured (8 kv heads of 128): 64 decode rows over 4 096 to 65 536 keys in pages of 64, 49 MB of index: 24 us,
// 2.1 TB/s; 2 rows over half a million keys in pages of 16, 127 MB: scored in 31 us, 4.1 TB/s, chosen in 12;
// a chunk of 1000 tokens over 32 768 keys in pages of 64, 15 MB: 35 us, of which rounding queries, scoring and
// choosing take a third each.  256 dims spill 5 or 6 registers of the 64 that two workgroups a CU leave.
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
  int tokens;  // tokens of a tile: consecutive ones of a sequence that a workgroup scores together
  long long stride;  // keys of a token's row: PPS rounded up to 16
  int first;   // the split form's first tile
  uint32_t chunk_magic;  // ceil(2^32 / (D / 8)): i / (D / 8) for i < 2^27
};

// A token's sequence and its newest page (-1: no key is visible, or no such token).
struct Place {
  int seq, pos;
};

// The sequence of token t and its position there: the number of sequences that end at or before t (cu
// is non-decreasing; anything else stays in range, and a negative length counts as 0).  One round trip to memory where there are up to 64
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
    return lo >= n || t < begin || t >= end ? Place{-1, -1} : Place{lo, max(len, 0) - (end - t)};
  }
  if (t < n && begin0 == t && end0 == t + 1) return {t, max(len0, 0) - 1};  // uniform: the same words in all lanes
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
  return t < begin || t >= end ? Place{-1, -1} : Place{lo, max(kv_lens[lo], 0) - (end - t)};
}

// The index-th tile of `size` (a power of two) consecutive tokens of one sequence: sequences in order,
// ceil(q_len / size) tiles each, then the tokens past the last (seq -1).  There are at most
// ceil(T / size) + N tiles.  count: its tokens, pos: its first token's position.  Offsets are taken into [0, T]
// and sums of tiles saturate, so whatever cu holds, first .. first + count are tokens of the call.
struct Tile {
  int seq, first, count, pos;
};

__device__ __forceinline__ Tile tile_of(const int32_t* cu, const int32_t* num_seqs, const int32_t* kv_lens, int N, int T, int size,
                                        int index) {
  if (size == 1) {
    const Place at = index < T ? place_of(cu, num_seqs, kv_lens, N, index) : Place{-1, -1};
    return {at.seq, index, index < T, at.pos};
  }
  const int lane = threadIdx.x % 64, shift = __builtin_ctz(size);
  int begin = cu[min(lane, N - 1)], end = cu[min(lane, N - 1) + 1], len = kv_lens[min(lane, N - 1)];
  const int n = min(max(*num_seqs, 0), N);
  const auto token = [T](int c) { return min(max(c, 0), T); };
  uint32_t before = 0;  // tiles of the sequences before this window's
  for (int base = 0; base < n; base += 64) {
    const int s = base + lane, from = token(begin), to = token(end);
    const uint32_t own = s < n && to > from ? (uint32_t)(to - from + size - 1) >> shift : 0u;
    uint32_t upto = own;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(upto, d);
      upto = sat_add(upto, lane >= d ? o : 0u);
    }
    const int here = __popcll(__ballot(before + upto <= (uint32_t)index));  // sequences of the window that lie before
    if (here < 64) {
      if (here) before += __shfl(upto, here - 1);
      const int e = __shfl(end, here), first = __shfl(from, here) + (int)(((uint32_t)index - before) << shift);
      return {base + here, first, min(size, __shfl(to, here) - first), max(__shfl(len, here), 0) - (e - first)};
    }
    before += __shfl(upto, 63);
    const int next = min(s + 64, N - 1);
    begin = cu[next], end = cu[next + 1], len = kv_lens[next];
  }
  const long long first = (n ? token(cu[n]) : 0) + ((long long)((uint32_t)index - before) << shift);
  return {-1, (int)min(first, (long long)T), (int)max(min((long long)size, T - first), 0ll), -1};
}

// The newest page of a token at `pos` (-1: it sees no key).
__device__ __forceinline__ int newest_page(int pos, int S, int PPS) {
  if (pos < 0) return -1;
  const int page = pos / S;
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
// One wave, 8 values a lane and step; the second pass finds them in the L1.
template <int STEPS>
__device__ __forceinline__ void round_queries(const SelectParams& p, int t, int h, int8_t* rows) {
  constexpr int kRow = STEPS * 64 + 16;
  const int lane = threadIdx.x % 64, chunks = p.D / 8, total = p.G * chunks;
  const uint16_t* q = p.q + t * p.q_token + (long long)h * p.G * p.q_head;
  float amax = 0.f;
#pragma unroll 1
  for (int i = lane; i < total; i += 64) {
    const int col = __umulhi((uint32_t)i, p.chunk_magic);
    float x[8];
    unpack8(*(const u32x4*)(q + col * p.q_head + 8 * (i - col * chunks)), x);
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[k]));  // fmaxf drops NaN
  }
  const float inv = pow2(-grid_exponent(wave_max(amax)));
#pragma unroll 1
  for (int i = lane; i < total; i += 64) {
    const int col = __umulhi((uint32_t)i, p.chunk_magic), c = i - col * chunks;
    float x[8];
    unpack8(*(const u32x4*)(q + col * p.q_head + 8 * c), x);
    u32x2 pos = {0, 0}, neg = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {  // the conversion to a byte turns negative values to 0
      const float y = x[k] == x[k] ? rintf(__builtin_amdgcn_fmed3f(x[k] * inv, -127.f, 127.f)) : 0.f;
      pos[k / 4] = __builtin_amdgcn_cvt_pk_u8_f32(y, k % 4, pos[k / 4]);
      neg[k / 4] = __builtin_amdgcn_cvt_pk_u8_f32(-y, k % 4, neg[k / 4]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) neg[k] = (0x80808080u - neg[k]) ^ 0x80808080u;  // minus each byte: they are at most 127
    for (int to = col; to < p.gp; to = to < p.G && to > 0 ? p.gp : max(to + 1, p.G)) {  // head 0's also past G
      *(u32x2*)(rows + to * kRow + 8 * c) = pos;
      *(u32x2*)(rows + to * kRow + p.D + 8 * c) = neg;
    }
  }
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

// The keys of pages [begin, end) of a sequence (begin a multiple of 16; the last 16 may pass end) for the
// `count` tokens of a tile, 16 pages a wave and turn.  last[i]: token i's newest page.  keys: token i's row
// at i * p.stride (LDS or global).  The next turn's page ids are
// loaded behind this turn's index rows.  The code is kept short: every workgroup runs it a few times
// only, and at first fetches it line by line.
template <int STEPS, int WAVES>
__device__ __forceinline__ void score_pages(const SelectParams& p, int seq, int h, const int8_t* rows, const int* last,
                                            int count, int begin, int end, uint32_t* keys) {
  constexpr int kRow = STEPS * 64 + 16;
  const int lane = threadIdx.x % 64, n = lane % 16, j = lane / 16;
  const int width = 1 << p.shift;
  const int columns = (count * p.gp + 15) / 16;  // tiles of 16
  const int32_t* table = p.table + (size_t)seq * p.PPS;
  constexpr int kStride = WAVES * 16;
  const int start = begin + threadIdx.x / 64 * 16;
  int next = table[min(start + n, end - 1)];
#pragma unroll 1
  for (int first = start; first < end; first += kStride) {
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
    next = table[min(first + kStride + n, end - 1)];
    // a token's columns share its four pages: column i of 4, 8 or 16 writes page i % 4
    const int i = n % 4, page = first + 4 * j + i;
    const float grid = pow2(min(max(__shfl(e, 4 * j + i), kExpMin), kExpMax));
    int best[4];
#pragma unroll 1
    for (int c = 0; c < columns; ++c) {
      i32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const i32x4 b = *(const i32x4*)(rows + (16 * c + n) * kRow + 64 * s + 16 * j);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s], b, acc, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int m = max_over(acc[k], width);
        best[k] = p.gp > 16 && c > 0 ? max(best[k], m) : m;
      }
      if (p.gp > 16 && c + 1 < columns) continue;  // one token over several tiles
      const int token = p.gp > 16 ? 0 : (16 * c + n) >> p.shift;
      if (token >= count) continue;
      const int newest = last[token];
      const int value = i & 2 ? (i & 1 ? best[3] : best[2]) : (i & 1 ? best[1] : best[0]);
      const uint32_t k = ordered((float)value * grid);
      keys[(size_t)token * p.stride + page] =
          page > newest ? 0 : page < p.sink || page > newest - p.recent ? kForced : k;
    }
  }
}

constexpr int kFew = 192;  // candidates that one wave ranks

struct WaveTeam {
  alignas(16) uint32_t key[kFew + 4];
  uint16_t page[kFew];  // of a row of at most kWaveRow
};

// What a workgroup shares while it chooses for a row.
template <int THREADS>
struct Team {
  static constexpr int kGroups = 256;  // maxima that bound the choice
  static constexpr int kMost = 512;    // candidates ranked
  int count[64];                       // zeroed before
  uint32_t bound;
  int found;                           // zeroed before
  Pair scan[THREADS / 64];
  alignas(16) uint32_t top[kGroups];
  unsigned long long key[kMost];  // candidates: key, then the page's complement
  int page[kGroups];           // chosen pages by rank
};

template <int THREADS>
__device__ __forceinline__ void clear_team(Team<THREADS>& team) {
  if (threadIdx.x < 64) team.count[threadIdx.x] = 0;
  if (threadIdx.x == 0) team.found = 0;
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

// The largest threshold that `need` of a wave's n keys reach, two bits a step from the top.
template <typename Key>
__device__ __forceinline__ uint32_t search_wave(const Key& key, int n, int need) {
  uint32_t threshold = 0;
  for (int shift = 30; shift >= 0; shift -= 2) {
    const uint32_t t1 = threshold | 1u << shift, t2 = threshold | 2u << shift, t3 = threshold | 3u << shift;
    int c1 = 0, c2 = 0, c3 = 0;
    for (int i = 0; i < n; i += 64) {
      const uint32_t k = key(i);
      c1 += __popcll(__ballot(k >= t1));
      c2 += __popcll(__ballot(k >= t2));
      c3 += __popcll(__ballot(k >= t3));
    }
    threshold = c3 >= need ? t3 : c2 >= need ? t2 : c1 >= need ? t1 : threshold;
  }
  return threshold;
}

// One wave writes the chosen pages of one row, ascending, from its n keys.
//
// Few keys survive a cheap bound: where 64 lanes' maxima, or four of each lane, hold `need` values of at least x,
// so do the keys, and none below x is chosen.  x is the need-th largest maximum to 16 bits; of n random keys not
// many more than `need` survive.  They are moved together and each is ranked against all of them.
__device__ __forceinline__ void choose_wave(const SelectParams& p, const uint32_t* keys, int n, int32_t* out, WaveTeam& team) {
  const int lane = threadIdx.x % 64;
  const unsigned long long below = (1ull << lane) - 1;
  const int need = choose_forced<64>(p, n, out);
  if (need == 0) return;
  out += p.sink;
  const auto key = [&](int i) {  // of page i + lane; forced pages and those past the row count as absent
    const uint32_t k = keys[min(i + lane, n - 1)];
    return i + lane < n && k != kForced ? k : 0u;
  };
  uint32_t top[4] = {0, 0, 0, 0};
#pragma unroll 1
  for (int i = 0; i < n; i += 256)
#pragma unroll
    for (int u = 0; u < 4; ++u) top[u] = max(top[u], key(i + 64 * u));
  const bool quick = need <= 32;  // 1000 tokens choose 30 of 512 pages in 32.8 us by 64 maxima, 33.8 by 256; 50 in 44 and 39
  if (quick) top[0] = max(max(top[0], top[1]), max(top[2], top[3]));
  const auto count = [&](uint32_t t) {
    int c = __popcll(__ballot(top[0] >= t));
    if (!quick) c += __popcll(__ballot(top[1] >= t)) + __popcll(__ballot(top[2] >= t)) + __popcll(__ballot(top[3] >= t));
    return c;
  };
  uint32_t bound = 0;
#pragma unroll 1
  for (int shift = 30; n > 64 && need < kFew && shift >= 16; shift -= 2) {
    const uint32_t t1 = bound | 1u << shift, t2 = bound | 2u << shift, t3 = bound | 3u << shift;
    const int c1 = count(t1), c2 = count(t2), c3 = count(t3);
    bound = c3 >= need ? t3 : c2 >= need ? t2 : c1 >= need ? t1 : bound;
    if ((c3 >= need ? c3 : c2 >= need ? c2 : c1) == need) break;
  }
  bound = max(bound, 1u);
  int found = 0;
  for (int i = 0; i < n; i += 256) {
    uint32_t k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) k[u] = key(i + 64 * u);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned long long who = __ballot(k[u] >= bound);
      const int to = found + __popcll(who & below);
      if (k[u] >= bound && to < kFew) team.key[to] = k[u], team.page[to] = (uint16_t)(i + 64 * u + lane);
      found += __popcll(who);
    }
  }
  int written = 0;
  if (found <= kFew) {
    if (lane < 4) team.key[found + lane] = 0;  // what the last four-word read passes
    wave_fence();
#pragma unroll 1
    for (int c = lane; c - lane < found; c += 64) {
      const uint32_t k = c < found ? team.key[c] : 0u;
      int rank = 0;
#pragma unroll 4
      for (int i = 0; i < (found + 3) / 4; ++i) {
        const u32x4 o = ((const u32x4*)team.key)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) rank += o[e] + (4 * i + e < c) > k;  // an equal key of an earlier page, too
      }
      const bool chosen = c < found && rank < need;
      const unsigned long long who = __ballot(chosen);
      if (chosen) out[written + __popcll(who & below)] = team.page[c];
      written += __popcll(who);
    }
    wave_fence();
    return;
  }
  // too many: the threshold that `need` of all keys reach, and its own key's first pages as far as they go
  const uint32_t threshold = search_wave(key, n, need);
  int above = 0, ties = 0;
  for (int i = 0; i < n; i += 64) above += __popcll(__ballot(key(i) > threshold));
  for (int i = 0; i < n; i += 64) {
    const uint32_t k = key(i);
    const unsigned long long equal = __ballot(k == threshold);
    const bool chosen = (k > threshold) | ((k == threshold) & (ties + __popcll(equal & below) < need - above));
    const unsigned long long who = __ballot(chosen);
    if (chosen) out[written + __popcll(who & below)] = i + lane;
    written += __popcll(who), ties += __popcll(equal);
  }
}

// The same by a workgroup, for longer rows.  256 maxima bound the choice, searched by one wave; candidates come
// together in any order, each is ranked by key and page against all of them, and the chosen ones by page among
// themselves, so the order of the atomics leaves no trace.  Rows of up to kBatch keys a thread are read
// once.
template <int THREADS, int kBatch>  // kBatch: keys of a thread in flight
__device__ __forceinline__ void choose(const SelectParams& p, const uint32_t* keys, int n, int32_t* out, Team<THREADS>& team) {
  constexpr int kWaves = THREADS / 64;
  constexpr int kGroups = Team<THREADS>::kGroups, kMost = Team<THREADS>::kMost;
  const int tid = threadIdx.x, lane = tid % 64;
  const int need = choose_forced<THREADS>(p, n, out);
  if (need == 0) return;
  out += p.sink;
  const auto key = [&](int i) {
    const uint32_t k = keys[min(i, n - 1)];
    return i < n && k != kForced ? k : 0u;
  };
  if (need <= kGroups / 4 * 3) {
    uint32_t k[kBatch], top = 0;
    const auto load = [&](int i) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) k[u] = i + THREADS * u < n ? keys[min(i + THREADS * u + tid, n - 1)] : 0u;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) k[u] = i + THREADS * u + tid < n && k[u] != kForced ? k[u] : 0u;
    };
    for (int i = 0; i < n; i += kBatch * THREADS) {
      load(i);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) top = max(top, k[u]);
    }
    constexpr int kWide = THREADS / kGroups;  // threads of a group: 4
    static_assert(kWide == 4, "a quad");
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp((int)top, (int)top, 0xB1, 0xf, 0xf, false));  // quad_perm 1 0 3 2
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp((int)top, (int)top, 0x4E, 0xf, 0xf, false));  // quad_perm 2 3 0 1
    if (tid % kWide == 0) team.top[tid / kWide] = top;
    __syncthreads();
    if (tid < 64) {
      const u32x4 mine = ((const u32x4*)team.top)[lane];
      const auto count = [&](uint32_t t) {
        return __popcll(__ballot(mine[0] >= t)) + __popcll(__ballot(mine[1] >= t)) + __popcll(__ballot(mine[2] >= t)) +
               __popcll(__ballot(mine[3] >= t));
      };
      uint32_t bound = 0;
#pragma unroll 1
      for (int shift = 30; shift >= 14; shift -= 2) {
        const uint32_t t1 = bound | 1u << shift, t2 = bound | 2u << shift, t3 = bound | 3u << shift;
        const int c1 = count(t1), c2 = count(t2), c3 = count(t3);
        bound = c3 >= need ? t3 : c2 >= need ? t2 : c1 >= need ? t1 : bound;
        if ((c3 >= need ? c3 : c2 >= need ? c2 : c1) == need) break;
      }
      if (lane == 0) team.bound = max(bound, 1u);
    }
    __syncthreads();
    const uint32_t bound = team.bound;
    for (int i = 0; i < n; i += kBatch * THREADS) {
      if (n > kBatch * THREADS) load(i);
      int own = 0;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) own += k[u] >= bound;
      if (own) {
        int to = atomicAdd(&team.found, own);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (k[u] >= bound) {
            if (to < kMost) team.key[to] = (unsigned long long)k[u] << 32 | (uint32_t)~(i + THREADS * u + tid);
            ++to;
          }
      }
    }
    __syncthreads();
    const int found = team.found;
    if (found <= kMost) {
      // each candidate against every kWide-th of them
      for (int c = tid / kWide; c < found; c += kGroups) {
        const unsigned long long mine = team.key[c];
        int rank = 0;
#pragma unroll 4
        for (int i = tid % kWide; i < found; i += kWide) rank += team.key[i] > mine;
        rank += __builtin_amdgcn_update_dpp(0, rank, 0xB1, 0xf, 0xf, false);
        rank += __builtin_amdgcn_update_dpp(0, rank, 0x4E, 0xf, 0xf, false);
        if (tid % kWide == 0 && rank < need) team.page[rank] = ~(uint32_t)mine;
      }
      __syncthreads();
      for (int r = tid / kWide; r < need; r += kGroups) {
        const int page = team.page[r];
        int at = 0;
#pragma unroll 4
        for (int i = tid % kWide; i < need; i += kWide) at += team.page[i] < page;
        at += __builtin_amdgcn_update_dpp(0, at, 0xB1, 0xf, 0xf, false);
        at += __builtin_amdgcn_update_dpp(0, at, 0x4E, 0xf, 0xf, false);
        if (tid % kWide == 0) out[at] = page;
      }
      return;
    }
  }
  // too many: a search by thresholds with a barrier a step, over consecutive keys of each thread
  const int per = (n + THREADS - 1) / THREADS, own = tid * per, end = min(own + per, n);
  uint32_t threshold = 0;
  __syncthreads();
#pragma unroll 1
  for (int step = 0; step < 16; ++step) {
    const int shift = 30 - 2 * step;
    const uint32_t t1 = threshold | 1u << shift, t2 = threshold | 2u << shift, t3 = threshold | 3u << shift;
    int c1 = 0, c2 = 0, c3 = 0;
    for (int i = own; i < end; ++i) {
      const uint32_t k = key(i);
      c1 += k >= t1, c2 += k >= t2, c3 += k >= t3;
    }
    if (c1) atomicAdd(&team.count[4 * step], c1);
    if (c2) atomicAdd(&team.count[4 * step + 1], c2);
    if (c3) atomicAdd(&team.count[4 * step + 2], c3);
    __syncthreads();
    c1 = team.count[4 * step], c2 = team.count[4 * step + 1], c3 = team.count[4 * step + 2];
    threshold = c3 >= need ? t3 : c2 >= need ? t2 : c1 >= need ? t1 : threshold;
  }
  Pair mine = {0, 0}, total;
  for (int i = own; i < end; ++i) mine.a += key(i) > threshold, mine.b += key(i) == threshold;
  Pair at = scan_pairs<kWaves>(mine, total, team.scan);
  const uint32_t ties = (uint32_t)need - total.a;  // of the threshold's own key, the first ones
  for (int i = own; i < end; ++i) {
    const uint32_t k = key(i);
    const bool above = k > threshold, equal = k == threshold;
    if (above | (equal & (at.b < ties))) out[at.a + min(at.b, ties)] = i;
    at.a += above, at.b += equal;
  }
}

// The workgroup's tile, its queries rounded, a wave a token, and its tokens' newest pages.
template <int STEPS, int WAVES>
__device__ __forceinline__ Tile prepare_tile(const SelectParams& p, int index, int h, int* last, int8_t* rows) {
  const Tile tile = tile_of(p.cu, p.num_seqs, p.kv_lens, p.N, p.T, p.tokens, index);
  for (int i = threadIdx.x / 64; i < p.tokens; i += WAVES) {
    int8_t* const mine = rows + (size_t)i * p.gp * (STEPS * 64 + 16);
    const bool live = i < tile.count && tile.seq >= 0;
    if (live) {
      round_queries<STEPS>(p, tile.first + i, h, mine);
    } else {
      zero_queries<STEPS>(p, mine);
    }
    const int newest = live ? newest_page(tile.pos + i, p.S, p.PPS) : -1;
    if (threadIdx.x % 64 == 0) last[i] = newest;
  }
  return tile;
}

// One launch for rows whose keys fit the LDS: a workgroup scores a tile's tokens, or in decode batches one
// token, for a head.  WAVE: a row is chosen by a wave, otherwise (one token) by the whole workgroup.
constexpr int kSelectThreads = 1024;

template <int STEPS, bool WAVE>
__global__ __launch_bounds__(kSelectThreads, 8) void select_kernel(SelectParams p) {
  constexpr int kThreads = kSelectThreads, kWaves = kThreads / 64;
  extern __shared__ __align__(16) uint8_t lds[];
  uint32_t* const keys = (uint32_t*)lds;
  int8_t* const rows = (int8_t*)(lds + (size_t)p.tokens * p.stride * 4);
  __shared__ int s_last[16];
  __shared__ typename std::conditional<WAVE, WaveTeam, Team<kThreads>>::type s_team[WAVE ? kWaves : 1];
  const int tid = threadIdx.x, wave = tid / 64;
  const int h = blockIdx.x % p.Hkv;
  if constexpr (!WAVE) clear_team(s_team[0]);
  const Tile tile = prepare_tile<STEPS, kWaves>(p, blockIdx.x / p.Hkv, h, s_last, rows);
  if (tile.count == 0) return;  // uniform
  __syncthreads();
  const int visible = s_last[tile.count - 1] + 1;
  if (visible > p.K) score_pages<STEPS, kWaves>(p, tile.seq, h, rows, s_last, tile.count, 0, visible, keys);
  __syncthreads();
  int32_t* const out = p.out + ((size_t)tile.first * p.Hkv + h) * p.K;
  if constexpr (WAVE) {
    for (int i = wave; i < tile.count; i += kWaves)
      choose_wave(p, keys + (size_t)i * p.stride, s_last[i] + 1, out + (size_t)i * p.Hkv * p.K, s_team[wave]);
  } else {
    choose<kThreads, 4>(p, keys, s_last[0] + 1, out, s_team[0]);  // from LDS
  }
}

constexpr int kSplitPages = 256;  // pages a workgroup of the split form scores (two rows of 31 000 pages of 16 keys
                                   // 49.5 us, one of them 28.2; 49.8 and 30.8 with 512, 55.7 and 36.7 with 1024)

// The split form, for few rows or rows past the LDS: keys to global memory, then a launch that chooses.
// Token i of the z-th tile and head h have row (z * p.tokens + i) * Hkv + h of the keys.
template <int STEPS>
__global__ __launch_bounds__(256) void score_kernel(SelectParams p) {
  constexpr int kWaves = 4;
  extern __shared__ __align__(16) uint8_t lds[];
  int8_t* const rows = (int8_t*)lds;
  __shared__ int s_last[16];
  const int h = blockIdx.y, begin = blockIdx.x * kSplitPages;
  const Tile tile = prepare_tile<STEPS, kWaves>(p, p.first + blockIdx.z, h, s_last, rows);
  if (tile.seq < 0 || tile.count == 0) return;  // uniform
  __syncthreads();
  const int visible = s_last[tile.count - 1] + 1;
  if (visible <= p.K || visible <= begin) return;
  uint32_t* const keys = p.keys + ((size_t)blockIdx.z * p.tokens * p.Hkv + h) * p.stride;
  p.stride *= p.Hkv;
  score_pages<STEPS, kWaves>(p, tile.seq, h, rows, s_last, tile.count, begin, min(visible, begin + kSplitPages), keys);
}

__global__ __launch_bounds__(1024) void choose_kernel(SelectParams p) {
  constexpr int kThreads = 1024;
  __shared__ Team<kThreads> s_team;
  const int h = blockIdx.x % p.Hkv, row = blockIdx.x / p.Hkv, i = row % p.tokens;
  clear_team(s_team);
  const Tile tile = tile_of(p.cu, p.num_seqs, p.kv_lens, p.N, p.T, p.tokens, p.first + row / p.tokens);
  if (i >= tile.count) return;  // uniform
  const int newest = tile.seq < 0 ? -1 : newest_page(tile.pos + i, p.S, p.PPS);
  __syncthreads();
  choose<kThreads, 32>(p, p.keys + (size_t)blockIdx.x * p.stride, newest + 1, p.out + ((size_t)(tile.first + i) * p.Hkv + h) * p.K,
                   s_team);
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
  if (s->num_tokens + 16ll * s->max_num_seqs > 0x7fffffffll)
    return fail(RPA_E_INVALID, "num_tokens + 16 * max_num_seqs overflows int32");
  if (s->pages_per_seq > kMostIndex || s->num_pages > kMostIndex)
    return fail(RPA_E_UNSUPPORTED, "pages_per_seq and num_pages must be at most 2^31 - 2^16 - 1");
  if (s->num_q_heads / s->num_kv_heads > 256) return fail(RPA_E_UNSUPPORTED, "more than 256 query heads per kv head");
  return RPA_OK;
}

// How a call is laid out, from its sizes alone.
struct SelectPlan {
  int gp, tokens, steps;
  long long stride;
  bool tile, split;
  size_t lds;       // dynamic, of the scoring kernel
  long long tiles;
  long long batch;  // split: tiles scored before their pages are chosen
  size_t bytes;     // split: workspace
};

constexpr long long kWaveRow = 2048;  // keys of a row that one wave chooses from
// The same in decode batches, where the other waves have no row of their own: 200 rows of 8 heads and up to 256 pages
// take 34 us by a wave and 38 by the workgroup, 64 rows of up to 1024 pages 25 and 24, 128 of them chosen 34 and 28.
constexpr long long kWaveDecode = 512;
constexpr size_t kSelectLds = 58 * 1024;
constexpr size_t kSelectWorkspace = 256u << 20;  // the split form works through more rows in turns

SelectPlan plan_select(const rpa_sparse_shape_t& s) {
  SelectPlan r = {};
  const int G = s.num_q_heads / s.num_kv_heads;
  r.stride = ((long long)s.pages_per_seq + 15) / 16 * 16;
  const int need = (2 * s.head_dim + 63) / 64;
  r.steps = need <= 2 ? 2 : need <= 4 ? 4 : 8;
  const size_t row = r.steps * 64 + 16, keys = (size_t)r.stride * 4;
  const long long rows = (long long)s.num_tokens * s.num_kv_heads;
  // Tiles or rows, by the tokens a table row has, as the attention (32 heads, 8 kv heads, 32 768 keys in pages of 64; us as
  // tiles and as rows): 64 decode rows beside a chunk of 16 29 and 25, of 66 29 and 34, of 200 29 and 56; 64 sequences of 2
  // tokens 21 and 32.
  r.tile = s.num_tokens > 2 * s.max_num_seqs && G <= 16;
  if (r.tile) {
    r.gp = G <= 4 ? 4 : G <= 8 ? 8 : 16;
    const int least = 16 / r.gp;  // the tokens of one column tile
    const size_t token = r.gp * row;
    for (r.tokens = 16; r.tokens > least && r.tokens * (token + keys) > kSelectLds; r.tokens /= 2) {
    }
    r.split = r.tokens * (token + keys) > kSelectLds || r.stride > kWaveRow;
    for (r.tokens = r.split ? 16 : r.tokens; r.tokens > least && r.tokens * token > kSelectLds; r.tokens /= 2) {
    }
    r.lds = r.tokens * (token + (r.split ? 0 : keys));
  } else {
    r.gp = (G + 15) / 16 * 16;
    r.tokens = 1;
    // Few rows of long tables are split over workgroups: 32 rows of up to 2048 pages take 20 us split and 26 whole, 128 rows
    // 26 and 26; of up to 8192 pages 128 rows 67 and 108, 248 rows 121 and 123.  248 rows of up to 2048 pages would be
    // faster whole, 34 us where they take 43.
    r.split = r.gp * row + keys > kSelectLds || (rows < 256 && r.stride > 1024);
    r.lds = r.gp * row + (r.split ? 0 : keys);
  }
  r.tiles = r.tokens == 1 ? s.num_tokens : ((long long)s.num_tokens + r.tokens - 1) / r.tokens + s.max_num_seqs;
  if (r.split) {
    const long long tile = r.tokens * (long long)s.num_kv_heads * keys, most = (long long)kSelectWorkspace / tile;
    const long long launch = kMostThreads / 1024 / (r.tokens * (long long)s.num_kv_heads);  // of choosing; at least 3
    r.batch = most < 1 ? 1 : most > 65535 ? 65535 : most;
    if (r.batch > launch) r.batch = launch;
    if (r.batch > r.tiles) r.batch = r.tiles;
    r.bytes = (size_t)(r.batch * tile);
  }
  return r;
}

template <int STEPS>
int launch_select(const SelectPlan& plan, SelectParams p, hipStream_t stream) {
  if (!plan.split) {
    if (const int rc = check_launch(plan.tiles * p.Hkv, kSelectThreads)) return rc;
    const bool wave = plan.stride <= (plan.tokens > 1 ? kWaveRow : kWaveDecode);
    const auto kernel = wave ? select_kernel<STEPS, true> : select_kernel<STEPS, false>;
    kernel<<<(unsigned)(plan.tiles * p.Hkv), kSelectThreads, plan.lds, stream>>>(p);
    return launched("select_pages");
  }
  for (long long first = 0; first < plan.tiles; first += plan.batch) {
    p.first = (int)first;
    const int tiles = (int)(plan.tiles - first < plan.batch ? plan.tiles - first : plan.batch);
    const dim3 grid((p.PPS + kSplitPages - 1) / kSplitPages, p.Hkv, tiles);
    score_kernel<STEPS><<<grid, 256, plan.lds, stream>>>(p);
    choose_kernel<<<tiles * plan.tokens * p.Hkv, 1024, 0, stream>>>(p);
    const int rc = launched("select_pages");
    if (rc) return rc;
  }
  return RPA_OK;
}

}  // namespace
}  // namespace rpa_sparse
