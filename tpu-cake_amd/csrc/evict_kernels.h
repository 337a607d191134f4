// Eviction: which rows of a sequence each kv head keeps, and the moves that bring them together.
//
// Mathematics: a row's key is its weight as an unsigned whole number of the same order (0 for NaN), the largest of all for
// rows that stay in any case.  The budget-th largest key of a (sequence, head) is found digit by digit: counts of the
// next bits over the rows that share the bits so far, three times.  Rows above it stay, and of the rows at it
// the lowest ones, as many as fit.  Kept rows at or past `budget` and rows below it that go are equally many: the i-th of the
// one take the places of the i-th of the other.  Counts are whole numbers, so nothing depends on an order.
//
// A cache's rows are in no order for attention, so only what lies past the budget is moved, not everything behind the
// first gap; the ledger's positions tell the recent rows.  Moves read past the budget and write before it: they
// do not meet, and a list that is applied twice gives the same.
//
// Latency bounds the choice: 512 lists of 2112 rows read 5 MB and take 15 us, three passes over keys in LDS with a barrier
// or two each; 24 lists of 105 000 to 126 000 rows (23 MB, 4 us at 6.3 TB/s) take 49 us: keys and their first digits 14,
// the digits 10 + 4 + 7, tallies 4, the list 12.  Moves are copies: 64 lists of 8 heads, 64 entries each at most, 11 MB, 5.6 us;
// six fp8 prompts' 2048 entries a head, 49 MB, 7.8 us at 6.3 TB/s, 20 where rows change their scale and 9.6 where all
// pages have one: a full division a value makes it five times the vector instructions.
#pragma once

#include "attend_kernels.h"

namespace rpa_sparse {
namespace {

struct ChooseParams {
  const float* weights;
  const int32_t *positions, *kv_lens, *table, *num_seqs, *dropped;
  int32_t* moves;
  uint32_t* found;   // of each (sequence, head): the budget-th largest key (first its first digit) and its rank among those
  struct Long* longs;  // of each sequence
  // of each block of a long sequence's head, kKeyRows rows:
  uint32_t* keys;
  uint32_t* near;    // the keys that have the first digit: those of each kSegment rows at their beginning,
  uint32_t* held;    // so many
  uint32_t* counts;  // kDigits
  uint32_t* tallies; // a Tally
  int N, PPS, Hkv, P, S, budget, limit, sinks, recent, M;
  int first;         // the launch's first sequence
  int block_room;    // blocks of a head that the workspace holds
  int room;          // keys that fit a workgroup's LDS
  int quads;         // four neighbouring entries from a multiple of four on are 16 aligned bytes of one page
};

// The order of weights as whole numbers, 0 for NaN; zeros of both signs are equal.
__device__ __forceinline__ uint32_t weight_key(float w) { return w == w ? ordered(w + 0.f) : 0u; }

// Rows of a sequence whose keys fit LDS: one workgroup does all (48 lists of 32768: 36 us, 37 by blocks; 512: 92 and 119; of
// 16384: 23 and 33, 53 and 82).  Past them its VALU would be what counts (24 lists of 131072: 132 us), so all that goes over
// rows is done by blocks of kKeyRows, and one workgroup a list sums the blocks' counts and goes over the keys that share
// the first digit: 49 us in six launches.  Which of them run follows the table's width, the only length the host knows: 512
// lists of 2112 rows take 15 us in a table as wide and 44 in one of 131072 rows, 22 of them in the rows kernel, whose 128 KB
// of LDS leave one list a CU, and the rest in launches that find nothing.
constexpr int kChooseRows = 32768;
constexpr int kKeyRows = 4096, kSegment = kKeyRows / 4;  // a wave's rows of a block
constexpr int kDigits = 2048;       // 11 bits, 11 bits, 10 bits

// The rows of a sequence of `len` keys, 0 where it is not cut.
__device__ __forceinline__ int rows_cut(const ChooseParams& p, int len) {
  const int n = min(len, p.PPS * p.S);
  return len > p.limit && n > p.budget ? n : 0;
}

// A sequence that is cut: its rows, and the position past its last.
struct Cut {
  int rows;
  long long end;
};
__device__ __forceinline__ Cut cut_of(const ChooseParams& p, int seq, bool flag) {
  const int count = *p.num_seqs, len = p.kv_lens[seq], gone = p.dropped ? p.dropped[seq] : 0;
  const int n = seq < count ? len : 0;
  if (flag && n > p.PPS * p.S) flag_error(RPA_SPARSE_ERR_LEN);
  return {rows_cut(p, n), (long long)n + gone};
}

// Long sequences' blocks lie one sequence behind the other, so that the workspace holds what the pool's rows need and
// not what the table has room for (64 requests of 2100 keys with tables of 131072 rows, 8 heads: 672 MB by the table).
// Distinct pages cannot have more.  A sequence that finds no room all the same, as others hold its pages too, is
// done by one workgroup a head from the ledger.
__device__ __forceinline__ int blocks_of(int rows) { return (rows + kKeyRows - 1) / kKeyRows; }

struct Long {
  int rows;   // 0: all its keys fit LDS, or its blocks have no room
  int place;  // its first block, of as many as one head has
  __device__ __forceinline__ size_t block0(const ChooseParams& p, int h) const {
    return (size_t)place * p.Hkv + (size_t)h * blocks_of(rows);
  }
};

// A sequence's, by each wave for itself.
__device__ __forceinline__ Long long_of(const ChooseParams& p, int seq, int rows) {
  const int count = *p.num_seqs;
  long long before = 0;
  for (int i = threadIdx.x % 64; i < min(seq, count); i += 64) {
    const int n = rows_cut(p, p.kv_lens[i]);
    before += n > p.room ? blocks_of(n) : 0;
  }
  for (int d = 1; d < 64; d *= 2) before += __shfl_xor(before, d);
  return before + blocks_of(rows) <= p.block_room ? Long{rows, (int)before} : Long{0, 0};
}

// Four rows' keys, from `row` (a multiple of four) on; rows from n on are 0.
__device__ __forceinline__ u32x4 keys_at(const ChooseParams& p, const int32_t* table, int h, const Cut& cut, int row) {
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  int at[4] = {0, 0, 0, 0};
  bool ok[4] = {false, false, false, false};
  if (p.quads) {
    const int page = row < cut.rows ? table[row / p.S] : -1;
    if (page >= 0 && page < p.P) {
      const size_t from = ((size_t)page * p.Hkv + h) * p.S + row % p.S;
      const f32x4 x = *(const f32x4*)(p.weights + from);
      const i32x4 y = *(const i32x4*)(p.positions + from);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i], at[i] = y[i], ok[i] = row + i < cut.rows;
    } else if (row < cut.rows) {
      flag_error(RPA_SPARSE_ERR_PAGE);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (row + i >= cut.rows) continue;
      const int page = table[(row + i) / p.S];
      if (page < 0 || page >= p.P) {
        flag_error(RPA_SPARSE_ERR_PAGE);
        continue;
      }
      const size_t from = ((size_t)page * p.Hkv + h) * p.S + (row + i) % p.S;
      w[i] = p.weights[from], at[i] = p.positions[from], ok[i] = true;
    }
  }
  u32x4 key;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    key[i] = !ok[i] ? 0u : at[i] < p.sinks || at[i] >= cut.end - p.recent ? 0xffffffffu : weight_key(w[i]);
  return key;
}

// Rows at the key before the budget and past it, above it and past, below it and before.
struct Tally {
  uint32_t same_low, same_high, more, less;

  __device__ __forceinline__ void rows(int row, const u32x4& key, int n, int budget, uint32_t bound) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (row + u >= n) continue;
      const bool low = row + u < budget, same = key[u] == bound;
      same_low += same && low, same_high += same && !low;
      more += key[u] > bound && !low, less += key[u] < bound && low;
    }
  }
  __device__ __forceinline__ void add(const Tally& o) {
    same_low += o.same_low, same_high += o.same_high, more += o.more, less += o.less;
  }
  __device__ __forceinline__ void of_wave() {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      same_low += __shfl_xor(same_low, d), same_high += __shfl_xor(same_high, d);
      more += __shfl_xor(more, d), less += __shfl_xor(less, d);
    }
  }
};

// Writes a (sequence, head)'s list from some row on, by one wave.
struct Lister {
  int32_t* list;
  const int32_t* table;
  uint32_t bound, rank;       // the key, and how many of the rows at it stay, the lowest
  uint32_t same, late, holes; // rows at the key, rows that move and places for them before the next row

  __device__ __forceinline__ void start(const Tally& before, uint32_t all_low) {
    const uint32_t stay_low = min(rank, all_low);
    same = before.same_low + before.same_high;
    late = before.more + (min(rank, same) > stay_low ? min(rank, same) - stay_low : 0u);
    holes = before.less + before.same_low - min(rank, before.same_low);
  }
  __device__ __forceinline__ uint32_t moved(const Tally& all) const {
    return all.more + min(rank, all.same_low + all.same_high) - min(rank, all.same_low);
  }
  __device__ __forceinline__ void rows(const ChooseParams& p, int row, int lane, const u32x4& key, int end) {  // of the whole wave
    const auto slot_of = [&](int at) {  // -1: no such page
      const int page = table[at / p.S];
      return page >= 0 && page < p.P ? page * p.S + at % p.S : -1;
    };
    int slot = -1;  // of the first, where the four are of one page
    if (p.quads && row < end) slot = slot_of(row);
    const uint64_t below = (1ull << lane) - 1;
    uint32_t mine = same;  // rows at the key before this lane's
    bool is[4];
    uint32_t count = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      is[u] = row + u < end && key[u] == bound;
      const uint64_t votes = __ballot(is[u]);
      mine += __popcll(votes & below), count += __popcll(votes);
    }
    same += count;
    bool comes[4], goes[4];
    uint32_t late_at = late, hole_at = holes;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool there = row + u < end, kept = there && (key[u] > bound || (is[u] && mine < rank));
      mine += is[u];
      comes[u] = kept && row + u >= p.budget, goes[u] = there && !kept && row + u < p.budget;
      const uint64_t a = __ballot(comes[u]), b = __ballot(goes[u]);
      late_at += __popcll(a & below), hole_at += __popcll(b & below);
      late += __popcll(a), holes += __popcll(b);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (!comes[u] && !goes[u]) continue;
      const int at = !p.quads ? slot_of(row + u) : slot < 0 ? -1 : slot + u;
      if (comes[u] && late_at < (uint32_t)p.M) list[2 * (size_t)late_at + 1] = at;
      if (goes[u] && hole_at < (uint32_t)p.M) list[2 * (size_t)hole_at] = at;
      late_at += comes[u], hole_at += goes[u];
    }
  }
};

// Keys of long sequences, and how many of a block's rows have each first digit.
__global__ __launch_bounds__(256) void choose_keys_kernel(ChooseParams p) {
  __shared__ uint32_t s_count[kDigits];
  const int tid = threadIdx.x, h = blockIdx.y % p.Hkv, seq = p.first + blockIdx.y / p.Hkv, first = blockIdx.x * kKeyRows;
  const Cut cut = cut_of(p, seq, false);
  const bool lead = first == 0 && h == 0;
  if (cut.rows <= p.room || first >= cut.rows) {  // uniform
    if (lead && tid == 0) p.longs[seq] = Long{0, 0};
    return;
  }
  const Long its = long_of(p, seq, cut.rows);
  if (lead && tid == 0) p.longs[seq] = its;
  if (!its.rows) return;  // uniform
  for (int i = tid; i < kDigits; i += 256) s_count[i] = 0;
  __syncthreads();
  const size_t block0 = its.block0(p, h);
  uint32_t* const keys = p.keys + block0 * kKeyRows;
#pragma unroll
  for (int i = 0; i < kKeyRows / 1024; ++i) {
    const int row = first + 1024 * i + 4 * tid;
    const u32x4 key = keys_at(p, p.table + (size_t)seq * p.PPS, h, cut, row);
    if (row < cut.rows) *(u32x4*)(keys + row) = key;  // a multiple of four is there
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (row + u < cut.rows) atomicAdd(&s_count[key[u] >> 21], 1u);
  }
  __syncthreads();
  uint32_t* const counts = p.counts + (block0 + blockIdx.x) * kDigits;
  for (int i = tid; i < kDigits; i += 256) counts[i] = s_count[i];
}

struct ChooseShared {
  uint32_t count[kDigits];
  uint32_t sum[16], found[2];
  Tally waves[16];
};

// The digit at which the counts, from the largest digit on, reach `rank`; `prefix` takes it on, `rank` counts on from there.
template <int THREADS>
__device__ __forceinline__ void next_digit(ChooseShared& sh, int bits, uint32_t& prefix, uint32_t& rank) {
  constexpr int kBins = kDigits / THREADS;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  __syncthreads();
  uint32_t own = 0;
  const int top = kDigits - 1 - tid * kBins;  // thread 0 has the last kBins
#pragma unroll
  for (int i = 0; i < kBins; ++i) own += sh.count[top - i];
  uint32_t upto = own;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o = __shfl_up(upto, d);
    upto += lane >= d ? o : 0u;
  }
  if (lane == 63) sh.sum[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += sh.sum[w];
  if (upto - own < rank && rank <= upto) {
    uint32_t above = upto - own;
    int d = top;
    while (above + sh.count[d] < rank) above += sh.count[d--];
    sh.found[0] = prefix << bits | d, sh.found[1] = rank - above;
  }
  __syncthreads();
  prefix = sh.found[0], rank = sh.found[1];
}

// The budget-th largest of keys in LDS (HELD; the first digit brings them there) or of the ledger's, and which one it
// is of the rows at it: its digits one after another.
template <int THREADS, bool HELD>
__device__ __forceinline__ void find_key(const ChooseParams& p, const Cut& cut, int h, const int32_t* table, uint32_t* s_keys,
                                         ChooseShared& sh, uint32_t& prefix, uint32_t& rank) {
  const int tid = threadIdx.x, n = cut.rows;
  prefix = 0, rank = p.budget;
  for (int shift = 21, bits = 11; shift >= 0; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1, bits = shift ? 11 : 10) {
    for (int i = tid; i < kDigits; i += THREADS) sh.count[i] = 0;
    __syncthreads();
    for (int row = 4 * tid; row < n; row += 4 * THREADS) {
      u32x4 key;
      if (!HELD || shift == 21) {
        key = keys_at(p, table, h, cut, row);
        if (HELD) *(u32x4*)(s_keys + row) = key;
      } else {
        key = *(const u32x4*)(s_keys + row);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (row + u < n && (shift == 21 || key[u] >> (shift + bits) == prefix))
          atomicAdd(&sh.count[key[u] >> shift & ((1u << bits) - 1)], 1u);
    }
    next_digit<THREADS>(sh, bits, prefix, rank);
  }
}

// Of a long sequence: the first digit, from the counts of its blocks from block0 on.
template <int THREADS>
__device__ __forceinline__ void first_digit(const ChooseParams& p, int n, size_t block0, ChooseShared& sh) {
  constexpr int kBins = kDigits / THREADS;
  const int tid = threadIdx.x, used = blocks_of(n);
  const uint32_t* const from = p.counts + block0 * kDigits + tid * kBins;
  uint32_t sum[kBins] = {};
#pragma unroll 16
  for (int b = 0; b < used; ++b)
#pragma unroll
    for (int i = 0; i < kBins; ++i) sum[i] += from[(size_t)b * kDigits + i];
#pragma unroll
  for (int i = 0; i < kBins; ++i) sh.count[tid * kBins + i] = sum[i];
  uint32_t prefix = 0, rank = p.budget;
  next_digit<THREADS>(sh, 11, prefix, rank);
  if (tid == 0) p.found[2 * (size_t)blockIdx.x] = prefix, p.found[2 * (size_t)blockIdx.x + 1] = rank;
}

// Long sequences: the keys that have it, each wave's at the beginning of its rows'.
__global__ __launch_bounds__(256) void choose_near_kernel(ChooseParams p) {
  const int lane = threadIdx.x % 64, segment = blockIdx.x * 4 + threadIdx.x / 64, from = segment * kSegment + 4 * lane;
  const int seq = p.first + blockIdx.y / p.Hkv, h = blockIdx.y % p.Hkv;
  const Long its = p.longs[seq];
  const uint32_t prefix = p.found[2 * ((size_t)seq * p.Hkv + h)];  // beside it; of no meaning where there are no rows
  const int n = its.rows;
  if (segment * kSegment >= n) return;
  const size_t block0 = its.block0(p, h);
  const uint32_t* const keys = p.keys + block0 * kKeyRows;
  uint32_t* const to = p.near + block0 * kKeyRows + segment * kSegment;
  u32x4 key[kSegment / 256];
#pragma unroll
  for (int x = 0; x < kSegment / 256; ++x)
    if (from + 256 * x < n) key[x] = *(const u32x4*)(keys + from + 256 * x);
  uint32_t held = 0;
#pragma unroll
  for (int x = 0; x < kSegment / 256; ++x)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool is = from + 256 * x + u < n && key[x][u] >> 21 == prefix;
      const uint64_t votes = __ballot(is);
      if (is) to[held + __popcll(votes & ((1ull << lane) - 1))] = key[x][u];
      held += __popcll(votes);
    }
  if (lane == 0) p.held[block0 * (kKeyRows / kSegment) + segment] = held;
}

// Long sequences: the other digits, from those keys, a segment a wave at a time.
__global__ __launch_bounds__(1024) void choose_last_kernel(ChooseParams p) {
  constexpr int kAhead = 8;  // segments whose first keys are in flight
  __shared__ ChooseShared sh;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = p.longs[blockIdx.x / p.Hkv].rows;
  if (!n) return;  // uniform
  const size_t block0 = p.longs[blockIdx.x / p.Hkv].block0(p, blockIdx.x % p.Hkv);
  const int segments = (n + kSegment - 1) / kSegment;
  const uint32_t *const held = p.held + block0 * (kKeyRows / kSegment), *const keys = p.near + block0 * kKeyRows;
  uint32_t prefix = p.found[2 * (size_t)blockIdx.x], rank = p.found[2 * (size_t)blockIdx.x + 1];
  for (int shift = 10, bits = 11; shift >= 0; shift -= 10, bits = 10) {
    for (int i = tid; i < kDigits; i += 1024) sh.count[i] = 0;
    __syncthreads();
    const auto count = [&](uint32_t key) {
      if (key >> (shift + bits) == prefix) atomicAdd(&sh.count[key >> shift & ((1u << bits) - 1)], 1u);
    };
    for (int base = wave; base < segments; base += 16 * kAhead) {
      uint32_t most[kAhead], key[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int segment = base + 16 * x;
        most[x] = segment < segments ? held[segment] : 0;
        if (segment < segments) key[x] = keys[(size_t)segment * kSegment + lane];  // counted or not: a segment has its room
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        if ((uint32_t)lane < most[x]) count(key[x]);
        for (uint32_t i = lane + 64; i < most[x]; i += 64) count(keys[(size_t)(base + 16 * x) * kSegment + i]);
      }
    }
    next_digit<1024>(sh, bits, prefix, rank);
  }
  if (tid == 0) p.found[2 * (size_t)blockIdx.x] = prefix, p.found[2 * (size_t)blockIdx.x + 1] = rank;
}

// The list of rows whose keys are in LDS (HELD) or the ledger's: every wave has a stretch of rows.
template <int THREADS, bool HELD>
__device__ __forceinline__ int list_rows(const ChooseParams& p, const Cut& cut, int h, const uint32_t* s_keys, ChooseShared& sh,
                                         Lister out) {
  constexpr int kWaves = THREADS / 64;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = cut.rows;
  const auto key_at = [&](int row) { return HELD ? *(const u32x4*)(s_keys + row) : keys_at(p, out.table, h, cut, row); };
  const int stretch = ((n + kWaves - 1) / kWaves + 255) / 256 * 256, from = min(wave * stretch, n), to = min(from + stretch, n);
  Tally own = {};
  for (int row = from + 4 * lane; row < to; row += 256) own.rows(row, key_at(row), n, p.budget, out.bound);
  own.of_wave();
  if (lane == 0) sh.waves[wave] = own;
  __syncthreads();
  Tally before = {}, all = {};
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before.add(sh.waves[w]);
    all.add(sh.waves[w]);
  }
  out.start(before, all.same_low);
  for (int base = from; base < to; base += 256) {
    const int row = base + 4 * lane;
    out.rows(p, row, lane, row < to ? key_at(row) : u32x4{0, 0, 0, 0}, to);
  }
  const uint32_t moved = out.moved(all);
  if (moved > (uint32_t)p.M && tid == 0) flag_error(RPA_SPARSE_ERR_LEN);
  return (int)min(moved, (uint32_t)p.M);
}

// One workgroup a (kv head, sequence).  A step's loads are of 256 rows a wave, four neighbouring rows a lane.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void choose_rows_kernel(ChooseParams p) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ ChooseShared s_rest;
  const int h = blockIdx.x % p.Hkv, seq = blockIdx.x / p.Hkv;
  const int32_t* const table = p.table + (size_t)seq * p.PPS;
  int32_t* const list = p.moves + (size_t)blockIdx.x * p.M * 2;
  const Long its = THREADS == 1024 && p.block_room ? p.longs[seq] : Long{0, 0};
  const Cut cut = cut_of(p, seq, threadIdx.x == 0);
  uint32_t bound, rank;
  int done = 0;  // entries of the list
  if (THREADS == 1024 && cut.rows > p.room) {
    if (its.rows) return first_digit<THREADS>(p, its.rows, its.block0(p, h), s_rest);  // the rest by blocks
    find_key<THREADS, false>(p, cut, h, table, s_keys, s_rest, bound, rank);
    done = list_rows<THREADS, false>(p, cut, h, s_keys, s_rest, Lister{list, table, bound, rank});
  } else if (cut.rows) {
    find_key<THREADS, true>(p, cut, h, table, s_keys, s_rest, bound, rank);
    done = list_rows<THREADS, true>(p, cut, h, s_keys, s_rest, Lister{list, table, bound, rank});
  }
  for (long long i = 2ll * done + threadIdx.x; i < 2ll * p.M; i += THREADS) list[i] = -1;
}

// Long sequences' lists, by blocks of kKeyRows: a wave has a quarter of a block.  First the blocks' tallies, then,
// with those of the blocks before, the list.
template <bool LIST>
__global__ __launch_bounds__(256) void choose_list_kernel(ChooseParams p) {
  constexpr int kSteps = kKeyRows / 1024;
  __shared__ Tally s_waves[4], s_before[4], s_all[4];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, seq = p.first + blockIdx.y / p.Hkv, h = blockIdx.y % p.Hkv;
  const Long its = p.longs[seq];
  const size_t of = (size_t)seq * p.Hkv + h;
  const uint32_t bound = p.found[2 * of], rank = p.found[2 * of + 1];
  const int n = its.rows, used = blocks_of(n), block = blockIdx.x;
  if (block >= used) return;  // uniform
  const size_t block0 = its.block0(p, h);
  Tally* const tallies = (Tally*)p.tallies + block0;
  const uint32_t* const keys = p.keys + block0 * kKeyRows;
  const int from = block * kKeyRows + wave * (kKeyRows / 4) + 4 * lane;
  u32x4 key[kSteps];
#pragma unroll
  for (int x = 0; x < kSteps; ++x) key[x] = from + 256 * x < n ? *(const u32x4*)(keys + from + 256 * x) : u32x4{0, 0, 0, 0};
  Tally before = {}, all = {};  // of the blocks
  if (LIST) {
    for (int b = tid; b < used; b += 256) {
      const Tally one = tallies[b];
      if (b < block) before.add(one);
      all.add(one);
    }
    before.of_wave(), all.of_wave();
    if (lane == 0) s_before[wave] = before, s_all[wave] = all;
  }
  Tally own = {};
#pragma unroll
  for (int x = 0; x < kSteps; ++x) own.rows(from + 256 * x, key[x], n, p.budget, bound);
  own.of_wave();
  if (lane == 0) s_waves[wave] = own;
  __syncthreads();
  if (!LIST) {
    if (tid) return;
    for (int w = 1; w < 4; ++w) own.add(s_waves[w]);
    tallies[block] = own;
    return;
  }
  before = all = Tally{};
  for (int w = 0; w < 4; ++w) {
    before.add(s_before[w]), all.add(s_all[w]);
    if (w < wave) before.add(s_waves[w]);
  }
  int32_t* const list = p.moves + of * p.M * 2;
  Lister out = {list, p.table + (size_t)seq * p.PPS, bound, rank};
  out.start(before, all.same_low);
#pragma unroll
  for (int x = 0; x < kSteps; ++x) out.rows(p, from + 256 * x, lane, key[x], n);
  const uint32_t moved = out.moved(all);
  if (block == 0 && tid == 0 && moved > (uint32_t)p.M) flag_error(RPA_SPARSE_ERR_LEN);
  const long long done = min(moved, (uint32_t)p.M);
  for (long long i = 2 * done + block * 256 + tid; i < 2ll * p.M; i += 256ll * used) list[i] = -1;
}

struct MoveParams {
  const int32_t* moves;
  const float* scales;
  uint8_t* kv;
  float* weights;
  int32_t* positions;
  long long rows;            // P * S
  int entries;               // of all lists
  int M, Hkv, S, chunks;     // chunks: 16 bytes each, of a head's key and value row, which lie together
};

constexpr int kMoveEntries = 16;  // of a wave

// One entry a wave took 57 us where this takes 19 (the six fp8 prompts), as slots, scales and rows are a chain of loads.
// A wave takes kMoveEntries entries of the lists: their slots, scales and ledger entries a lane each, then their rows,
// LANES lanes a row, four loads in flight.
template <bool FP8, int LANES>
__global__ __launch_bounds__(256) void move_kernel(MoveParams p) {
  constexpr int kRows = 64 / LANES, kTurns = kMoveEntries / kRows, kHold = kTurns < 4 ? kTurns : 4;
  const int lane = threadIdx.x % 64, first = (blockIdx.x * 4 + threadIdx.x / 64) * kMoveEntries;
  const int entry = first + lane;
  int to = -1, from = -1, h = 0;
  if (lane < kMoveEntries && entry < p.entries) {
    const u32x2 slots = *(const u32x2*)(p.moves + 2 * (size_t)entry);
    to = (int)slots[0], from = (int)slots[1];
    h = entry / p.M % p.Hkv;
  }
  bool live = to >= 0 && from >= 0;
  if (live && (to >= p.rows || from >= p.rows)) {
    flag_error(RPA_SPARSE_ERR_SLOT);
    live = false;
  }
  if (!__ballot(live)) return;
  float ratio_from[2] = {1.f, 1.f}, ratio_to[2] = {1.f, 1.f};  // the K and V scales there and here
  if (live) {
    const size_t head_from = (size_t)(from / p.S) * p.Hkv + h, head_to = (size_t)(to / p.S) * p.Hkv + h;
    const size_t a = head_from * p.S + from % p.S, b = head_to * p.S + to % p.S;
    const float weight = p.weights[a];
    const int position = p.positions[a];
    if (FP8 && p.scales) {
#pragma unroll
      for (int i = 0; i < 2; ++i) ratio_from[i] = p.scales[2 * head_from + i], ratio_to[i] = p.scales[2 * head_to + i];
    }
    p.weights[b] = weight;
    p.positions[b] = position;
  }
  const int c = lane % LANES, part = 2 * c >= p.chunks;
  const size_t row_bytes = 16ull * p.chunks;
#pragma unroll
  for (int turn = 0; turn < kTurns; turn += kHold) {
    u32x4 w[kHold];
    int dst[kHold], head[kHold];
    float there[kHold], here[kHold];
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      const int e = (turn + u) * kRows + lane / LANES;
      const int src = __shfl(from, e), place = __shfl(live ? to : -1, e);
      dst[u] = c < p.chunks ? place : -1;
      head[u] = __shfl(h, e);
      if (FP8) {
        const float k0 = __shfl(ratio_from[0], e), v0 = __shfl(ratio_from[1], e);
        const float k1 = __shfl(ratio_to[0], e), v1 = __shfl(ratio_to[1], e);
        there[u] = part ? v0 : k0, here[u] = part ? v1 : k1;
      }
      if (dst[u] >= 0) w[u] = *(const u32x4*)(p.kv + ((size_t)src * p.Hkv + head[u]) * row_bytes + 16 * c);
    }
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      if (dst[u] < 0) continue;
      if (FP8 && there[u] != here[u]) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          fp8_values(u32x2{w[u][2 * i], w[u][2 * i + 1]}, there[u], x);
          const u32x2 codes = fp8_codes(x, here[u]);
          w[u][2 * i] = codes[0], w[u][2 * i + 1] = codes[1];
        }
      }
      *(u32x4*)(p.kv + ((size_t)dst[u] * p.Hkv + head[u]) * row_bytes + 16 * c) = w[u];
    }
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
  if ((long long)s->max_num_seqs * s->num_kv_heads > 0x7fffffff / 1024)
    return fail(RPA_E_UNSUPPORTED, "more lists than one launch takes");
  return RPA_OK;
}

struct ChoosePlan {
  int threads, room;
  int blocks, block_room;  // of the longest sequence that the table has room for (0: all keys fit LDS), and of the workspace
  size_t longs, keys, near, held, counts, tallies, bytes;  // where each begins
};

// Waves of a workgroup: sixteen while every list has a CU to itself (256 lists of 4096 rows: 13.0 us, 16.6 with four; of
// 8192: 16.8 and 27.1), four where lists share one (512 of 4096: 24.1 and 19.3; of 8192: 35.0 and 33.2) or rows are
// few, sixteen again past 8192 rows (512 of 16384: 52 and 57; of 24576: 69 and 137, as LDS holds one list either way).
ChoosePlan plan_choose(const rpa_choose_shape_t& s) {
  ChoosePlan r = {};
  const long long capacity = (long long)s.pages_per_seq * s.page_size;
  r.threads = capacity > (s.max_num_seqs * (long long)s.num_kv_heads <= 256 ? 1024 : 8192) ? 1024 : 256;
  r.room = (int)((capacity < kChooseRows ? capacity : kChooseRows) + 3) / 4 * 4;
  if (capacity > kChooseRows) {
    const long long N = s.max_num_seqs, rows = (long long)s.total_pages * s.page_size;
    r.blocks = (int)((capacity + kKeyRows - 1) / kKeyRows);
    // distinct pages: long sequences have at most the pool's rows, and each all but one of its blocks whole
    const long long most = rows / (kChooseRows + 1), longest = N < most ? N : most;
    const long long by_pool = (rows + (kKeyRows - 1) * longest) / kKeyRows, by_table = N * r.blocks;
    r.block_room = (int)(by_pool < by_table ? by_pool : by_table);
    if (!longest) r.block_room = 0;
    const size_t lists = (size_t)N * s.num_kv_heads, room = (size_t)r.block_room * s.num_kv_heads;
    r.longs = (lists * 8 + 15) / 16 * 16;
    r.keys = r.longs + ((size_t)N * sizeof(Long) + 15) / 16 * 16;
    r.near = r.keys + room * kKeyRows * 4;
    r.held = r.near + room * kKeyRows * 4;
    r.counts = r.held + room * (kKeyRows / kSegment) * 4;
    r.tallies = r.counts + room * kDigits * 4;
    r.bytes = r.tallies + room * sizeof(Tally);
  }
  return r;
}

long long move_groups(long long entries) { return (entries + 4 * kMoveEntries - 1) / (4 * kMoveEntries); }

int check_move(const rpa_move_shape_t* s) {
  if (!s) return fail(RPA_E_INVALID, "shape is NULL");
  if (s->num_lists < 0 || s->max_moves <= 0) return fail(RPA_E_INVALID, "non-positive dimension in shape");
  int rc = check_heads(s->num_kv_heads, s->head_dim, s->kv_dtype);
  if (rc || (rc = check_pool(s->total_pages, s->page_size))) return rc;
  const __int128 entries = (__int128)s->num_lists * s->num_kv_heads * s->max_moves;
  if (entries > kMostIndex) return fail(RPA_E_UNSUPPORTED, "more rows than one launch takes");
  return check_launch(move_groups((long long)entries), 256);
}

}  // namespace
}  // namespace rpa_sparse
