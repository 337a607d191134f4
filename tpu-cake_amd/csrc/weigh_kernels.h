// Attention over a paged cache that accounts for the weight each key got.
//
// Mathematics: o_t = sum_x p_tx v_x, p_tx = 2^(s_tx - m_t) / l_t over the keys x up to token t's position (log2 domain),
// and for each key the sum of p_tx over the step's tokens and the group's heads.  The row's maximum m and sum l are
// known only once every key has been seen, so weights take the scores a second time.
//
// Rows (sequences of one token) leave their scores, 4 bytes a (head, key), and the launch after them makes weights of
// those; prompt chunks multiply K once more instead, which costs less than what a chunk's scores would weigh.  Launches: rows,
// tiles (where a step may have chunks), joins of parts with the weights of rows, weights of chunks.
//
// HBM bounds rows.  64 sequences of 1024 to 8192 keys, 64 heads of 128 over 8, bf16: 855 MB, 136 us at the 6.3 TB/s of a plain
// read; 191 to 198 us, of which rows 170 (845 MB read, 52 MB of scores and 10 MB of parts written: 5.3 TB/s) and weights 24.
// Without their scores rows took 136, without any product 132 to 140: it is the mixed stores that cost.  Two sequences of
// 245 000 keys, 32 heads, fp8 pages of 16: 1.03 GB, 163 us; 277, of which rows 249 (4.3 TB/s; their loads alone take 195, the
// conversions and the three products of P do not hide entirely) and weights 36.
//
// Tried for rows and not kept: loads that stay in the caches (191 us where nontemporal ones take 168); a barrier that
// keeps the heads' waves at the same keys (195 and 191; fp8 230 and 195 for the loads); scores through LDS, at other
// places or with other cache policies (the same).
#pragma once

#include "attend_kernels.h"

namespace rpa_sparse {
namespace {

// v / d for 0 <= v < 2^31: (v * m) >> (31 + s) with s = ceil(log2 d), m = floor(2^(31 + s) / d) + 1.  m d is past
// 2^(31 + s) by at most 2^s, so the quotient is exact.
struct Divisor {
  uint32_t m;
  int shift;
};
Divisor divisor(int d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return {(uint32_t)((1ull << (31 + s)) / (uint32_t)d + 1), 31 + s};
}
__device__ __forceinline__ int div_by(int v, Divisor d) { return (int)(((uint64_t)(uint32_t)v * d.m) >> d.shift); }

// A load that nothing else will want.
__device__ __forceinline__ u32x4 load16_once(global_bytes at) {
  return __builtin_nontemporal_load((const __attribute__((address_space(1))) u32x4*)at);
}

constexpr int kWeighWaves = 4, kWeighThreads = 64 * kWeighWaves;
constexpr int kMostWaves = 8;  // of a workgroup of rows

struct WeighParams {
  const uint16_t* q;
  const uint8_t* kv;
  const float* scales;
  const int32_t *kv_lens, *table, *cu, *num_seqs, *dropped;
  float* weights;
  int32_t* positions;
  uint16_t* out;
  float2* stats;  // (m, 1 / l) of every token and head
  float* scores;
  long long score_room;  // blocks of 16 keys
  struct JoinOf* joins;  // for each workgroup of rows, then of tiles
  float* parts;   // two for each workgroup: (m, l) of 16 rows, then the rows' O
  long long q_token, q_head;
  int T, Hkv, G, D, P, S, N, PPS;
  int tiles;      // 16-head tiles of a group
  int near, ways; // rows: kv heads of a workgroup, waves that share a head's keys
  int block_shift;  // log2 of the keys of a block of rows' work: two units of 32 for each wave of a head
  int rows_grid, tiles_grid;  // workgroups of rows and of tiles
  int few;        // at most kFewSeqs sequences, and all sums of work fit 32 bits
  int one_page;   // 32 keys from a multiple of 32 on lie in one page
  int quads;      // four neighbouring weights from a multiple of four on are 16 aligned bytes
  int chunk;      // sequences of more than one token are done in tiles
  float* tile_parts;  // of tiles: two for each workgroup, (m, l) of kColumns columns, then their O
  Divisor page, group;
  float scale, cap, v_scale, decay;  // scale: of q.k; times log2 e where cap is 0
};

// What a workgroup leaves to be joined: the row (of `near` kv heads from h on) or tile that ends in its share and began in
// workgroup `first`'s; first -1: none.
struct alignas(32) JoinOf {
  int first;
  int late;  // the first one's part is its slot 1
  int t, h;  // rows: the token; tiles: the sequence's first
  int tile;  // rows: of 16 heads; tiles: of kColumns columns
  int rows;  // tiles: the sequence's rows
};

struct Sequence {
  int first, tokens, keys;  // its first token, its tokens, its keys
};

// Sequence i, its offsets taken into [0, T] and its length into the page table.
__device__ __forceinline__ Sequence sequence_at(const WeighParams& p, int i, bool flag = false) {
  const int begin = min(max(p.cu[i], 0), p.T), end = min(max(p.cu[i + 1], 0), p.T), len = max(p.kv_lens[i], 0);
  const int capacity = p.PPS * p.S;
  if (flag && len > capacity && end > begin) flag_error(RPA_SPARSE_ERR_LEN);
  return {begin, max(end - begin, 0), min(len, capacity)};
}

// Scores of a sequence with one token, which its weights take instead of K once more: blocks of 16 keys, of which
// [kv head][head of the group][key].  They are kept while they fit the workspace, which holds all that distinct pages can
// have.
__device__ __forceinline__ long long score_blocks(const Sequence& s) { return s.tokens == 1 ? (s.keys + 15) / 16 : 0; }
__device__ __forceinline__ bool scores_fit(const WeighParams& p, const Sequence& s, long long before) {
  return s.tokens == 1 && before + score_blocks(s) <= p.score_room;
}

// Rows' work: the blocks of keys of a row, and those of all rows of a sequence.
__device__ __forceinline__ int row_blocks(const WeighParams& p, const Sequence& s) { return max((s.keys + (1 << p.block_shift) - 1) >> p.block_shift, 1); }
__device__ __forceinline__ bool in_tiles(const WeighParams& p, const Sequence& s, bool pad) { return p.chunk && s.tokens > 1 && !pad; }
__device__ __forceinline__ long long row_units(const WeighParams& p, const Sequence& s, bool pad) {
  return in_tiles(p, s, pad) ? 0 : (long long)s.tokens * (p.Hkv / p.near) * p.tiles * row_blocks(p, s);
}

// A workgroup's share of all the work: sequences in order, and behind them (`pad`) the tokens past the last one; the
// total in shares of equal size.
struct Share {
  int index;           // of the shares in order
  long long from, to;  // units
  int seq, count;      // the sequence that `from` lies in, of how many
  Sequence s;
  long long before, scores, rows;  // before it: units, blocks of scores, units of rows
  long long row_total, total;      // units of rows, and of all the work
};

// Sequence i of `count`, in the order of the work.
__device__ __forceinline__ Sequence work_sequence(const WeighParams& p, int count, int i) {
  if (i < count) return sequence_at(p, i);
  const int end = count ? min(max(p.cu[count], 0), p.T) : 0;
  return {end, p.T - end, 0};
}

// The index of a workgroup's share, of as many as hold anything.  NEAR: XCDs take workgroups in turn; neighbouring shares,
// which read the same keys, go to one of them.
template <bool NEAR>
__device__ __forceinline__ int share_index(int block, int blocks, int used) {
  if (!NEAR) return block;
  const int xcd = block % 8;
  return block < used ? xcd * (used / 8) + min(xcd, used % 8) + block / 8 : blocks;
}

// As share_of, where there are at most kFewSeqs sequences and all sums fit 32 bits: each wave by itself, four sequences a
// lane, without LDS or a barrier.  Four short sequences' call takes 18.0 us with it, 19.5 without.
constexpr int kFewSeqs = 255;

template <bool NEAR, typename Amount>
__device__ __forceinline__ Share share_of_few(const WeighParams& p, int block, int blocks, Amount amount, bool flag) {
  constexpr int kEach = (kFewSeqs + 64) / 64;
  const int lane = threadIdx.x % 64, capacity = p.PPS * p.S, each = p.N / 64 + 1;
  int c0[kEach], c1[kEach], len[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = min(lane * each + k, p.N);
    c0[k] = p.cu[i], c1[k] = p.cu[min(i + 1, p.N)], len[k] = p.kv_lens[min(i, p.N - 1)];
  }
  const int count = min(max(*p.num_seqs, 0), p.N);
  Sequence s[kEach];
  int units[kEach][3], own[3] = {0, 0, 0};
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = lane * each + k, begin = min(max(c0[k], 0), p.T), end = min(max(c1[k], 0), p.T);
    const bool ok = k < each && i < count, pad = k < each && i == count;
    s[k] = {pad && !count ? 0 : begin, ok ? max(end - begin, 0) : pad ? p.T - (count ? begin : 0) : 0, ok ? min(max(len[k], 0), capacity) : 0};
    if (flag && ok && s[k].tokens && len[k] > capacity) flag_error(RPA_SPARSE_ERR_LEN);
    units[k][0] = (int)amount(s[k], pad), units[k][1] = ok ? (int)score_blocks(s[k]) : 0, units[k][2] = (int)row_units(p, s[k], pad);
#pragma unroll
    for (int u = 0; u < 3; ++u) own[u] += units[k][u];
  }
  int upto[3] = {own[0], own[1], own[2]};
#pragma unroll
  for (int d = 1; d < 64; d *= 2)
#pragma unroll
    for (int u = 0; u < 3; ++u) {
      const int o = __shfl_up(upto[u], d);
      upto[u] += lane >= d ? o : 0;
    }
  const int total = __builtin_amdgcn_readlane(upto[0], 63), row_total = __builtin_amdgcn_readlane(upto[2], 63);
  const int each_share = (int)(((long long)total + blocks - 1) / blocks);
  const int index = total ? share_index<NEAR>(block, blocks, (total + each_share - 1) / each_share) : block;
  const int from = (int)min((long long)index * each_share, (long long)total), to = min(from + each_share, total);
  if (from >= to) return Share{0, 0, 0, 0, 0, {0, 0, 0}, 0, 0, 0, 0, total};
  int before[3] = {upto[0] - own[0], upto[1] - own[1], upto[2] - own[2]}, at = 0;
  const int hit = __builtin_ctzll(__ballot(from >= before[0] && from < upto[0]));
  Sequence mine = s[0];
  bool past = true;  // of the sequences so far
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    past = past && k < each && from >= before[0] + units[k][0];
    if (past) {
#pragma unroll
      for (int u = 0; u < 3; ++u) before[u] += units[k][u];
      at = k + 1;
      if (k + 1 < kEach) mine = s[k + 1];
    }
  }
  const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, hit); };
  return Share{index, from, to, hit * each + of(at), count, {of(mine.first), of(mine.tokens), of(mine.keys)}, of(before[0]), of(before[1]),
               of(before[2]), row_total, total};
}

// amount(sequence, pad): its units.
template <bool NEAR, typename Amount>
__device__ __forceinline__ Share share_of(const WeighParams& p, int block, int blocks, Amount amount, bool flag = false) {
  if (p.few) return share_of_few<NEAR>(p, block, blocks, amount, flag);
  __shared__ long long s_sum[3][kMostWaves];
  __shared__ Share s_share;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, waves = blockDim.x / 64, capacity = p.PPS * p.S;
  const int each = p.N / (int)blockDim.x + 1, i0 = min(tid * each, p.N + 1), i1 = min(i0 + each, p.N + 1);
  // the first of this thread's sequences, loaded beside their number
  const int c0 = p.cu[min(i0, p.N)], c1 = p.cu[min(i0 + 1, p.N)], len0 = p.kv_lens[min(i0, p.N - 1)];
  const int count = min(max(*p.num_seqs, 0), p.N);
  const auto sequence = [&](int i) {
    if (i > count) return Sequence{0, 0, 0};
    if (i != i0) return work_sequence(p, count, i);
    const int begin = min(max(c0, 0), p.T), end = min(max(c1, 0), p.T);
    return i < count ? Sequence{begin, max(end - begin, 0), min(max(len0, 0), capacity)}
                     : Sequence{count ? begin : 0, p.T - (count ? begin : 0), 0};
  };
  long long own[3] = {0, 0, 0};
  for (int i = i0; i < i1; ++i) {
    const Sequence s = sequence(i);
    if (flag && i < count && s.tokens && (i == i0 ? len0 : p.kv_lens[i]) > capacity) flag_error(RPA_SPARSE_ERR_LEN);
    own[0] += amount(s, i == count), own[2] += row_units(p, s, i == count);
    own[1] += i < count ? score_blocks(s) : 0;
  }
  long long upto[3] = {own[0], own[1], own[2]}, total[3] = {0, 0, 0};
#pragma unroll
  for (int d = 1; d < 64; d *= 2)
#pragma unroll
    for (int u = 0; u < 3; ++u) {
      const long long o = __shfl_up(upto[u], d);
      upto[u] += lane >= d ? o : 0;
    }
#pragma unroll
  for (int u = 0; u < 3; ++u)
    if (lane == 63) s_sum[u][wave] = upto[u];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 3; ++u)
    for (int w = 0; w < waves; ++w) {
      upto[u] += w < wave ? s_sum[u][w] : 0;
      total[u] += s_sum[u][w];
    }
  const long long each_share = (total[0] + blocks - 1) / blocks;
  const int index = total[0] ? share_index<NEAR>(block, blocks, (int)((total[0] + each_share - 1) / each_share)) : block;
  const long long from = min(index * each_share, total[0]), to = min(from + each_share, total[0]);
  if (from < to && from >= upto[0] - own[0] && from < upto[0]) {
    long long before[3] = {upto[0] - own[0], upto[1] - own[1], upto[2] - own[2]};
    int i = i0;
    Sequence s = sequence(i);
    for (long long a; from >= before[0] + (a = amount(s, i == count)); s = sequence(++i))
      before[0] += a, before[1] += i < count ? score_blocks(s) : 0, before[2] += row_units(p, s, i == count);
    s_share = {index, from, to, i, count, s, before[0], before[1], before[2], total[2], total[0]};
  }
  __syncthreads();
  if (from < to) return s_share;
  return Share{0, 0, 0, 0, 0, {0, 0, 0}, 0, 0, 0, 0, total[0]};
}

// The parts of a row that several workgroups had: those of workgroups first .. last.
struct RowParts {
  int first, last;
  bool late;  // the first one's is its slot 1
};
// begin: the row's first unit.
__device__ __forceinline__ RowParts row_parts(const WeighParams& p, long long total, long long begin, int blocks) {
  const long long each = (total + p.rows_grid - 1) / p.rows_grid;
  const int first = (int)(begin / each);
  return {first, (int)((begin + blocks - 1) / each), begin != first * each};
}
// head: of the `near` ones
__device__ __forceinline__ const float* row_part(const WeighParams& p, const RowParts& r, int w, int head) {
  return p.parts + ((2 * (size_t)w + (w == r.first && r.late)) * p.near + head) * (32 + 16 * (size_t)p.D);
}

// Rows: a token's heads, up to 16 of one kv head, as the columns of v_mfma_f32_16x16x32_bf16.  A workgroup takes the rows of
// `near` kv heads, a wave each (where there are few, `ways` waves share a head's keys): a key's rows of all these heads
// lie together, and the waves walk the same keys.  Keys come in blocks, the blocks of all rows in equal shares, one a
// workgroup: a long sequence's rows are spread over as many workgroups as their blocks need, and short ones' share a
// workgroup.  A row that a workgroup does not have whole leaves a part: the first in the workgroup's slot 0, the last in slot 1.
//
// bf16: a wave reads a key's K and V row, which lie together, in whole lines, a unit of 32 keys ahead, and takes both through
// LDS; fp8 K comes straight into the product's operand, 64 bytes of 16 keys at a time.  P goes into its product in three
// bf16 parts, 24 bits: rounded to one it would be off by 2^-9, and two lose what large values leave of small differences.
template <int DP, bool FULL, bool FP8>
__global__ __launch_bounds__(DP == 256 ? 256 : 64 * kMostWaves, DP == 256 ? 1 : 2) void weigh_rows_kernel(WeighParams p) {
  constexpr int kKRow = DP * 2 + 16, kVRow = DP * 2 + 32;
  constexpr int kV = FP8 ? 0 : 32 * kKRow;             // V behind K
  constexpr int kWave = kV + 32 * kVRow;               // a wave's LDS; later its 16 rows of O in fp32
  constexpr int kORow = DP + 4;
  constexpr int kElem = FP8 ? 1 : 2;
  constexpr int kSteps = DP / 32;
  constexpr int kChunks = DP / 4, kApart = 64 / kChunks, kLoads = 32 / kApart;  // bf16: chunks of a key, keys of a load
  constexpr int kCodes = DP / 64;                      // fp8: loads of a lane for a key row's K (or V)
  constexpr int kSets = FP8 ? 2 : 1;
  static_assert(16 * kORow * 4 <= kWave, "O rows fit the wave's region");
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ float s_m[kMostWaves][16], s_l[kMostWaves][16];
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 16, j = lane / 16;
  const int threads = blockDim.x, groups = p.Hkv / p.near;
  const Share share =
      share_of<false>(p, blockIdx.x, gridDim.x, [&](const Sequence& s, bool pad) { return row_units(p, s, pad); });
  if (share.from == share.to) {
    if (tid == 0) p.joins[blockIdx.x].first = -1;
    return;
  }

  const int row_bytes = p.D * kElem, mine = wave % p.near, way = wave / p.near;
  const uint64_t row_stride = 2ull * p.Hkv * row_bytes;
  const global_bytes zero = zero_row();
  uint8_t* const own_lds = lds + wave * kWave;
  const int count = share.count;
  int seq = share.seq;
  Sequence s = share.s;
  long long before = share.before, at = share.from, score_at = share.scores;
  while (at < share.to) {
    for (long long units; at >= before + (units = row_units(p, s, seq == count));) {
      before += units;
      score_at += seq < count ? score_blocks(s) : 0;
      s = work_sequence(p, count, ++seq);
    }
    const int blocks = row_blocks(p, s);
    const long long row = (at - before) / blocks;
    const int first_block = (int)(at - before - row * blocks);
    const int end_block = (int)min((long long)blocks, first_block + (share.to - at));
    const int token = (int)(row / (groups * p.tiles)), group_tile = (int)(row - (long long)token * (groups * p.tiles));
    const int h = group_tile / p.tiles * p.near + mine, tile = group_tile % p.tiles, t = s.first + token;
    const int keys = max(s.keys - (s.tokens - 1 - token), 0);
    const bool known = seq < count;
    const int32_t* const table = p.table + (size_t)(known ? seq : 0) * p.PPS;

    bf16x8 q[kSteps];
    {
      const int head = tile * 16 + n;
      const uint16_t* src = p.q + t * p.q_token + ((long long)h * p.G + head) * p.q_head;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int dim = FP8 ? 64 * (i / 2) + 16 * j + 8 * (i % 2) : 32 * i + 8 * j;
        u32x4 w = {0, 0, 0, 0};
        if (head < p.G && (FULL || dim < p.D)) w = *(const u32x4*)(src + dim);
        q[i] = __builtin_bit_cast(bf16x8, w);
      }
    }
    const global_bytes rows = (global_bytes)(uint64_t)p.kv + 2 * (size_t)h * row_bytes;
    const int end_key = (int)min((long long)keys, (long long)end_block << p.block_shift), end_unit = (end_key + 31) / 32;
    const bool keep = known && scores_fit(p, s, score_at);
    float* const scores = p.scores + ((size_t)score_at * p.Hkv + h) * p.G * 16;
    // Loads in flight: of bf16 the unit after the one in LDS, of fp8 (half the bytes) two units.
    struct {
      u32x4 w[FP8 ? 4 * kCodes : kLoads];
      int id;            // the page of key lane % 32, found before the set's last unit was loaded
      uint32_t seen;     // which keys of the loaded unit exist
      float ks, vs;      // fp8: the scales of key lane % 32
    } set[kSets];
    const auto find = [&](int x, int unit) {
      const int key = max(min(unit * 32 + lane % 32, end_key - 1), 0);
      set[x].id = table[div_by(key, p.page)];
    };
    const auto load = [&](int x, int unit) {
      const int key = unit * 32 + lane % 32, id = set[x].id;
      u32x4* const w = set[x].w;
      const bool ok = key < end_key && id >= 0 && id < p.P;
      if (key < end_key && !ok) flag_error(RPA_SPARSE_ERR_PAGE);
      const int slot = ok ? id * p.S + (key - div_by(key, p.page) * p.S) : -1;
      const uint32_t seen = set[x].seen = (uint32_t)__ballot(ok);
      if (FP8) {
        if (p.scales) {
          const float2 scale = *(const float2*)(p.scales + ((size_t)(ok ? id : 0) * p.Hkv + h) * 2);
          set[x].ks = ok ? scale.x : 1.f, set[x].vs = ok ? scale.y : 1.f;
        } else {
          set[x].ks = set[x].vs = 1.f;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int at_slot = __shfl(slot, 16 * b + n);
          const global_bytes src = at_slot >= 0 ? rows + (uint32_t)at_slot * row_stride : zero;
#pragma unroll
          for (int i = 0; i < kCodes; ++i) {
            const int byte = 64 * i + 16 * j;
            const global_bytes from = FULL || byte < row_bytes ? src : zero;
            w[2 * kCodes * b + i] = load16_once(from + byte);
            w[2 * kCodes * b + kCodes + i] = load16_once(from + row_bytes + byte);
          }
        }
      } else {
        const int c = lane % kChunks, part = c >= kChunks / 2, byte = 16 * (c - part * (kChunks / 2));
        const bool inside = FULL || byte < row_bytes;
        if (p.one_page && seen == 0xffffffffu) {  // uniform: 32 keys that lie together
          const global_bytes src = rows + (uint32_t)__builtin_amdgcn_readfirstlane(slot) * row_stride;
          const uint32_t off = (uint32_t)(lane / kChunks) * (uint32_t)row_stride + part * row_bytes + byte;
#pragma unroll
          for (int i = 0; i < kLoads; ++i)
            w[i] = load16_once(inside ? src + (uint64_t)(i * kApart) * row_stride + off : zero + byte);
        } else {
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const int at_slot = __shfl(slot, kApart * i + lane / kChunks);
            w[i] = load16_once(inside && at_slot >= 0 ? rows + (uint32_t)at_slot * row_stride + part * row_bytes + byte : zero + byte);
          }
        }
      }
      find(x, unit + kSets * p.ways);
    };
    const auto store = [&] {  // bf16: the loaded unit's K and V
      const int c = lane % kChunks, part = c >= kChunks / 2;
      uint8_t* const dst = own_lds + (part ? kV + lane / kChunks * kVRow + 16 * (c - kChunks / 2) : lane / kChunks * kKRow + 16 * c);
      const int step = kApart * (part ? kVRow : kKRow);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) *(u32x4*)(dst + i * step) = set[0].w[i];
    };
    f32x4 o[DP / 16];
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kLowest, l = 0.f;
    uint32_t here = 0;
    // One unit's keys, of fp8 those in set x; its loads' successors leave in between.
    const auto take = [&](int x, int unit) {
      f32x4 sc[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        sc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          u32x4 a;
          if (FP8) a = bf16_of_codes(set[x].w[2 * kCodes * b + i / 2][2 * (i % 2)], set[x].w[2 * kCodes * b + i / 2][2 * (i % 2) + 1]);
          else a = *(const u32x4*)(own_lds + (16 * b + n) * kKRow + 64 * i + 16 * j);
          sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), q[i], sc[b], 0, 0, 0);
        }
      }
      // Scores leave after the loads of the next unit, by buffer stores, which drop what lies past their end (heads that are
      // none, or all of it): no branch, so the compiler knows that they follow the loads and waits for those alone.
      const auto keep_scores = [&] {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const bool write = keep && unit * 32 + 16 * b < end_key;  // uniform
          const auto to = __builtin_amdgcn_make_buffer_rsrc(scores + (size_t)(2 * unit + b) * p.Hkv * p.G * 16, 0,
                                                            write ? p.G * 64 : 0, 0x00027000);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sc[b]), to, (tile * 16 + n) * 64 + 16 * j, 0, 0);
        }
      };
      float vk[2][4];
      if (FP8) {
        here = set[x].seen;
        wave_fence();  // the last unit's V has been read
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < kCodes; ++i) {
            uint8_t* dst = own_lds + (16 * b + n) * kVRow + 128 * i + 32 * j;
            const u32x4 y = set[x].w[2 * kCodes * b + kCodes + i];
            *(u32x4*)dst = bf16_of_codes(y[0], y[1]);
            *(u32x4*)(dst + 16) = bf16_of_codes(y[2], y[3]);
          }
        wave_fence();
        const float ks = set[x].ks, vs = set[x].vs;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sc[b][r] = scaled(sc[b][r], p.scale * __shfl(ks, 16 * b + 4 * j + r));
            vk[b][r] = __shfl(vs, 16 * b + 4 * j + r);
          }
        if (unit + kSets * p.ways < end_unit) load(x, unit + kSets * p.ways);
      } else {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[b][r] = scaled(sc[b][r], p.scale);
      }
      if (p.cap != 0.f) cap_scores(sc, p.cap);
      if (here != 0xffffffffu) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[b][r] = here >> (16 * b + 4 * j + r) & 1 ? sc[b][r] : -__builtin_inff();
      }
      float top = max_of(max_of(max_of(sc[0][0], sc[0][1]), max_of(sc[0][2], sc[0][3])),
                         max_of(max_of(sc[1][0], sc[1][1]), max_of(sc[1][2], sc[1][3])));
      if (__ballot(top > m + kRescale)) {
        top = swap_max(top);
        const float next = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - next);
        m = next;
        l *= f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[d] *= f;
      }
      u32x4 parts[3];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = __builtin_amdgcn_exp2f(sc[b][r] - m);
          l += e[r];
          if (FP8) e[r] *= vk[b][r];
        }
        const Parts lo = split_bf16(e[0], e[1]), hi = split_bf16(e[2], e[3]);
#pragma unroll
        for (int i = 0; i < 3; ++i) parts[i][2 * b] = lo.of[i], parts[i][2 * b + 1] = hi.of[i];
      }
      if (FP8) keep_scores();
      typedef __attribute__((address_space(3))) i16x4* lds_i16x4;
      const uint8_t* vt = own_lds + kV + (4 * j + n / 4) * kVRow + 8 * (n % 4);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(vt + 32 * d));
        const i16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(vt + 16 * kVRow + 32 * d));
        const bf16x8 f = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int i = 0; i < 3; ++i)
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, parts[i]), o[d], 0, 0, 0);
      }
      if (!FP8) {
        if (unit + p.ways < end_unit) {
          wave_fence();
          here = set[0].seen;
          store();
          if (unit + 2 * p.ways < end_unit) load(0, unit + 2 * p.ways);
        }
        keep_scores();
      }
    };
    const int first_unit = first_block << (p.block_shift - 5);
    int unit = first_unit + way;
#pragma unroll
    for (int x = 0; x < kSets; ++x) find(x, unit + x * p.ways);
    // Waited for on every path into the loop, and the queries, loaded before, with them: on one where the compiler saw the
    // queries still under way, every turn would wait for all that is.
#pragma unroll
    for (int x = 0; x < kSets; ++x) asm volatile("" : "+v"(set[x].id));
#pragma unroll
    for (int x = 0; x < kSets; ++x)
      if (unit + x * p.ways < end_unit) load(x, unit + x * p.ways);
    if (!FP8 && unit < end_unit) {
      wave_fence();
      here = set[0].seen;
      store();
      if (unit + p.ways < end_unit) load(0, unit + p.ways);
    }
    if (!FP8) {
      const auto none = __builtin_amdgcn_make_buffer_rsrc(scores, 0, 0, 0x00027000);
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{0, 0, 0, 0}, none, 0, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{0, 0, 0, 0}, none, 16, 0, 0);
    }
    for (; unit < end_unit; unit += kSets * p.ways)
#pragma unroll
      for (int x = 0; x < kSets; ++x)
        if (unit + x * p.ways < end_unit) take(x, unit + x * p.ways);

    const bool own = first_block == 0 && end_block == blocks;
    if (at == share.from && tid == 0) {
      const RowParts r = row_parts(p, share.row_total, at - first_block, blocks);
      p.joins[blockIdx.x] = {first_block && end_block == blocks ? r.first : -1, r.late, t, h - mine, tile, 0};
    }
    const int live = min(p.G - tile * 16, 16);
    float* const part = p.parts + ((2 * (size_t)blockIdx.x + (at > share.from)) * p.near) * (32 + 16 * (size_t)p.D);
    l = swap_sum(l);
    if (p.ways == 1) {  // the wave has all of the row
      if (n < live) {
        float* const to = part + mine * (32 + 16 * (size_t)p.D);
        const size_t to_row = (size_t)t * p.Hkv * p.G + h * p.G + tile * 16 + n;
        const float g = l == 0.f ? 0.f : p.v_scale / l;
        if (j == 0 && own) p.stats[to_row] = {m, l == 0.f ? 0.f : 1.f / l};
        if (j == 0 && !own) to[2 * n] = m, to[2 * n + 1] = l;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          const int dim = 16 * d + 4 * j;
          if (!FULL && dim >= p.D) break;
          if (own)
            *(u32x2*)(p.out + to_row * p.D + dim) =
                l == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(o[d][0] * g, o[d][1] * g), pack_bf16(o[d][2] * g, o[d][3] * g)};
          else
            *(f32x4*)(to + 32 + n * p.D + dim) = o[d];
        }
      }
    } else {
      if (j == 0) s_m[wave][n] = m, s_l[wave][n] = l;
      __syncthreads();  // every wave is done with its V, too
      float all = kLowest;
      for (int x = 0; x < p.ways; ++x) all = fmaxf(all, s_m[x * p.near + mine][n]);
      const float f = __builtin_amdgcn_exp2f(m - all);
      float* const rows_o = (float*)own_lds + n * kORow;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) *(f32x4*)(rows_o + 16 * d + 4 * j) = o[d] * f;
      __syncthreads();
      const int quads = p.D / 4;
      for (int i = tid; i < p.near * live * quads; i += threads) {
        const int head = i / (live * quads), r = (i - head * live * quads) / quads, d = i % quads * 4;
        float top = kLowest, sum = 0.f;
        for (int x = 0; x < p.ways; ++x) top = fmaxf(top, s_m[x * p.near + head][r]);
        f32x4 x4 = {0.f, 0.f, 0.f, 0.f};
        for (int x = 0; x < p.ways; ++x) {
          const int from = x * p.near + head;
          sum += s_l[from][r] * __builtin_amdgcn_exp2f(s_m[from][r] - top);
          x4 += *(const f32x4*)((const float*)(lds + from * kWave) + r * kORow + d);
        }
        if (!own) {
          float* const to = part + head * (32 + 16 * (size_t)p.D);
          if (d == 0) to[2 * r] = top, to[2 * r + 1] = sum;
          *(f32x4*)(to + 32 + r * p.D + d) = x4;
          continue;
        }
        const size_t to_row = (size_t)t * p.Hkv * p.G + (h - mine + head) * p.G + tile * 16 + r;
        const float g = sum == 0.f ? 0.f : p.v_scale / sum;
        if (d == 0) p.stats[to_row] = {top, sum == 0.f ? 0.f : 1.f / sum};
        *(u32x2*)(p.out + to_row * p.D + d) =
            sum == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(x4[0] * g, x4[1] * g), pack_bf16(x4[2] * g, x4[3] * g)};
      }
      __syncthreads();  // the next row's LDS
    }
    at += end_block - first_block;
  }
}

// Joins a row's parts, a workgroup a kv head.  Four dims of a head are a thread's, or, of many parts, 8 threads', a share
// of the parts each.
__device__ __forceinline__ void join_rows(const WeighParams& p, int block) {
  constexpr int kParts = 4;
  const int head = block % p.near;
  const JoinOf join = p.joins[block / p.near];
  if (join.first < 0) return;  // uniform
  const RowParts parts = {join.first, block / p.near, join.late != 0};
  const int h = join.h + head, tile = join.tile, t = join.t;
  const int live = min(p.G - tile * 16, 16), quads = p.D / 4, lanes = parts.last - parts.first > 8 ? 8 : 1;
  for (int i0 = 0; i0 < live * quads; i0 += kWeighThreads / lanes) {
    const int i = min(i0 + (int)threadIdx.x / lanes, live * quads - 1), lane = threadIdx.x % lanes;
    const int r = i / quads, d = i % quads * 4;
    float top = kLowest, sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int w = parts.first + lane; w <= parts.last; w += kParts * lanes) {
      float m[kParts], l[kParts];
      f32x4 o[kParts];
#pragma unroll
      for (int u = 0; u < kParts; ++u) {
        const float* part = row_part(p, parts, min(w + u * lanes, parts.last), head);
        m[u] = part[2 * r], l[u] = w + u * lanes <= parts.last ? part[2 * r + 1] : 0.f;
        o[u] = *(const f32x4*)(part + 32 + r * p.D + d);
      }
#pragma unroll
      for (int u = 0; u < kParts; ++u) {
        if (l[u] == 0.f) continue;  // no keys
        const float next = fmaxf(top, m[u]), mine = __builtin_amdgcn_exp2f(top - next), its = __builtin_amdgcn_exp2f(m[u] - next);
        top = next;
        sum = sum * mine + l[u] * its;
        x = x * mine + o[u] * its;
      }
    }
    for (int e = 1; e < lanes; e *= 2) {
      const float m = __shfl_xor(top, e), l = __shfl_xor(sum, e);
      f32x4 o;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = __shfl_xor(x[u], e);
      const float next = fmaxf(top, m), mine = __builtin_amdgcn_exp2f(top - next), its = __builtin_amdgcn_exp2f(m - next);
      top = next;
      // a side without keys has no O
      sum = sum * mine + l * its;
      x = (sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : x * mine + o * its);
    }
    if (lane || i0 + (int)threadIdx.x / lanes >= live * quads) continue;
    const size_t to = (size_t)t * p.Hkv * p.G + h * p.G + tile * 16 + r;
    const float g = sum == 0.f ? 0.f : p.v_scale / sum;
    *(u32x2*)(p.out + to * p.D + d) =
        sum == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(x[0] * g, x[1] * g), pack_bf16(x[2] * g, x[3] * g)};
  }
}

// Adds x to the weight of a key of the sequence, whose first new key is `old`.
__device__ __forceinline__ void add_weight(const WeighParams& p, int seq, int h, int old, int key, float x) {
  const int page = div_by(key, p.page), id = p.table[(size_t)seq * p.PPS + page];
  if (id < 0 || id >= p.P) return;
  const size_t to = ((size_t)id * p.Hkv + h) * p.S + (key - page * p.S);
  if (key >= old) p.positions[to] = (p.dropped ? p.dropped[seq] : 0) + key;
  else if (p.decay != 0.f) x += p.decay * p.weights[to];
  p.weights[to] = x;
}

// Where the sums of a kv head's rows begin, in `of`: (m, 1 / l) of row (token, g) of a sequence that rows did, from its
// parts, by `lanes` neighbouring lanes (a power of two), each a share of them.
__device__ __forceinline__ float2 row_stat(const WeighParams& p, const Share& share, const Sequence& s, long long rows_before, int token,
                                           int h, int g, int lane, int lanes) {
  const int blocks = row_blocks(p, s);
  const long long begin = rows_before + (((long long)token * (p.Hkv / p.near) + h / p.near) * p.tiles + g / 16) * blocks;
  const RowParts parts = row_parts(p, share.row_total, begin, blocks);
  if (parts.first == parts.last) return p.stats[(size_t)(s.first + token) * p.Hkv * p.G + h * p.G + g];
  float top = kLowest, sum = 0.f;
#pragma unroll 4
  for (int w = parts.first + lane; w <= parts.last; w += lanes) {
    const float* part = row_part(p, parts, w, h % p.near) + 2 * (g % 16);
    const float m = part[0], l = part[1];
    const float next = l == 0.f ? top : fmaxf(top, m);
    sum = sum * __builtin_amdgcn_exp2f(top - next) + (l == 0.f ? 0.f : l * __builtin_amdgcn_exp2f(m - next));
    top = next;
  }
  for (int d = 1; d < lanes; d *= 2) {
    const float m = __shfl_xor(top, d), l = __shfl_xor(sum, d), next = fmaxf(top, m);
    sum = sum * __builtin_amdgcn_exp2f(top - next) + l * __builtin_amdgcn_exp2f(m - next);
    top = next;
  }
  return {top, sum == 0.f ? 0.f : 1.f / sum};
}

// The weights of the sequences that rows did.  Of a sequence with one token the scores are there: a workgroup takes
// kScoreKeys keys of as many kv heads as make 256 rows, a wave a head at a time, a lane four keys, summed over the group's
// heads.  Of one with more (a batch with few tokens that has such a sequence), or whose scores did not fit, K is multiplied
// once more, 32 keys a wave with 16 rows (token, head) at a time.
constexpr int kScoreKeys = 256, kRowKeys = 32 * kWeighWaves;

template <int DP, bool FULL, bool FP8>
__device__ __forceinline__ void weigh_rows(const WeighParams& p, int block, int blocks) {
  constexpr int kElem = FP8 ? 1 : 2;
  constexpr int kLoads = DP * kElem / 64;
  constexpr int kSteps = DP / 32;
  __shared__ float2 s_stat[256];
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 16, j = lane / 16;
  const int heads = min(p.Hkv, 256 / p.G), chunks = (p.Hkv + heads - 1) / heads;  // G is at most 256
  const auto items = [&](const Sequence& s, bool pad) {
    if (pad || !s.tokens || in_tiles(p, s, pad)) return 0ll;
    return s.tokens == 1 ? (long long)((s.keys + kScoreKeys - 1) / kScoreKeys) * chunks
                         : (long long)((s.keys + kRowKeys - 1) / kRowKeys) * p.Hkv;
  };
  const Share share = share_of<true>(p, block, blocks, items, true);
  if (share.from == share.to) return;
  int seq = share.seq, stat_of = -1;  // stat_of: the sequence and head that s_stat begins with
  Sequence s = share.s;
  long long before = share.before, score_at = share.scores, rows_at = share.rows;
  for (long long at = share.from; at < share.to; ++at) {
    for (long long units; at >= before + (units = items(s, false));) {
      before += units;
      score_at += score_blocks(s), rows_at += row_units(p, s, false);
      s = work_sequence(p, share.count, ++seq);
      stat_of = -1;
    }
    const bool one = s.tokens == 1;
    const int keys_of = one ? kScoreKeys : kRowKeys, of_head = (s.keys + keys_of - 1) / keys_of;
    const int head_chunk = (int)((at - before) / of_head), part = (int)((at - before) - (long long)head_chunk * of_head);
    const int h0 = one ? head_chunk * heads : head_chunk, h1 = one ? min(h0 + heads, p.Hkv) : h0 + 1;
    const int old = s.keys - s.tokens;  // keys before the step's
    if (scores_fit(p, s, score_at)) {
      const int key0 = part * kScoreKeys + 4 * lane;  // this lane's four keys
      const bool four = p.quads && key0 + 4 <= old;   // in one page, none of them new
      const int page = div_by(key0, p.page), id = four ? p.table[(size_t)seq * p.PPS + page] : -1;
      if (stat_of != h0) {
        __syncthreads();  // the last use of s_stat
        const int of = (h1 - h0) * p.G, width = of <= 32 ? 8 : of <= 64 ? 4 : of <= 128 ? 2 : 1;
        if (tid < of * width) {  // lanes of a row stay together
          const int r = tid / width;
          const float2 st = row_stat(p, share, s, rows_at, 0, h0 + r / p.G, r % p.G, tid % width, width);
          if (tid % width == 0) s_stat[r] = st;
        }
        __syncthreads();
        stat_of = h0;
      }
      if (key0 < s.keys) {
        const bool whole = four && id >= 0 && id < p.P;
        for (int h = h0 + wave; h < h1; h += kWeighWaves) {
          const float* const from = p.scores + (((size_t)score_at + key0 / 16) * p.Hkv + h) * p.G * 16 + key0 % 16;
          const float2* const stat = s_stat + (h - h0) * p.G;
          float* const to = p.weights + ((size_t)(whole ? id : 0) * p.Hkv + h) * p.S + (key0 - page * p.S);
          f32x4 was = {0.f, 0.f, 0.f, 0.f};
          if (whole && p.decay != 0.f) was = *(const f32x4*)to;
          f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
          for (int g = 0; g < p.G; ++g) {
            const f32x4 x = *(const f32x4*)(from + g * 16);
            const float2 st = stat[g];
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[r] += __builtin_amdgcn_exp2f(x[r] - st.x) * st.y;
          }
          if (whole) {
            if (p.decay != 0.f) sum += p.decay * was;
            *(f32x4*)to = sum;
          } else if (!four) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (key0 + r < s.keys) add_weight(p, seq, h, old, key0 + r, sum[r]);
          }
        }
      }
      continue;
    }
    for (int h = h0; h < h1; ++h) {  // no barrier in here
      const int32_t* const table = p.table + (size_t)seq * p.PPS;
      const int row_bytes = p.D * kElem;
      const uint64_t row_stride = 2ull * p.Hkv * row_bytes;
      const global_bytes zero = zero_row(), rows = (global_bytes)(uint64_t)p.kv + 2 * (size_t)h * row_bytes;
      const int first = part * keys_of, last = min(first + keys_of, s.keys);
      for (int key0 = first + 32 * wave; key0 < last; key0 += kRowKeys) {
        bf16x8 k[2][kSteps];
        float ks[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int key = key0 + 16 * b + n, page = div_by(min(key, last - 1), p.page), id = table[page];
          const bool ok = key < last && id >= 0 && id < p.P;
          const global_bytes src = ok ? rows + (uint32_t)(id * p.S + (key - page * p.S)) * row_stride : zero;
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const int byte = 64 * i + 16 * j;
            const u32x4 w = load16((FULL || byte < row_bytes ? src : zero) + byte);
            if (FP8) {
              k[b][2 * i] = __builtin_bit_cast(bf16x8, bf16_of_codes(w[0], w[1]));
              k[b][2 * i + 1] = __builtin_bit_cast(bf16x8, bf16_of_codes(w[2], w[3]));
            } else {
              k[b][i] = __builtin_bit_cast(bf16x8, w);
            }
          }
          ks[b] = FP8 && p.scales && ok ? p.scales[((size_t)id * p.Hkv + h) * 2] : 1.f;
        }
        float scale[2][4], sum[2][4] = {};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) scale[b][r] = FP8 ? p.scale * __shfl(ks[b], 4 * j + r) : p.scale;
        const int end = s.tokens * p.G;
        for (int base = max(key0 - old, 0) * p.G; base < end; base += 16) {
          const int row = min(base + n, end - 1), token = div_by(row, p.group), g = row - token * p.G, t = s.first + token;
          const bool live = base + n < end;
          const uint16_t* src = p.q + t * p.q_token + ((long long)h * p.G + g) * p.q_head;
          f32x4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const int dim = FP8 ? 64 * (i / 2) + 16 * j + 8 * (i % 2) : 32 * i + 8 * j;
            u32x4 w = {0, 0, 0, 0};
            if (live && (FULL || dim < p.D)) w = *(const u32x4*)(src + dim);
#pragma unroll
            for (int b = 0; b < 2; ++b)
              sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[b][i], __builtin_bit_cast(bf16x8, w), sc[b], 0, 0, 0);
          }
          const float2 stat = row_stat(p, share, s, rows_at, token, h, g, 0, 1);
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[b][r] = scaled(sc[b][r], scale[b][r]);
          if (p.cap != 0.f) cap_scores(sc, p.cap);
          const int seen = live ? old + token : -1;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float e = __builtin_amdgcn_exp2f(sc[b][r] - stat.x) * stat.y;
              sum[b][r] += key0 + 16 * b + 4 * j + r <= seen ? e : 0.f;
            }
        }
        float mine = 0.f;  // lane n < 8: of key 16 (n / 4) + 4 j + n % 4
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          float x = sum[u / 4][u % 4];
#pragma unroll
          for (int d = 1; d < 16; d *= 2) x += __shfl_xor(x, d);
          mine = n == u ? x : mine;
        }
        const int key = key0 + 16 * (n / 4) + 4 * j + n % 4;
        if (n < 8 && key < last) add_weight(p, seq, h, old, key, mine);
      }
    }
  }
}

}  // namespace
}  // namespace rpa_sparse
