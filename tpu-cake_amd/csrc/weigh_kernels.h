// Attention over a paged cache that accounts for the weight each key got.
//
// Mathematics: o_t = sum_x p_tx v_x, p_tx = 2^(s_tx - m_t) / l_t over the keys x up to token t's position (log2 domain),
// and for each key the sum of p_tx over the step's tokens and the group's heads.  The row's maximum m and sum l are
// known only once every key has been seen, so weights take the scores a second time.
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

constexpr int kWeighWaves = 4, kWeighThreads = 64 * kWeighWaves;
constexpr int kBlockKeys = 256;  // keys of a block of rows' work: two units of 32 for each wave

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
  float* parts;   // two for each workgroup: (m, l) of 16 rows, then the rows' O
  long long q_token, q_head;
  int T, Hkv, G, D, P, S, N, PPS;
  int tiles;      // 16-head tiles of a group
  int chunk;      // sequences of more than one token are done in tiles
  float* tile_parts;  // of tiles: two for each workgroup, (m, l) of kColumns columns, then their O
  Divisor page, group;
  float scale, cap, v_scale, decay;  // scale: of q.k; times log2 e where cap is 0
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

// Where a workgroup's share of all the work begins: sequences in order, `amount(i)` units of work each, the total in
// shares of equal size.
struct Share {
  int index;           // of the shares in order
  long long from, to;  // units
  int seq;             // that `from` lies in
  long long before;    // units of the sequences before it
  long long scores;    // and their blocks of scores
};

// NEAR: XCDs take workgroups in turn; neighbouring shares, which read the same keys, go to one of them.
template <bool NEAR, typename Amount, typename Scores>
__device__ __forceinline__ Share share_of(int n, Amount amount, Scores scores) {
  const int count = gridDim.x;
  __shared__ long long s_sum[kWeighWaves], s_scores[kWeighWaves];
  __shared__ Share s_share;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int each = (n + kWeighThreads - 1) / kWeighThreads, i0 = min(tid * each, n), i1 = min(i0 + each, n);
  long long own = 0, mine = 0;
  for (int i = i0; i < i1; ++i) own += amount(i), mine += scores(i);
  long long upto = own, stored = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const long long o = __shfl_up(upto, d), u = __shfl_up(stored, d);
    upto += lane >= d ? o : 0, stored += lane >= d ? u : 0;
  }
  if (lane == 63) s_sum[wave] = upto, s_scores[wave] = stored;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWeighWaves; ++w) {
    upto += w < wave ? s_sum[w] : 0, stored += w < wave ? s_scores[w] : 0;
    total += s_sum[w];
  }
  const long long each_share = (total + count - 1) / count;
  int index = blockIdx.x;
  if (NEAR && total) {
    const int used = (int)((total + each_share - 1) / each_share), xcd = index % 8;
    index = index < used ? xcd * (used / 8) + min(xcd, used % 8) + index / 8 : count;
  }
  const long long from = min(index * each_share, total);
  const long long to = min(from + each_share, total);
  long long before = upto - own;
  stored -= mine;
  if (from < to && from >= before && from < upto) {
    int i = i0;
    for (;; ++i) {
      const long long a = amount(i);
      if (from < before + a) break;
      before += a, stored += scores(i);
    }
    s_share = {index, from, to, i, before, stored};
  }
  __syncthreads();
  return from < to ? s_share : Share{0, 0, 0, 0, 0, 0};
}
template <bool NEAR, typename Amount>
__device__ __forceinline__ Share share_of(int n, Amount amount) {
  return share_of<NEAR>(n, amount, [](int) { return 0ll; });
}

// Scores of a sequence with one token, which its weights take instead of K once more: blocks of 16 keys, of which
// [kv head][head of the group][key].  They are kept while they fit the workspace, which holds all that distinct pages can
// have.
__device__ __forceinline__ long long score_blocks(const Sequence& s) { return s.tokens == 1 ? (s.keys + 15) / 16 : 0; }
__device__ __forceinline__ bool scores_fit(const WeighParams& p, const Sequence& s, long long before) {
  return s.tokens == 1 && before + score_blocks(s) <= p.score_room;
}

// The blocks of keys of one row of sequence i; sequence n stands for the tokens past the last one.
__device__ __forceinline__ int row_blocks(const Sequence& s) { return max((s.keys + kBlockKeys - 1) / kBlockKeys, 1); }

__device__ __forceinline__ Sequence row_sequence(const WeighParams& p, int n, int i) {
  if (i < n) {
    Sequence s = sequence_at(p, i);
    if (p.chunk && s.tokens > 1) s.tokens = 0;
    return s;
  }
  const int end = n ? min(max(p.cu[n], 0), p.T) : 0;
  return {end, p.T - end, 0};
}

// Rows: a token's heads, up to 16 of one kv head.  Their keys come in blocks, blocks of all rows in shares, one a
// workgroup: a long sequence's rows are spread over as many workgroups as their blocks need, and short ones' share a workgroup.
// A row that a workgroup does not have whole leaves a part: the first in the workgroup's slot 0, the last in slot 1.
template <int DP, bool FULL, bool FP8>
__global__ __launch_bounds__(kWeighThreads) void weigh_rows_kernel(WeighParams p) {
  constexpr int kRow = DP * 2 + 32;
  constexpr int kWave = 32 * kRow;
  constexpr int kORow = DP + 4;
  constexpr int kElem = FP8 ? 1 : 2;
  constexpr int kLoads = DP * kElem / 64;
  constexpr int kSteps = DP / 32;
  static_assert(16 * kORow * 4 <= kWave, "O rows fit the wave's V region");
  __shared__ __align__(16) uint8_t s_v[kWeighWaves * kWave];
  __shared__ float s_m[kWeighWaves][16], s_l[kWeighWaves][16];
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 16, j = lane / 16;
  const int count = min(max(*p.num_seqs, 0), p.N);
  const int heads = p.Hkv * p.tiles;
  const Share share = share_of<false>(
      count + 1,
      [&](int i) {
        const Sequence s = row_sequence(p, count, i);
        return (long long)s.tokens * heads * row_blocks(s);
      },
      [&](int i) { return i < count ? score_blocks(sequence_at(p, i)) : 0ll; });
  if (share.from == share.to) return;

  const int row_bytes = p.D * kElem;
  const uint64_t row_stride = 2ull * p.Hkv * row_bytes;
  const global_bytes zero = zero_row();
  uint8_t* const tile_v = s_v + wave * kWave;
  int seq = share.seq;
  Sequence s = row_sequence(p, count, seq);
  long long before = share.before, at = share.from, score_at = share.scores;
  while (at < share.to) {
    int blocks = row_blocks(s);
    while (at >= before + (long long)s.tokens * heads * blocks) {
      before += (long long)s.tokens * heads * blocks;
      score_at += seq < count ? score_blocks(s) : 0;
      s = row_sequence(p, count, ++seq);
      blocks = row_blocks(s);
    }
    const long long row = (at - before) / blocks;
    const int first_block = (int)(at - before - row * blocks);
    const int end_block = (int)min((long long)blocks, first_block + (share.to - at));
    const int token = (int)(row / heads), head_tile = (int)(row - (long long)token * heads), h = head_tile / p.tiles;
    const int tile = head_tile - h * p.tiles, t = s.first + token;
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
    const int end_key = min(keys, end_block * kBlockKeys), end_unit = (end_key + 31) / 32;
    const bool keep = known && scores_fit(p, s, score_at);
    float* const scores = p.scores + ((size_t)score_at * p.Hkv + h) * p.G * 16 + (tile * 16 + n) * 16 + 4 * j;
    int ids[2];  // the pages of key n and n + 16 of a unit: found a turn before its keys are loaded
    u32x4 k[2][kLoads], v[2][kLoads];
    uint32_t seen[2];
    float ks[2], vs[2];  // fp8: the scales of key n of the 16
    const auto find = [&](int unit) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int key = unit * 32 + 16 * b + n;
        ids[b] = key < end_key ? table[div_by(key, p.page)] : -1;
      }
    };
    const auto load = [&](int unit) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int key = unit * 32 + 16 * b + n, id = ids[b];
        const bool ok = key < end_key && id >= 0 && id < p.P;
        if (key < end_key && !ok) flag_error(RPA_SPARSE_ERR_PAGE);
        seen[b] = (uint32_t)__ballot(ok) & 0xffffu;
        const int slot = ok ? id * p.S + (key - div_by(key, p.page) * p.S) : 0;
        const global_bytes src = ok ? rows + (uint32_t)slot * row_stride : zero;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int byte = 64 * i + 16 * j;
          const global_bytes from = FULL || byte < row_bytes ? src : zero;
          k[b][i] = load16(from + byte);
          v[b][i] = load16(from + row_bytes + byte);
        }
        if (FP8) {
          const float* scale = p.scales && ok ? p.scales + ((size_t)id * p.Hkv + h) * 2 : nullptr;
          ks[b] = scale ? scale[0] : 1.f, vs[b] = scale ? scale[1] : 1.f;
        }
      }
      if (unit + kWeighWaves < end_unit) find(unit + kWeighWaves);
    };
    f32x4 o[DP / 16];
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kLowest, l = 0.f;
    int unit = first_block * (kBlockKeys / 32) + wave;
    if (unit < end_unit) find(unit), load(unit);
    for (; unit < end_unit; unit += kWeighWaves) {
      f32x4 sc[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        sc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const u32x4 a = FP8 ? bf16_of_codes(k[b][i / 2][2 * (i % 2)], k[b][i / 2][2 * (i % 2) + 1]) : k[b][FP8 ? 0 : i];
          sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), q[i], sc[b], 0, 0, 0);
        }
      }
      wave_fence();  // the last unit's V has been read
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          uint8_t* dst = tile_v + (16 * b + n) * kRow + (FP8 ? 128 * i + 32 * j : 64 * i + 16 * j);
          if (FP8) {
            *(u32x4*)dst = bf16_of_codes(v[b][i][0], v[b][i][1]);
            *(u32x4*)(dst + 16) = bf16_of_codes(v[b][i][2], v[b][i][3]);
          } else {
            *(u32x4*)dst = v[b][i];
          }
        }
      wave_fence();
      const bool whole = (seen[0] & seen[1]) == 0xffffu;
      const uint32_t here[2] = {seen[0] >> (4 * j), seen[1] >> (4 * j)};
      float vk[2][4];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sc[b][r] = scaled(sc[b][r], FP8 ? p.scale * __shfl(ks[b], 4 * j + r) : p.scale);
          vk[b][r] = FP8 ? __shfl(vs[b], 4 * j + r) : 1.f;
        }
      if (unit + kWeighWaves < end_unit) load(unit + kWeighWaves);
      if (p.cap != 0.f) cap_scores(sc, p.cap);
      if (!whole) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[b][r] = here[b] >> r & 1 ? sc[b][r] : -__builtin_inff();
      }
      if (keep) {  // uniform
#pragma unroll
        for (int b = 0; b < 2; ++b)
          if (tile * 16 + n < p.G && unit * 32 + 16 * b < end_key)
            *(f32x4*)(scores + (size_t)(2 * unit + b) * p.Hkv * p.G * 16) = sc[b];
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
      typedef __attribute__((address_space(3))) i16x4* lds_i16x4;
      const uint8_t* vt = tile_v + (4 * j + n / 4) * kRow + 8 * (n % 4);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(vt + 32 * d));
        const i16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(vt + 16 * kRow + 32 * d));
        const bf16x8 f = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int i = 0; i < 3; ++i)
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, parts[i]), o[d], 0, 0, 0);
      }
    }

    // join the waves
    l = swap_sum(l);
    if (j == 0) s_m[wave][n] = m, s_l[wave][n] = l;
    __syncthreads();  // every wave is done with its V, too
    float all = s_m[0][n];
#pragma unroll
    for (int w = 1; w < kWeighWaves; ++w) all = fmaxf(all, s_m[w][n]);
    const float f = __builtin_amdgcn_exp2f(m - all);
    float* const mine = (float*)tile_v + n * kORow;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) *(f32x4*)(mine + 16 * d + 4 * j) = o[d] * f;
    __syncthreads();
    const bool own = first_block == 0 && end_block == blocks;
    const int live = min(p.G - tile * 16, 16), quads = p.D / 4;
    float* const part = p.parts + (2 * (size_t)blockIdx.x + (at > share.from)) * (32 + 16 * (size_t)p.D);
    for (int i = tid; i < live * quads; i += kWeighThreads) {
      const int r = i / quads, d = i % quads * 4;
      float top = s_m[0][r], sum = 0.f;
#pragma unroll
      for (int w = 1; w < kWeighWaves; ++w) top = fmaxf(top, s_m[w][r]);
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWeighWaves; ++w) {
        sum += s_l[w][r] * __builtin_amdgcn_exp2f(s_m[w][r] - top);
        x += *(const f32x4*)((const float*)(s_v + w * kWave) + r * kORow + d);
      }
      if (!own) {
        if (d == 0) part[2 * r] = top, part[2 * r + 1] = sum;
        *(f32x4*)(part + 32 + r * p.D + d) = x;
        continue;
      }
      const size_t to = (size_t)t * p.Hkv * p.G + h * p.G + tile * 16 + r;
      const float g = sum == 0.f ? 0.f : p.v_scale / sum;
      if (d == 0) p.stats[to] = {top, sum == 0.f ? 0.f : 1.f / sum};
      *(u32x2*)(p.out + to * p.D + d) =
          sum == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(x[0] * g, x[1] * g), pack_bf16(x[2] * g, x[3] * g)};
    }
    __syncthreads();  // the next row's V
    at += end_block - first_block;
  }
}

// Joins the parts of rows that several workgroups had: one workgroup for each share, which takes the row that ends in
// it and began before it.
__global__ __launch_bounds__(kWeighThreads) void weigh_join_kernel(WeighParams p) {
  const int count = min(max(*p.num_seqs, 0), p.N), heads = p.Hkv * p.tiles;
  const Share share = share_of<false>(count + 1, [&](int i) {
    const Sequence s = row_sequence(p, count, i);
    return (long long)s.tokens * heads * row_blocks(s);
  });
  if (share.from == share.to) return;
  const Sequence s = row_sequence(p, count, share.seq);
  const int blocks = row_blocks(s);
  const long long row = (share.from - share.before) / blocks, begin = share.before + row * blocks, end = begin + blocks;
  if (begin == share.from || end > share.to) return;  // uniform
  const long long each = share.from / blockIdx.x;  // every share before the last has as many; block 0 begins a row
  const int first = (int)(begin / each), last = blockIdx.x;
  const int token = (int)(row / heads), head_tile = (int)(row - (long long)token * heads), h = head_tile / p.tiles;
  const int tile = head_tile - h * p.tiles, t = s.first + token;
  const int live = min(p.G - tile * 16, 16), quads = p.D / 4;
  const size_t stride = 32 + 16 * (size_t)p.D;
  for (int i = threadIdx.x; i < live * quads; i += kWeighThreads) {
    const int r = i / quads, d = i % quads * 4;
    float top = kLowest, sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int w = first; w <= last; ++w) {
      const float* part = p.parts + (2 * (size_t)w + (w == first && begin % each != 0)) * stride;
      const float m = part[2 * r], l = part[2 * r + 1];
      if (l == 0.f) continue;
      const f32x4 o = *(const f32x4*)(part + 32 + r * p.D + d);
      const float next = fmaxf(top, m), mine = __builtin_amdgcn_exp2f(top - next), its = __builtin_amdgcn_exp2f(m - next);
      top = next;
      sum = sum * mine + l * its;
      x = x * mine + o * its;
    }
    const size_t to = (size_t)t * p.Hkv * p.G + h * p.G + tile * 16 + r;
    const float g = sum == 0.f ? 0.f : p.v_scale / sum;
    if (d == 0) p.stats[to] = {top, sum == 0.f ? 0.f : 1.f / sum};
    *(u32x2*)(p.out + to * p.D + d) =
        sum == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(x[0] * g, x[1] * g), pack_bf16(x[2] * g, x[3] * g)};
  }
}

// Prompt chunks: tiles of kColumns columns, the (token, head) rows of one sequence and kv head in order, 32 a wave, on
// v_mfma_f32_32x32x16_bf16: S = K Q^T (32 keys x 32 columns), O^T += V^T P^T.  A tile's keys pass through LDS once for
// its four waves, two buffers in turn.  A lane's scores are the keys its P operand needs, as in rows.  Tiles' keys come in
// slots of about kBlockKeys, slots in shares, as blocks of rows do.
constexpr int kColumns = 128;

// Slots of a (sequence, head)'s first j tiles, by the keys that the tiles see: old + kColumns (j' + 1) / G each.
__device__ __forceinline__ long long slots_before(const WeighParams& p, int old, long long j) {
  return j + (2 * j * old * p.G + kColumns * j * (j + 1)) / (2 * kBlockKeys * p.G);
}
__device__ __forceinline__ long long tiles_of(const WeighParams& p, const Sequence& s) {
  return ((long long)s.tokens * p.G + kColumns - 1) / kColumns;
}
// Of one kv head; 0 for sequences that rows do.
__device__ __forceinline__ long long tile_slots(const WeighParams& p, const Sequence& s) {
  return s.tokens > 1 ? slots_before(p, max(s.keys - s.tokens, 0), tiles_of(p, s)) : 0;
}

// The tile that slot y of a (sequence, head) belongs to.
struct TileOf {
  int j, slot, slots, keys, size;  // the slot's index among the tile's, the keys the tile sees, keys of a slot
};
__device__ __forceinline__ TileOf tile_at(const WeighParams& p, const Sequence& s, long long y) {
  const int old = max(s.keys - s.tokens, 0);
  long long lo = 0, hi = tiles_of(p, s);  // slots_before(lo) <= y < slots_before(hi)
  while (hi - lo > 1) {
    const long long mid = (lo + hi) / 2;
    if (slots_before(p, old, mid) <= y) lo = mid;
    else hi = mid;
  }
  const long long first = slots_before(p, old, lo);
  const int slots = (int)(slots_before(p, old, lo + 1) - first);
  const int last = (int)min((long long)s.tokens, ((lo + 1) * kColumns + p.G - 1) / p.G);  // tokens up to the tile's end
  const int keys = max(s.keys - s.tokens + last, 0);
  return {(int)lo, (int)(y - first), slots, keys, (int)(((keys + slots - 1ll) / slots + 63) / 64 * 64)};
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DP, bool FULL, bool FP8>
__global__ __launch_bounds__(kWeighThreads, DP > 128 ? 1 : 2) void weigh_tiles_kernel(WeighParams p) {
  constexpr int kKeys = DP > 128 ? 32 : 64;  // of a turn
  constexpr int kBlocks = kKeys / 32;
  constexpr int kKRow = DP * 2 + 16, kVRow = DP * 2 + 32;
  constexpr int kBuffer = kKeys * (kKRow + kVRow);
  constexpr int kElem = FP8 ? 1 : 2;
  constexpr int kHalf = DP * kElem / 16, kChunks = 2 * kHalf;  // 16-byte chunks of a key row, of it and its value row
  constexpr int kLoads = kKeys * kChunks / kWeighThreads;
  constexpr int kSteps = DP / 16;
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int s_slot[4][kKeys];
  __shared__ float s_ks[2][kKeys], s_vs[2][kKeys];
  __shared__ int s_bad, s_again;
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 32, half = lane / 32;
  const int count = min(max(*p.num_seqs, 0), p.N);
  const Share share = share_of<true>(count, [&](int i) { return tile_slots(p, sequence_at(p, i)) * p.Hkv; });
  if (share.from == share.to) return;
  const int row_bytes = p.D * kElem;
  const uint64_t row_stride = 2ull * p.Hkv * row_bytes;
  const global_bytes zero = zero_row();
  int seq = share.seq;
  Sequence s = sequence_at(p, seq);
  long long before = share.before, at = share.from;
  while (at < share.to) {
    long long per_head = tile_slots(p, s);
    while (at >= before + per_head * p.Hkv) {
      before += per_head * p.Hkv;
      s = sequence_at(p, ++seq);
      per_head = tile_slots(p, s);
    }
    const int h = (int)((at - before) / per_head);
    const TileOf tile = tile_at(p, s, at - before - h * per_head);
    const int end_slot = (int)min((long long)tile.slots, tile.slot + (share.to - at));
    const int from = (int)min((long long)tile.slot * tile.size, (long long)tile.keys);
    const int to = (int)min((long long)end_slot * tile.size, (long long)tile.keys);
    const int32_t* const table = p.table + (size_t)seq * p.PPS;
    const global_bytes rows = (global_bytes)(uint64_t)p.kv + 2 * (size_t)h * row_bytes;

    // this lane's column; the wave's first and last position
    const int end_row = s.tokens * p.G, row0 = tile.j * kColumns + wave * 32, row = row0 + n;
    const bool live = row < end_row;
    const int token = div_by(min(row, end_row - 1), p.group), g = min(row, end_row - 1) - token * p.G, t = s.first + token;
    const int old = s.keys - s.tokens, pos = live ? old + token : -1;
    const int first_pos = row0 < end_row ? old + div_by(row0, p.group) : -1;
    const int last_pos = row0 < end_row ? old + div_by(min(row0 + 31, end_row - 1), p.group) : -1;
    bf16x8 q[kSteps];
    {
      const uint16_t* src = p.q + t * p.q_token + ((long long)h * p.G + g) * p.q_head;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int dim = 16 * i + 8 * half;
        u32x4 w = {0, 0, 0, 0};
        if (live && (FULL || dim < p.D)) w = *(const u32x4*)(src + dim);
        q[i] = __builtin_bit_cast(bf16x8, w);
      }
    }
    f32x16 o[DP / 32];
    float m, l;
    // Attends to the keys from `from` on, up to position `last`.
    const auto attend = [&](int last) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
      m = kLowest, l = 0.f;
      const int end = min(to, last + 1), units = end > from ? (end - from + kKeys - 1) / kKeys : 0;
      const auto page_of = [&](int unit) {  // threads below kKeys: the page of the unit's tid-th key
        const int key = from + unit * kKeys + tid;
        return key < end ? table[div_by(key, p.page)] : -1;
      };
      const auto keep = [&](int unit, int id) {
        const int key = from + unit * kKeys + tid;
        int slot = -1;
        if (key < end) {
          if (id >= 0 && id < p.P) slot = id * p.S + (key - div_by(key, p.page) * p.S);
          else flag_error(RPA_SPARSE_ERR_PAGE), s_bad = 1;
        }
        s_slot[unit & 3][tid] = slot;
      };
      u32x4 w[kLoads];
      float ks = 1.f, vs = 1.f;
      const auto load = [&](int unit) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int c = tid % kChunks, slot = s_slot[unit & 3][tid / kChunks + i * (kWeighThreads / kChunks)];
          const int part = c >= kHalf, byte = 16 * (c - part * kHalf);
          const global_bytes src = slot >= 0 && (FULL || byte < row_bytes) ? rows + (uint32_t)slot * row_stride : zero;
          w[i] = load16(src + part * row_bytes + byte);
        }
        if (FP8 && p.scales && tid < kKeys) {
          const int slot = s_slot[unit & 3][tid];
          const float* scale = p.scales + ((size_t)div_by(max(slot, 0), p.page) * p.Hkv + h) * 2;
          ks = slot >= 0 ? scale[0] : 1.f, vs = slot >= 0 ? scale[1] : 1.f;
        }
      };
      const auto store = [&](int unit) {
        uint8_t* const buffer = lds + (unit & 1) * kBuffer;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int c = tid % kChunks, key = tid / kChunks + i * (kWeighThreads / kChunks);
          const int part = c >= kHalf, byte = 16 * (c - part * kHalf);
          uint8_t* const dst = buffer + (part ? kKeys * kKRow + key * kVRow : key * kKRow) + byte * (FP8 ? 2 : 1);
          if (FP8) {
            *(u32x4*)dst = bf16_of_codes(w[i][0], w[i][1]);
            *(u32x4*)(dst + 16) = bf16_of_codes(w[i][2], w[i][3]);
          } else {
            *(u32x4*)dst = w[i];
          }
        }
        if (FP8 && tid < kKeys) s_ks[unit & 1][tid] = ks, s_vs[unit & 1][tid] = vs;
      };
      __syncthreads();  // the last use of LDS
      if (tid == 0) s_bad = 0;
      __syncthreads();
      if (tid < kKeys && units > 0) {
        keep(0, page_of(0));
        keep(1, page_of(1));
      }
      __syncthreads();
      if (units > 0) load(0), store(0);
      __syncthreads();
#pragma unroll 1
      for (int unit = 0; unit < units; ++unit) {
        int id = 0;
        if (unit + 1 < units) load(unit + 1);
        if (tid < kKeys && unit + 2 < units) id = page_of(unit + 2);
        const int key0 = from + unit * kKeys;
        if (key0 <= last_pos) {  // uniform
          const uint8_t* const kt = lds + (unit & 1) * kBuffer;
#pragma unroll 1
          for (int b = 0; b < kBlocks; ++b) {
            f32x16 sc;
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
              const u32x4 a = *(const u32x4*)(kt + (32 * b + n) * kKRow + 32 * i + 16 * half);
              sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), q[i], sc, 0, 0, 0);
            }
            const bool whole = key0 + 32 * b + 32 <= min(first_pos + 1, end) && !s_bad;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int key = 32 * b + 8 * (r / 4) + 4 * half + r % 4;
              sc[r] = scaled(sc[r], FP8 ? p.scale * s_ks[unit & 1][key] : p.scale);
            }
            if (p.cap != 0.f) {
#pragma unroll
              for (int r = 0; r < 16; ++r) sc[r] = scaled(p.cap * tanhf(sc[r] / p.cap), kLog2e);
            }
            if (!whole) {
              const int most = min(pos, end - 1);
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int key = 32 * b + 8 * (r / 4) + 4 * half + r % 4;
                const bool counts = key0 + key <= most && s_slot[unit & 3][key] >= 0;
                sc[r] = counts ? sc[r] : -__builtin_inff();
              }
            }
            float top = kLowest;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = max_of(top, sc[r]);
            if (__ballot(top > m + kRescale)) {  // of the lane's own keys: any lane's
              top = fmaxf(top, __shfl_xor(top, 32));
              const float next = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - next);
              m = next;
              l *= f;
#pragma unroll
              for (int d = 0; d < DP / 32; ++d) o[d] *= f;
            }
            typedef __attribute__((address_space(3))) i16x4* lds_i16x4;
            const uint8_t* const vt =
                kt + kKeys * kKRow + (32 * b + 4 * half + lane % 16 / 4) * kVRow + 8 * (lane % 4) + 32 * (lane / 16 % 2);
#pragma unroll
            for (int u = 0; u < 2; ++u) {  // 16 keys: 4 half + 0 .. 3 and 8 + 4 half + 0 .. 3
              u32x4 parts[3];
#pragma unroll
              for (int r = 0; r < 8; r += 2) {
                float e[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  e[x] = __builtin_amdgcn_exp2f(sc[8 * u + r + x] - m);
                  l += e[x];
                  if (FP8) e[x] *= s_vs[unit & 1][32 * b + 16 * u + 8 * (r / 4) + 4 * half + r % 4 + x];
                }
                const Parts two = split_bf16(e[0], e[1]);
#pragma unroll
                for (int i = 0; i < 3; ++i) parts[i][r / 2] = two.of[i];
              }
#pragma unroll
              for (int d = 0; d < DP / 32; ++d) {
                const uint8_t* const v = vt + 16 * u * kVRow + 64 * d;
                const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)v);
                const i16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(v + 8 * kVRow));
                const bf16x8 f = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int i = 0; i < 3; ++i)
                  o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, __builtin_bit_cast(bf16x8, parts[i]), o[d], 0, 0, 0);
              }
            }
          }
        }
        if (unit + 1 < units) store(unit + 1);
        if (tid < kKeys && unit + 2 < units) keep(unit + 2, id);
        __syncthreads();
      }
    };
    const bool own = tile.slot == 0 && end_slot == tile.slots;
    float* const part = p.tile_parts + (2 * (size_t)share.index + (at > share.from)) * (kColumns * (2 + (size_t)p.D));
    // The columns' results: those of token `only`, or all (-1).
    const auto write = [&](int only) {
      const float sum = l + __shfl_xor(l, 32);
      if (!live || (only >= 0 && token != only)) return;
      const int column = wave * 32 + n;
      if (!own) {
        if (half == 0) part[2 * column] = m, part[2 * column + 1] = sum;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const int dim = 32 * d + 8 * a + 4 * half;
            if (FULL || dim < p.D)
              *(f32x4*)(part + 2 * kColumns + (size_t)column * p.D + dim) =
                  f32x4{o[d][4 * a], o[d][4 * a + 1], o[d][4 * a + 2], o[d][4 * a + 3]};
          }
        return;
      }
      const size_t to_row = (size_t)t * p.Hkv * p.G + h * p.G + g;
      const float f = sum == 0.f ? 0.f : p.v_scale / sum;
      if (half == 0) p.stats[to_row] = {m, sum == 0.f ? 0.f : 1.f / sum};
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int dim = 32 * d + 8 * a + 4 * half;
          if (FULL || dim < p.D)
            *(u32x2*)(p.out + to_row * p.D + dim) =
                sum == 0.f ? u32x2{0, 0}
                           : u32x2{pack_bf16(o[d][4 * a] * f, o[d][4 * a + 1] * f), pack_bf16(o[d][4 * a + 2] * f, o[d][4 * a + 3] * f)};
        }
    };
    // Keys that some columns see and others do not may hold infinities or NaN as values, which P = 0 does not silence:
    // where a result is not finite the tile is done again token by token, each reading its own keys only.
    const int first_token = div_by(tile.j * kColumns, p.group);
    const int last_token = div_by(min(tile.j * kColumns + kColumns - 1, end_row - 1), p.group);
#pragma unroll 1
    for (int only = first_token - 1; only <= last_token; ++only) {  // first all of them
      const bool all = only < first_token;
      attend(all ? tile.keys - 1 : old + only);
      if (all) {
        bool finite = true;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) finite &= fabsf(o[d][r]) < __builtin_inff();
        if (tid == 0) s_again = 0;
        __syncthreads();
        if (!finite) s_again = 1;
        __syncthreads();
        if (s_again) continue;
      }
      write(all ? -1 : only);
      if (all) break;
    }
    at += end_slot - tile.slot;
  }
}

// Joins the parts of tiles, as weigh_join_kernel those of rows; kColumns / gridDim.y columns a workgroup.
__global__ __launch_bounds__(kWeighThreads) void weigh_join_tiles_kernel(WeighParams p) {
  const int count = min(max(*p.num_seqs, 0), p.N), index = blockIdx.x;
  const Share share = share_of<false>(count, [&](int i) { return tile_slots(p, sequence_at(p, i)) * p.Hkv; });
  if (share.from == share.to) return;
  const Sequence s = sequence_at(p, share.seq);
  const long long per_head = tile_slots(p, s);
  const int h = (int)((share.from - share.before) / per_head);
  const TileOf tile = tile_at(p, s, share.from - share.before - h * per_head);
  const long long begin = share.from - tile.slot, end = begin + tile.slots;
  if (begin == share.from || end > share.to) return;  // uniform
  const long long each = share.from / index;
  const int first = (int)(begin / each), last = index;
  const int columns = kColumns / gridDim.y, c0 = blockIdx.y * columns, quads = p.D / 4;
  const size_t stride = kColumns * (2 + (size_t)p.D);
  for (int i = threadIdx.x; i < columns * quads; i += kWeighThreads) {
    const int c = c0 + i / quads, d = i % quads * 4, row = tile.j * kColumns + c;
    if (row >= s.tokens * p.G) break;
    float top = kLowest, sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int w = first; w <= last; ++w) {
      const float* part = p.tile_parts + (2 * (size_t)w + (w == first && begin % each != 0)) * stride;
      const float m = part[2 * c], l = part[2 * c + 1];
      if (l == 0.f) continue;
      const f32x4 o = *(const f32x4*)(part + 2 * kColumns + (size_t)c * p.D + d);
      const float next = fmaxf(top, m), mine = __builtin_amdgcn_exp2f(top - next), its = __builtin_amdgcn_exp2f(m - next);
      top = next;
      sum = sum * mine + l * its;
      x = x * mine + o * its;
    }
    const int token = div_by(row, p.group), g = row - token * p.G;
    const size_t to = (size_t)(s.first + token) * p.Hkv * p.G + h * p.G + g;
    const float f = sum == 0.f ? 0.f : p.v_scale / sum;
    if (d == 0) p.stats[to] = {top, sum == 0.f ? 0.f : 1.f / sum};
    *(u32x2*)(p.out + to * p.D + d) =
        sum == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(x[0] * f, x[1] * f), pack_bf16(x[2] * f, x[3] * f)};
  }
}

// The weights of a sequence's keys, a block of them for a kv head at a time.  Of a sequence with one token the scores are
// there, and its block is kScoreKeys.  Of others a block is kWeighKeys, 64 a wave, whose K stays in registers as the
// products' A operand while every row (token, head) that sees one of them passes through LDS, kWeighRows at a time: the
// scores once more.  A lane sums its keys over its columns, and lanes meet once at the end.
constexpr int kScoreKeys = 1024, kWeighRows = 32;

template <int DP, bool FULL, bool FP8>
__global__ __launch_bounds__(kWeighThreads, 2) void weigh_keys_kernel(WeighParams p) {
  constexpr int kElem = FP8 ? 1 : 2;
  constexpr int kSteps = DP / 16;
  constexpr int kWave = DP > 128 ? 32 : 64, kBlocks = kWave / 32;  // keys of a wave
  constexpr int kKeys = kWave * kWeighWaves;
  constexpr int kRow = DP * 2 + 16;
  constexpr int kLoads = kWeighRows * DP * 2 / 16 / kWeighThreads;
  __shared__ __align__(16) uint8_t s_q[2][kWeighRows * kRow];
  __shared__ float2 s_stat[2][kWeighRows];
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 32, half = lane / 32;
  const int count = min(max(*p.num_seqs, 0), p.N);
  const auto blocks_of = [&](const Sequence& s) {
    const int keys = s.tokens == 1 ? kScoreKeys : kKeys;
    return s.tokens ? (s.keys + keys - 1) / keys : 0;
  };
  const Share share = share_of<true>(
      count, [&](int i) { return (long long)blocks_of(sequence_at(p, i, true)) * p.Hkv; },
      [&](int i) { return score_blocks(sequence_at(p, i)); });
  if (share.from == share.to) return;
  const int row_bytes = p.D * kElem;
  const uint64_t row_stride = 2ull * p.Hkv * row_bytes;
  const global_bytes zero = zero_row();
  int seq = share.seq;
  Sequence s = sequence_at(p, seq);
  long long before = share.before, score_at = share.scores;
  for (long long at = share.from; at < share.to; ++at) {
    while (at >= before + (long long)blocks_of(s) * p.Hkv) {
      before += (long long)blocks_of(s) * p.Hkv;
      score_at += score_blocks(s);
      s = sequence_at(p, ++seq);
    }
    const int blocks = blocks_of(s), h = (int)((at - before) / blocks), block = (int)((at - before) - (long long)h * blocks);
    const int32_t* const table = p.table + (size_t)seq * p.PPS;
    const int old = s.keys - s.tokens;  // keys before the step's
    // adds x to a key's weight
    const auto add = [&](int key, float x) {
      const int page = div_by(key, p.page), id = table[page];
      if (id < 0 || id >= p.P) return;
      const size_t to = ((size_t)id * p.Hkv + h) * p.S + (key - page * p.S);
      if (key >= old) p.positions[to] = (p.dropped ? p.dropped[seq] : 0) + key;
      else if (p.decay != 0.f) x += p.decay * p.weights[to];
      p.weights[to] = x;
    };
    const bool kept = scores_fit(p, s, score_at);
    if (kept) {
      const float2* const stat = p.stats + (size_t)s.first * p.Hkv * p.G + h * p.G;
      const int key0 = block * kScoreKeys + 4 * tid;  // this thread's four keys
      if (key0 < s.keys) {
        const float* from = p.scores + (((size_t)score_at + key0 / 16) * p.Hkv + h) * p.G * 16 + key0 % 16;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int g = 0; g < p.G; ++g) {
          const f32x4 x = *(const f32x4*)(from + g * 16);
          const float2 st = stat[g];
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[r] += __builtin_amdgcn_exp2f(x[r] - st.x) * st.y;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + r < s.keys) add(key0 + r, sum[r]);
      }
      continue;
    }
    // a sequence with one token whose scores did not fit: its block in parts
    const int first_key = block * (s.tokens == 1 ? kScoreKeys : kKeys);
    const int end_key = min(s.keys, first_key + (s.tokens == 1 ? kScoreKeys : kKeys));
    for (int part = first_key; part < end_key; part += kKeys) {
      const int key0 = part + kWave * wave;
      const global_bytes rows = (global_bytes)(uint64_t)p.kv + 2 * (size_t)h * row_bytes;
      const auto slot_of = [&](int key) {
        if (key >= s.keys) return -1;
        const int page = div_by(key, p.page), id = table[page];
        return id >= 0 && id < p.P ? id * p.S + (key - page * p.S) : -1;
      };
      bf16x8 k[kBlocks][kSteps];
      float ks[kBlocks];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int slot = slot_of(key0 + 32 * b + n);
        const global_bytes src = slot >= 0 ? rows + (uint32_t)slot * row_stride : zero;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int dim = 16 * i + 8 * half;
          const global_bytes from = FULL || dim < p.D ? src : zero;
          if (FP8) {
            typedef const __attribute__((address_space(1))) u32x2* global_u32x2;
            const u32x2 w = *(global_u32x2)(from + dim);
            k[b][i] = __builtin_bit_cast(bf16x8, bf16_of_codes(w[0], w[1]));
          } else {
            k[b][i] = __builtin_bit_cast(bf16x8, load16(from + 2 * dim));
          }
        }
        ks[b] = FP8 && p.scales && slot >= 0 ? p.scales[((size_t)div_by(slot, p.page) * p.Hkv + h) * 2] : 1.f;
      }
      const int end_row = s.tokens * p.G, begin_row = max(part - old, 0) * p.G;
      u32x4 w[kLoads];
      float2 st = {0.f, 0.f};
      const auto load = [&](int base) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          constexpr int kChunks = DP * 2 / 16;
          const int row = base + tid / kChunks + i * (kWeighThreads / kChunks), dim = tid % kChunks * 8;
          const int token = div_by(min(row, end_row - 1), p.group), g = min(row, end_row - 1) - token * p.G;
          w[i] = u32x4{0, 0, 0, 0};
          if (row < end_row && (FULL || dim < p.D))
            w[i] = *(const u32x4*)(p.q + (s.first + token) * p.q_token + ((long long)h * p.G + g) * p.q_head + dim);
        }
        if (tid < kWeighRows) {
          const int row = base + tid, token = div_by(min(row, end_row - 1), p.group), g = min(row, end_row - 1) - token * p.G;
          st = row < end_row ? p.stats[(size_t)(s.first + token) * p.Hkv * p.G + h * p.G + g] : float2{0.f, 0.f};
        }
      };
      const auto store = [&](int turn) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          constexpr int kChunks = DP * 2 / 16;
          *(u32x4*)(s_q[turn & 1] + (tid / kChunks + i * (kWeighThreads / kChunks)) * kRow + tid % kChunks * 16) = w[i];
        }
        if (tid < kWeighRows) s_stat[turn & 1][tid] = st;
      };
      float sum[kBlocks][16];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[b][r] = 0.f;
      __syncthreads();  // the last use of LDS
      load(begin_row), store(0);
      __syncthreads();
      int turn = 0;
#pragma unroll 1
      for (int base = begin_row; base < end_row; base += kWeighRows, ++turn) {
        if (base + kWeighRows < end_row) load(base + kWeighRows);
        const int first = div_by(base, p.group), last = div_by(min(base + kWeighRows, end_row) - 1, p.group);  // tokens
        if (key0 <= old + last && key0 < s.keys) {  // uniform
          const float2 stat = s_stat[turn & 1][n];
          const bool whole = key0 + kWave - 1 <= old + first && base + kWeighRows <= end_row;
          const int token = div_by(min(base + n, end_row - 1), p.group), seen = base + n < end_row ? old + token : -1;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            f32x16 sc;
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
              const u32x4 x = *(const u32x4*)(s_q[turn & 1] + n * kRow + 32 * i + 16 * half);
              sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[b][i], __builtin_bit_cast(bf16x8, x), sc, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              float scale = p.scale;
              if (FP8) scale *= __shfl(ks[b], 8 * (r / 4) + 4 * half + r % 4);
              sc[r] = scaled(sc[r], scale);
            }
            if (p.cap != 0.f) {
#pragma unroll
              for (int r = 0; r < 16; ++r) sc[r] = scaled(p.cap * tanhf(sc[r] / p.cap), kLog2e);
            }
            if (whole) {
#pragma unroll
              for (int r = 0; r < 16; ++r) sum[b][r] += __builtin_amdgcn_exp2f(sc[r] - stat.x) * stat.y;
            } else {
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const float e = __builtin_amdgcn_exp2f(sc[r] - stat.x) * stat.y;
                sum[b][r] += key0 + 32 * b + 8 * (r / 4) + 4 * half + r % 4 <= seen ? e : 0.f;
              }
            }
          }
        }
        if (base + kWeighRows < end_row) store(turn + 1);
        __syncthreads();
      }
      // over the 32 columns: lane n then has key n's
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        float mine = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float x = sum[b][r];
#pragma unroll
          for (int d = 1; d < 32; d *= 2) x += __shfl_xor(x, d);
          mine = n == r ? x : mine;
        }
        const int key = key0 + 32 * b + 8 * (n / 4) + 4 * half + n % 4;
        if (n < 16 && key < s.keys) add(key, mine);
      }
    }
  }
}

// ---- host side ----
int check_weigh(const rpa_weigh_shape_t* s) {
  if (!s) return fail(RPA_E_INVALID, "shape is NULL");
  rpa_sparse_shape_t t = {s->num_tokens, s->num_q_heads, s->num_kv_heads, s->head_dim, s->total_pages, s->page_size,
                          s->max_num_seqs, s->pages_per_seq, s->kv_dtype, 1, s->q_token_stride, s->q_head_stride};
  const int rc = check_sparse(&t);
  if (rc) return rc;
  if ((long long)s->num_tokens * s->num_q_heads > kMostIndex)
    return fail(RPA_E_INVALID, "num_tokens * num_q_heads must be at most 2^31 - 2^16 - 1");
  if ((long long)s->pages_per_seq * s->page_size > kMostIndex || s->max_num_seqs > kMostIndex)
    return fail(RPA_E_INVALID, "pages_per_seq * page_size and max_num_seqs must be at most 2^31 - 2^16 - 1");
  return RPA_OK;
}

struct WeighPlan {
  int tiles, rows_grid, tiles_grid, keys_grid;  // tiles_grid 0: rows only
  long long score_room;
  size_t stats, parts, scores, bytes;
};

constexpr int kRowsGrid = 768, kTilesGrid = 512, kKeysGrid = 2048;

WeighPlan plan_weigh(const rpa_weigh_shape_t& s) {
  WeighPlan r = {};
  r.tiles = (s.num_q_heads / s.num_kv_heads + 15) / 16;
  const auto most = [](long long a, long long b) { return a > 0 && b > LLONG_MAX / a ? LLONG_MAX : a * b; };
  const long long capacity = (long long)s.pages_per_seq * s.page_size;
  const long long rows = (long long)s.num_tokens * s.num_kv_heads * r.tiles;
  const long long work = most(rows, capacity / kBlockKeys + 1);
  r.rows_grid = (int)(work < kRowsGrid ? work : kRowsGrid);
  const long long seqs = s.num_tokens < s.max_num_seqs ? s.num_tokens : s.max_num_seqs;
  const long long blocks = most(seqs * s.num_kv_heads, capacity / 128 + 1);
  r.keys_grid = (int)(blocks < kKeysGrid ? blocks : kKeysGrid);
  r.stats = ((size_t)s.num_tokens * s.num_q_heads * sizeof(float2) + 15) / 16 * 16;
  r.parts = (size_t)r.rows_grid * 2 * (32 + 16 * (size_t)s.head_dim) * 4;
  // of sequences with one token: their own keys, and no more than the pool holds
  const long long pool = (long long)s.total_pages * s.page_size / 16 + seqs, keys = most(seqs, capacity / 16 + 1);
  r.score_room = pool < keys ? pool : keys;
  r.scores = (size_t)r.score_room * s.num_q_heads * 64;
  r.bytes = r.stats + r.parts + r.scores;
  const int group = s.num_q_heads / s.num_kv_heads;
  // sums of tiles' keys stay in 64 bits
  const bool fits = most(4 * ((long long)s.num_tokens * group + group), capacity) < 1ll << 62;
  if (s.num_tokens > 2 * s.max_num_seqs && fits) {
    const long long tiles = ((long long)s.num_tokens * group + kColumns - 1) / kColumns + seqs;
    const long long slots = most(tiles * s.num_kv_heads, capacity / kBlockKeys + 2), fill = s.head_dim > 128 ? 256 : kTilesGrid;
    r.tiles_grid = (int)(slots < fill ? slots : fill);
    r.bytes += (size_t)r.tiles_grid * 2 * kColumns * (2 + (size_t)s.head_dim) * 4;
  }
  return r;
}

template <int DP, bool FULL, bool FP8>
int launch_weigh(const WeighPlan& plan, const WeighParams& p, hipStream_t stream) {
  weigh_rows_kernel<DP, FULL, FP8><<<plan.rows_grid, kWeighThreads, 0, stream>>>(p);
  int rc = launched("weighed_attention");
  if (rc) return rc;
  weigh_join_kernel<<<plan.rows_grid, kWeighThreads, 0, stream>>>(p);
  if ((rc = launched("weighed_attention (join)"))) return rc;
  if (plan.tiles_grid) {
    const size_t lds = 2 * (DP > 128 ? 32 : 64) * (size_t)(DP * 4 + 48);
    weigh_tiles_kernel<DP, FULL, FP8><<<plan.tiles_grid, kWeighThreads, lds, stream>>>(p);
    if ((rc = launched("weighed_attention (tiles)"))) return rc;
    weigh_join_tiles_kernel<<<dim3(plan.tiles_grid, 8), kWeighThreads, 0, stream>>>(p);
    if ((rc = launched("weighed_attention (join of tiles)"))) return rc;
  }
  weigh_keys_kernel<DP, FULL, FP8><<<plan.keys_grid, kWeighThreads, 0, stream>>>(p);
  return launched("weighed_attention (keys)");
}

}  // namespace
}  // namespace rpa_sparse
