// Prompt chunks in weighed_attention, and what follows rows and tiles.
#pragma once

#include "weigh_kernels.h"

namespace rpa_sparse {
namespace {

// Prompt chunks: tiles of kColumns columns, the (token, head) rows of one sequence and kv head in order, 32 a wave, on
// v_mfma_f32_32x32x16_bf16: S = K Q^T (32 keys x 32 columns), O^T += V^T P^T.  A tile's keys pass through LDS once for
// its four waves, two buffers in turn.  A lane's scores are the keys its P operand needs, as in rows.  Tiles' keys come in
// slots of about kSlotKeys, slots in shares, as blocks of rows do, and shares of the same keys go to one XCD.
//
// Products bound it: two chunks of 777 tokens over 6000 to 16384 keys, 32 heads of 128 over 8, take 193 GFLOP for scores and
// output, 176 us at the 1.1 PFLOP/s of a large bf16 product; P in three parts makes 387 of them, 352 us.  434 us, 0.89
// PFLOP/s of what is issued.  Spread over XCDs at random the whole call took 1097 us where neighbours on one take 809;
// products before the other wave's softmax (s_setprio) 450 where 476; a turn's products and exponentials pipelined in software took
// the same 432 and spilled registers.
constexpr int kColumns = 128, kSlotKeys = 256;

// Slots of a (sequence, head)'s first j tiles, by the keys that the tiles see: old + kColumns (j' + 1) / G each.
__device__ __forceinline__ long long slots_before(const WeighParams& p, int old, long long j) {
  return j + (2 * j * old * p.G + kColumns * j * (j + 1)) / (2 * kSlotKeys * p.G);
}
__device__ __forceinline__ long long tiles_of(const WeighParams& p, const Sequence& s) {
  return ((long long)s.tokens * p.G + kColumns - 1) / kColumns;
}
// Of one kv head; 0 for sequences that rows do.
__device__ __forceinline__ long long tile_slots(const WeighParams& p, const Sequence& s) {
  return s.tokens > 1 ? slots_before(p, max(s.keys - s.tokens, 0), tiles_of(p, s)) : 0;
}

__device__ __forceinline__ long long all_slots(const WeighParams& p, const Sequence& s, bool pad) {
  return pad ? 0 : tile_slots(p, s) * p.Hkv;
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

// Whether 16 bytes of values hold an infinity or NaN.
template <bool FP8>
__device__ __forceinline__ bool not_finite(const u32x4& v) {
  bool is = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (FP8) {  // 0x7f and 0xff: adding 1 to the other seven bits carries into the eighth
      is |= ((v[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    } else {
      is |= (v[i] & 0x7f80u) == 0x7f80u || (v[i] & 0x7f800000u) == 0x7f800000u;
    }
  }
  return is;
}

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
  __shared__ int s_bad, s_again, s_late;
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 32, half = lane / 32;
  const Share share = share_of<true>(p, blockIdx.x, gridDim.x, [&](const Sequence& s, bool pad) { return all_slots(p, s, pad); });
  JoinOf* const joins = p.joins + p.rows_grid;
  if (share.from == share.to) {  // a share of nothing keeps its workgroup's place
    if (tid == 0) joins[blockIdx.x].first = -1;
    return;
  }
  const int row_bytes = p.D * kElem;
  const uint64_t row_stride = 2ull * p.Hkv * row_bytes;
  const global_bytes zero = zero_row();
  int seq = share.seq;
  Sequence s = share.s;
  long long before = share.before, at = share.from;
  while (at < share.to) {
    long long per_head = tile_slots(p, s);
    while (at >= before + per_head * p.Hkv) {
      before += per_head * p.Hkv;
      s = work_sequence(p, share.count, ++seq);
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
      if (tid == 0) s_bad = s_again = s_late = 0;
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
        if (tid < kKeys && unit + 2 < units) id = page_of(unit + 2);
        if (unit + 1 < units) load(unit + 1);
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
            __builtin_amdgcn_s_setprio(1);  // products go before the other wave's softmax: 476 to 450 us
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
        __builtin_amdgcn_s_setprio(0);
        if (unit + 1 < units) store(unit + 1);
        if (tid < kKeys && unit + 2 < units) keep(unit + 2, id);
        __syncthreads();
      }
    };
    const bool own = tile.slot == 0 && end_slot == tile.slots;
    if (at == share.from && tid == 0) {
      JoinOf join = {-1, 0, s.first, h, tile.j, s.tokens * p.G};
      if (tile.slot && end_slot == tile.slots) {
        const long long each = share.from / share.index, begin = at - tile.slot;  // a share before this one has `each`
        join.first = (int)(begin / each), join.late = begin % each != 0;
      }
      joins[share.index] = join;
    }
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
    // where a result is not finite and such a value is there (at most kColumns - 1 keys), the tile is done again token by
    // token, each reading its own keys only.  Results that are not finite for another reason, a query or a value that all
    // columns see, stand: 1 + kColumns / G passes would find them again.
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
        if (live && !finite) s_again = 1;
        __syncthreads();
        if (s_again) {
          const int begin = max(from, old + first_token + 1);
#pragma unroll 1
          for (int i = tid; i < (to - begin) * kHalf; i += kWeighThreads) {
            const int key = begin + i / kHalf, byte = 16 * (i % kHalf), page = div_by(key, p.page), id = table[page];
            if (id < 0 || id >= p.P || byte >= row_bytes) continue;
            const u32x4 v = load16(rows + (uint32_t)(id * p.S + (key - page * p.S)) * row_stride + row_bytes + byte);
            if (not_finite<FP8>(v) || (FP8 && p.scales && !(fabsf(p.scales[((size_t)id * p.Hkv + h) * 2 + 1]) < __builtin_inff())))
              s_late = 1;
          }
          __syncthreads();
          if (s_late) continue;
        }
      }
      write(all ? -1 : only);
      if (all) break;
    }
    at += end_slot - tile.slot;
  }
}

// Joins the parts of tiles, as join_rows those of rows: kColumns / kJoinTiles columns a workgroup.
constexpr int kJoinTiles = 8;

__device__ __forceinline__ void join_tiles(const WeighParams& p, int block) {
  constexpr int kParts = 8;
  const int last = block / kJoinTiles;
  const JoinOf join = p.joins[p.rows_grid + last];
  if (join.first < 0) return;  // uniform
  const int first = join.first, h = join.h;
  const int columns = kColumns / kJoinTiles, c0 = block % kJoinTiles * columns, quads = p.D / 4;
  const size_t stride = kColumns * (2 + (size_t)p.D);
  const auto part_of = [&](int w) { return p.tile_parts + (2 * (size_t)w + (w == first && join.late)) * stride; };
  for (int i = threadIdx.x; i < columns * quads; i += kWeighThreads) {
    const int c = c0 + i / quads, d = i % quads * 4, row = join.tile * kColumns + c;
    if (row >= join.rows) break;
    float top = kLowest, sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int w = first; w <= last; w += kParts) {
      float m[kParts], l[kParts];
      f32x4 o[kParts];
#pragma unroll
      for (int u = 0; u < kParts; ++u) {
        const float* part = part_of(min(w + u, last));
        m[u] = part[2 * c], l[u] = w + u <= last ? part[2 * c + 1] : 0.f;
        o[u] = *(const f32x4*)(part + 2 * kColumns + (size_t)c * p.D + d);
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
    const int token = div_by(row, p.group), g = row - token * p.G;
    const size_t to = (size_t)(join.t + token) * p.Hkv * p.G + h * p.G + g;
    const float f = sum == 0.f ? 0.f : p.v_scale / sum;
    if (d == 0) p.stats[to] = {top, sum == 0.f ? 0.f : 1.f / sum};
    *(u32x2*)(p.out + to * p.D + d) =
        sum == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(x[0] * f, x[1] * f), pack_bf16(x[2] * f, x[3] * f)};
  }
}

// What follows rows and tiles, one launch: the joins, and the weights of the sequences that rows did, which wait for
// neither (they take a row's sum from its parts).
template <int DP, bool FULL, bool FP8>
__global__ __launch_bounds__(kWeighThreads) void weigh_finish_kernel(WeighParams p) {
  const int block = blockIdx.x, rows = p.rows_grid * p.near, tiles = p.tiles_grid * kJoinTiles;
  if (block < rows) join_rows(p, block);
  else if (block < rows + tiles) join_tiles(p, block - rows);
  else weigh_rows<DP, FULL, FP8>(p, block - rows - tiles, gridDim.x - rows - tiles);
}

// The weights of the sequences that tiles did, 256 keys of a kv head at a time, 64 a wave, whose K stays in registers
// as the products' A operand while every row (token, head) that sees one of them passes through LDS, kWeighRows at a time:
// the scores once more.  A lane sums its keys over its columns, and lanes meet once at the end.
// The two chunks above: 97 GFLOP, 88 us; 160, the exponentials beside the products.  fp8 takes 1.4 times as long as bf16 (388 us
// and 284, two chunks of 777 tokens over 9900 and 15700 keys): a shuffle for each score's scale, and 5 registers spilled; 18 in
// bf16 heads that do not fill 128 dims, which take what full ones do.  32 keys a wave take 205 to 235 us where 64
// took 182, as each key pays the rows' reads from LDS.
//
// Where keys are few (at most kSpread blocks of a wave's keys: 64, or 32 for heads of 256), a workgroup has one such block and
// its waves take 32 rows each in turn, straight from memory, as no two waves read the same: a prompt of 2000 tokens 363 to
// 187 us for the whole call, 175 tokens of 16 heads a group over 400 keys 143 to 82, two chunks of 500 over 2000 keys 177 to
// 150.  With both in one kernel 64 sequences of 8 tokens over 4000 keys take 435 us instead of 408; a launch for each costs all
// but those 2 to 5 us.
constexpr int kWeighRows = 64, kSpread = 1024;

template <int DP, bool FULL, bool FP8>
__global__ __launch_bounds__(kWeighThreads, 2) void weigh_keys_kernel(WeighParams p) {
  constexpr int kElem = FP8 ? 1 : 2;
  constexpr int kSteps = DP / 16;
  constexpr int kWave = DP > 128 ? 32 : 64, kBlocks = kWave / 32;  // keys of a wave
  constexpr int kRow = DP * 2 + 16;
  constexpr int kLoads = kWeighRows * DP * 2 / 16 / kWeighThreads;
  __shared__ __align__(16) uint8_t s_q[2][kWeighRows * kRow];
  __shared__ float2 s_stat[2][kWeighRows];
  __shared__ float s_other[kWeighWaves][kBlocks][16][2];
  const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), n = lane % 32, half = lane / 32;
  const bool may_spread = 4ll * p.N * p.Hkv <= kSpread;  // finding the share a second time costs 4 us
  int keys_of = kWave * (may_spread ? 1 : kWeighWaves);  // of the workgroup
  const auto blocks_of = [&](const Sequence& s) { return s.tokens > 1 ? (s.keys + keys_of - 1) / keys_of : 0; };
  const auto amount = [&](const Sequence& s, bool pad) { return pad ? 0 : (long long)blocks_of(s) * p.Hkv; };
  Share share = share_of<true>(p, blockIdx.x, gridDim.x, amount);
  const bool spread = may_spread && share.total <= kSpread;  // the same for every workgroup
  if (may_spread && !spread) keys_of *= kWeighWaves, share = share_of<true>(p, blockIdx.x, gridDim.x, amount);
  if (share.from == share.to) return;
  const int row_bytes = p.D * kElem;
  const uint64_t row_stride = 2ull * p.Hkv * row_bytes;
  const global_bytes zero = zero_row();
  int seq = share.seq;
  Sequence s = share.s;
  long long before = share.before;
  for (long long at = share.from; at < share.to; ++at) {
    while (at >= before + (long long)blocks_of(s) * p.Hkv) {
      before += (long long)blocks_of(s) * p.Hkv;
      s = work_sequence(p, share.count, ++seq);
    }
    const int blocks = blocks_of(s), h = (int)((at - before) / blocks), block = (int)((at - before) - (long long)h * blocks);
    const int32_t* const table = p.table + (size_t)seq * p.PPS;
    const int old = s.keys - s.tokens;  // keys before the step's
    const int part = block * keys_of, key0 = part + (spread ? 0 : kWave * wave);
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
    // This thread's rows of a stage, kApart apart, as (token, head) and where they lie: found once, then stepped.
    constexpr int kChunks = DP * 2 / 16, kApart = kWeighThreads / kChunks;
    const int dim = tid % kChunks * 8, step_tokens = div_by(kWeighRows, p.group), step_heads = kWeighRows - step_tokens * p.G;
    const long long step = step_tokens * p.q_token + step_heads * p.q_head, wrap = p.q_token - p.G * p.q_head;
    const uint16_t* at_q[kLoads];
    int head[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = begin_row + tid / kChunks + i * kApart, token = div_by(row, p.group);
      head[i] = row - token * p.G;
      at_q[i] = p.q + (s.first + token) * p.q_token + ((long long)h * p.G + head[i]) * p.q_head + dim;
    }
    const auto load = [&](int base) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        w[i] = u32x4{0, 0, 0, 0};
        if (base + tid / kChunks + i * kApart < end_row && (FULL || dim < p.D)) w[i] = *(const u32x4*)at_q[i];
        head[i] += step_heads;
        at_q[i] += step;
        if (head[i] >= p.G) head[i] -= p.G, at_q[i] += wrap;
      }
      if (tid < kWeighRows) {
        const int row = base + tid, token = div_by(min(row, end_row - 1), p.group), g = min(row, end_row - 1) - token * p.G;
        st = row < end_row ? p.stats[(size_t)(s.first + token) * p.Hkv * p.G + h * p.G + g] : float2{0.f, 0.f};
      }
    };
    const auto store = [&](int turn) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) *(u32x4*)(s_q[turn & 1] + (tid / kChunks + i * kApart) * kRow + tid % kChunks * 16) = w[i];
      if (tid < kWeighRows) s_stat[turn & 1][tid] = st;
    };
    float sum[kBlocks][16];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[b][r] = 0.f;
    // 32 rows from row0 on; x(i): this lane's row, dims 16 i + 8 half on
    const auto weigh = [&](int row0, float2 stat, auto x) {
      // a sum that is NaN goes into the exponentials, which a mask clears; a factor of NaN would reach the keys that the row
      // does not see, too
      if (!(stat.y == stat.y)) stat = {stat.y, 1.f};
      const int first = div_by(row0, p.group), last = div_by(min(row0 + 32, end_row) - 1, p.group);  // tokens
      if (key0 > old + last || key0 >= s.keys) return;  // uniform
      const bool whole = key0 + kWave - 1 <= old + first && row0 + 32 <= end_row;
      const int token = div_by(min(row0 + n, end_row - 1), p.group), seen = row0 + n < end_row ? old + token : -1;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        f32x16 sc;
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
          sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[b][i], __builtin_bit_cast(bf16x8, x(i)), sc, 0, 0, 0);
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
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = __builtin_amdgcn_exp2f(sc[r] - stat.x);
        if (!whole) {
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[r] = key0 + 32 * b + 8 * (r / 4) + 4 * half + r % 4 <= seen ? sc[r] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[b][r] = __builtin_fmaf(sc[r], stat.y, sum[b][r]);
      }
    };
    __syncthreads();  // the last use of LDS
    if (spread) {
#pragma unroll 1
      for (int row0 = begin_row + 32 * wave; row0 < end_row; row0 += 32 * kWeighWaves) {
        const int row = min(row0 + n, end_row - 1), token = div_by(row, p.group), g = row - token * p.G;
        const uint16_t* const src = p.q + (s.first + token) * p.q_token + ((long long)h * p.G + g) * p.q_head + 8 * half;
        const float2 stat = p.stats[(size_t)(s.first + token) * p.Hkv * p.G + h * p.G + g];
        u32x4 x[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) x[i] = FULL || 16 * i + 8 * half < p.D ? *(const u32x4*)(src + 16 * i) : u32x4{0, 0, 0, 0};
        weigh(row0, row0 + n < end_row ? stat : float2{0.f, 0.f}, [&](int i) { return x[i]; });
      }
    } else {
      load(begin_row), store(0);
      __syncthreads();
      int turn = 0;
#pragma unroll 1
      for (int base = begin_row; base < end_row; base += kWeighRows, ++turn) {
        if (base + kWeighRows < end_row) load(base + kWeighRows);
#pragma unroll 1
        for (int sub = 0; sub < kWeighRows && base + sub < end_row; sub += 32)
          weigh(base + sub, s_stat[turn & 1][sub + n],
                [&](int i) { return *(const u32x4*)(s_q[turn & 1] + (sub + n) * kRow + 32 * i + 16 * half); });
        if (base + kWeighRows < end_row) store(turn + 1);
        __syncthreads();
      }
    }
    // over the 32 columns: lane n then has key n's
    const auto of_block = [&](int b) {
      float mine = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = sum[b][r];
#pragma unroll
        for (int d = 1; d < 32; d *= 2) x += __shfl_xor(x, d);
        mine = n == r ? x : mine;
      }
      return mine;
    };
    if (spread) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const float mine = of_block(b);
        if (n < 16) s_other[wave][b][n][half] = mine;
      }
      __syncthreads();
      if (wave) continue;
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      float mine = 0.f;
      if (!spread) mine = of_block(b);
      else
        for (int w = 0; w < kWeighWaves; ++w) mine += s_other[w][b][n % 16][half];
      const int key = key0 + 32 * b + 8 * (n / 4) + 4 * half + n % 4;
      if (n < 16 && key < s.keys) add_weight(p, seq, h, old, key, mine);
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
  int tiles, near, ways, block_shift, rows_grid, tiles_grid, weigh_grid, keys_grid;  // tiles_grid 0: rows only
  bool few;
  size_t rows_lds;
  long long score_room;
  size_t stats, parts, scores, joins, bytes;
};

// Two workgroups a CU hold tiles (two chunks of 777 tokens over 6000 .. 16384 keys: 839 us, 1036 with 256 of them, 849 with
// 1024); the weights' grids count for little (640 or 2560 of them instead of 1280: 0.5 to 1% more; 1024 or 4096 of keys: the same).
constexpr int kRowsGrid = 256, kTilesGrid = 512, kWeighGrid = 1280, kKeysGrid = 2048;

WeighPlan plan_weigh(const rpa_weigh_shape_t& s) {
  WeighPlan r = {};
  r.tiles = (s.num_q_heads / s.num_kv_heads + 15) / 16;
  const auto most = [](long long a, long long b) { return a > 0 && b > LLONG_MAX / a ? LLONG_MAX : a * b; };
  const long long capacity = (long long)s.pages_per_seq * s.page_size;
  const long long rows = (long long)s.num_tokens * s.num_kv_heads * r.tiles;
  // rows: the waves of a workgroup, as many as its LDS takes, over neighbouring kv heads, then over a head's keys
  // (D 256: four waves, with all registers; eight of fp8 spill, 32 decode sequences with 16 heads over 4 take 157 us, not 100)
  const bool fp8 = s.kv_dtype == RPA_KV_FP8_E4M3;
  const int dims = s.head_dim <= 64 ? 64 : s.head_dim <= 128 ? 128 : 256, waves = dims == 256 ? 4 : kMostWaves;
  r.near = waves;
  while (s.num_kv_heads % r.near) --r.near;
  r.ways = 1;
  while (2 * r.ways * r.near <= waves) r.ways *= 2;
  r.block_shift = 6;
  while ((1 << r.block_shift) < 64 * r.ways) ++r.block_shift;
  r.rows_lds = (size_t)r.near * r.ways * 32 * (dims * 2 + 32 + (fp8 ? 0 : dims * 2 + 16));
  // One workgroup a CU: 64 sequences of 1024 .. 8192 keys, 64 heads of 128 over 8, take 272 us, and 278 with two, whose parts
  // are twice as many; with 32 heads of 64 148 us and 153.
  const long long work = most(rows / r.near, (capacity >> r.block_shift) + 1);
  r.rows_grid = (int)(work < kRowsGrid ? work : kRowsGrid);
  const long long seqs = s.num_tokens < s.max_num_seqs ? s.num_tokens : s.max_num_seqs;
  const long long blocks = most(seqs * s.num_kv_heads, capacity / 128 + 1);
  const long long spread = most(seqs * s.num_kv_heads, capacity / (dims == 256 ? 32 : 64) + 1);  // of a wave's keys
  r.keys_grid = (int)(spread <= kSpread ? spread : blocks < kKeysGrid ? blocks : kKeysGrid);
  r.weigh_grid = (int)(blocks < kWeighGrid ? blocks : kWeighGrid);
  r.stats = ((size_t)s.num_tokens * s.num_q_heads * sizeof(float2) + 15) / 16 * 16;
  r.parts = (size_t)r.rows_grid * 2 * r.near * (32 + 16 * (size_t)s.head_dim) * 4;
  // of sequences with one token: their own keys, and no more than the pool holds
  const long long pool = (long long)s.total_pages * s.page_size / 16 + seqs, keys = most(seqs, capacity / 16 + 1);
  r.score_room = pool < keys ? pool : keys;
  r.scores = (size_t)r.score_room * s.num_q_heads * 64;
  r.bytes = r.stats + r.parts + r.scores;
  const int group = s.num_q_heads / s.num_kv_heads;
  // sums of tiles' keys stay in 64 bits
  const bool fits = most(4 * ((long long)s.num_tokens * group + group), capacity) < 1ll << 62;
  // Tiles where some sequence has more than one token for sure.  32 sequences of 4000 keys, 32 heads of 128 over 8: of 2
  // tokens 226 us, by rows 275; of 4: 231 and 437; of 16: 262 and 1460; one of 65 tokens beside 63 of one: 275 and 479.  A step
  // of single tokens, which the launches would cost 16 of 228 us, has as many tokens as sequences at most.
  if (s.num_tokens > s.max_num_seqs && fits) {
    const long long tiles = ((long long)s.num_tokens * group + kColumns - 1) / kColumns + seqs;
    const long long slots = most(tiles * s.num_kv_heads, capacity / kSlotKeys + 2), fill = s.head_dim > 128 ? 256 : kTilesGrid;
    r.tiles_grid = (int)(slots < fill ? slots : fill);
    r.bytes += (size_t)r.tiles_grid * 2 * kColumns * (2 + (size_t)s.head_dim) * 4;
  }
  // the largest that share_of's sums can be, whatever the offsets say: each sequence may claim all tokens
  const long long claims = most(s.max_num_seqs, s.num_tokens);
  const long long by_rows = most(most(claims, s.num_kv_heads / r.near * r.tiles), (capacity >> r.block_shift) + 2);
  const long long by_tiles = most(most(most(claims, group) / kColumns + s.max_num_seqs, s.num_kv_heads), capacity / kSlotKeys + 2);
  const long long by_keys = most(most(s.max_num_seqs, s.num_kv_heads), capacity / 16 + 2), limit = 1 << 30;
  r.few = s.max_num_seqs <= kFewSeqs && by_rows < limit && by_tiles < limit && by_keys < limit;
  r.joins = (r.bytes + 31) / 32 * 32;
  r.bytes = r.joins + (size_t)(r.rows_grid + r.tiles_grid) * sizeof(JoinOf);
  return r;
}

template <int DP, bool FULL, bool FP8>
int launch_weigh(const WeighPlan& plan, const WeighParams& p, hipStream_t stream) {
  weigh_rows_kernel<DP, FULL, FP8><<<plan.rows_grid, 64 * plan.near * plan.ways, plan.rows_lds, stream>>>(p);
  int rc = launched("weighed_attention");
  if (rc) return rc;
  if (plan.tiles_grid) {
    const size_t lds = 2 * (DP > 128 ? 32 : 64) * (size_t)(DP * 4 + 48);
    weigh_tiles_kernel<DP, FULL, FP8><<<plan.tiles_grid, kWeighThreads, lds, stream>>>(p);
    if ((rc = launched("weighed_attention (tiles)"))) return rc;
  }
  weigh_finish_kernel<DP, FULL, FP8>
      <<<plan.weigh_grid + plan.rows_grid * plan.near + plan.tiles_grid * kJoinTiles, kWeighThreads, 0, stream>>>(p);
  if ((rc = launched("weighed_attention (finish)")) || !plan.tiles_grid) return rc;
  weigh_keys_kernel<DP, FULL, FP8><<<plan.keys_grid, kWeighThreads, 0, stream>>>(p);
  return launched("weighed_attention (keys)");
}

}  // namespace
}  // namespace rpa_sparse
