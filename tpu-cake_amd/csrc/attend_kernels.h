// Attention over chosen pages: for each (token, kv head) a list of logical pages of its sequence.
//
// Mathematics: softmax over the keys x of the listed pages up to the token's position, one pass with a
// running maximum m and sum l in fp32 (exp2 domain):  o = sum_x 2^(s_x - m) v_x / sum_x 2^(s_x - m).
// On v_mfma_f32_16x16x32_bf16, 32 keys at a time: S = K Q^T (A: 16 keys x 32 dims, B: the group's heads as
// 16 columns), O^T += V^T P^T (A: 16 dims x 32 keys).  A lane's scores are the keys its P operand needs,
// so P moves between no lanes; V passes through LDS as key rows and comes back transposed
// (ds_read_b64_tr_b16).  P is split into three bf16 parts, each the nearest to what the earlier ones leave, with an
// MFMA each: 24 bits, all that p has, where values cancel too.  Two parts (16 bits) lose what a token's values
// have in common; the third product hides behind a row's loads and takes a chunk's tiles from 92 to 100 us, in fp8
// pools from 104 to 123.  fp8 codes are exact in bf16; K scales multiply the scores and V scales P, both in fp32.
//
// Every listed key of a row is read once, 2 D elem bytes at 2 Hkv D elem apart: HBM bounds decode rows.
// Rows choose apart, so rows are what workgroups share nothing of: one row (its up to 16 heads) a
// workgroup, its keys over four waves, each with its own (m, l, O), joined at the end through LDS.  With
// few rows the list is split over workgroups as well, and a second launch joins their parts.
//
// Measured (8 kv heads of 128, 2048 keys a row): 64 decode rows of 64 heads, 539 MB: 92 us, 5.9 TB/s; of an fp8 pool,
// 271 MB: 59 us, 4.6 TB/s; 2 rows of an fp8 pool, 8.4 MB: 7.4 us and 4.0 for the join, launches and latency.  A plain
// read of 2 GiB reaches 6.3 TB/s.
#pragma once

#include "select_kernels.h"

namespace rpa_sparse {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kRescale = 8.f;      // the running maximum moves when a score passes it by more (log2)
constexpr int kAttendWaves = 4;
constexpr int kMaxBlocks = 1024;     // list blocks of a workgroup

// What keys that do not exist read: zeros, so that P = 0 never meets a NaN.
__device__ uint4 g_zero_row[64];

typedef const __attribute__((address_space(1))) uint8_t* global_bytes;

// Its address, kept in registers: the compiler would load it from the code object's table in every turn.
__device__ __forceinline__ global_bytes zero_row() {
  uint64_t at = (uint64_t)g_zero_row;
  asm volatile("" : "+s"(at));
  return (global_bytes)at;
}

__device__ __forceinline__ u32x4 load16(global_bytes at) {
  return *(const __attribute__((address_space(1))) u32x4*)at;
}

// The larger one, or the one that is a number; fmaxf spends instructions on signalling NaN first.
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, __builtin_inff()); }

struct AttendParams {
  const uint16_t* q;
  const uint8_t* kv;
  const float* scales;
  const int32_t *picked, *kv_lens, *table, *cu, *num_seqs;
  uint16_t* out;
  float* parts;  // splits > 1: (m, l) of 16 rows, then the rows' O, for each (row, split)
  long long q_token, q_head;
  int T, Hkv, G, D, P, S, N, PPS, K;
  int tiles;                // 16-head tiles of a group
  int width, subs, blocks;  // keys of a list block (a page, or 64 keys of one), blocks of a page, of a list
  uint32_t magic;           // ceil(2^32 / width): v / width for v < 2^26 (width > 1)
  int per, splits;          // blocks of a workgroup
  float scale, cap, v_scale;  // scale: of q.k; times log2 e where cap is 0
};

__device__ __forceinline__ u32x4 bf16_of_codes(uint32_t a, uint32_t b) {  // eight e4m3 codes, exactly
  u32x4 w;
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true));
  w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false));
  w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true));
  return w;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// Two values as three bf16 each: the nearest ones, and those nearest to what is left.
struct Parts {
  uint32_t of[3];
};
__device__ __forceinline__ Parts split_bf16(float a, float b) {
  Parts p;
  p.of[0] = pack_bf16(a, b);
  a -= bf16_lo(p.of[0]), b -= bf16_hi(p.of[0]);
  p.of[1] = pack_bf16(a, b);
  p.of[2] = pack_bf16(a - bf16_lo(p.of[1]), b - bf16_hi(p.of[1]));
  return p;
}

// A product that rounds by itself: joined with the subtraction of the maximum into one operation, the maximum's own
// rounding would remain, 2^100 and more for the largest scores.
__device__ __forceinline__ float scaled(float x, float scale) {
#pragma clang fp contract(off)
  return x * scale;
}

__device__ __forceinline__ void cap_scores(f32x4 s[2], float cap) {
#pragma unroll 1
  for (int b = 0; b < 2; ++b) {
    f32x4 x = b ? s[1] : s[0];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = scaled(cap * tanhf(x[r] / cap), kLog2e);
    if (b) s[1] = x;
    else s[0] = x;
  }
}

// DP: dims of a row in registers and LDS (64, 128 or 256), FULL: D == DP.
template <int DP, bool FULL, bool FP8>
__global__ __launch_bounds__(64 * kAttendWaves) void attend_kernel(AttendParams p) {
  constexpr int kRow = DP * 2 + 32;                    // an LDS key row of V
  constexpr int kWave = 32 * kRow;                     // a wave's V; later its 16 rows of O in fp32
  constexpr int kORow = DP + 4;                        // floats
  constexpr int kElem = FP8 ? 1 : 2;
  constexpr int kLoads = DP * kElem / 64;              // 16-byte loads of a lane for a key row's K (or V)
  constexpr int kSteps = DP / 32;
  static_assert(16 * kORow * 4 <= kWave, "O rows fit the wave's V region");
  extern __shared__ __align__(16) uint8_t lds[];
  int* const s_row = (int*)lds;                        // a block's first pool row
  int* const s_len = s_row + p.per;                    // its keys that the token sees
  float* const s_ks = (float*)(s_len + p.per);         // fp8: its scales
  float* const s_vs = s_ks + p.per;
  uint8_t* const s_v = lds + ((size_t)p.per * (FP8 ? 16 : 8) + 15) / 16 * 16;
  __shared__ float s_m[kAttendWaves][16], s_l[kAttendWaves][16];
  __shared__ int s_end;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, n = lane % 16, j = lane / 16;
  const int tile = blockIdx.x % p.tiles, pair = blockIdx.x / p.tiles, h = pair % p.Hkv, t = pair / p.Hkv;
  const int split = blockIdx.y;
  if (tid == 0) s_end = 0;
  const Place at = place_of(p.cu, p.num_seqs, p.kv_lens, p.N, t);
  const int newest = newest_page(at.pos, p.S, p.PPS);
  __syncthreads();
  if (newest >= 0) {
    const int32_t* list = p.picked + (size_t)pair * p.K;
    const int32_t* table = p.table + (size_t)at.seq * p.PPS;
    for (int b = tid; b < p.per; b += 64 * kAttendWaves) {
      const int block = split * p.per + b;
      int row = 0, len = 0;
      float ks = 0.f, vs = 0.f;
      if (block < p.blocks) {
        const int entry = block / p.subs, sub = block % p.subs;
        const int page = list[entry];
        if (page >= 0 && page <= newest) {
          const int first = sub * p.width;
          len = min(min(p.S - first, p.width), at.pos + 1 - (page * p.S + first));
          len = max(len, 0);
          const int phys = table[page];
          if (phys < 0 || phys >= p.P) {
            flag_error(RPA_SPARSE_ERR_PAGE);
            len = 0;
          } else {
            row = phys * p.S + first;
            if (FP8) {
              const float* s = p.scales ? p.scales + ((size_t)phys * p.Hkv + h) * 2 : nullptr;
              ks = s ? s[0] : 1.f, vs = s ? s[1] : 1.f;
            }
          }
        }
      }
      s_row[b] = row;
      s_len[b] = len;
      if (FP8) s_ks[b] = ks, s_vs[b] = vs;
      if (len > 0) atomicMax(&s_end, b + 1);
    }
  }
  __syncthreads();
  const int units = (s_end * p.width + 31) / 32;

  // the group's queries, B operand: column n, dims of k-slot group j
  bf16x8 q[kSteps];
  {
    const int head = tile * 16 + n;
    const uint16_t* src = p.q + t * p.q_token + ((long long)h * p.G + head) * p.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int dim = FP8 ? 64 * (s / 2) + 16 * j + 8 * (s % 2) : 32 * s + 8 * j;
      u32x4 w = {0, 0, 0, 0};
      if (head < p.G && (FULL || dim < p.D)) w = *(const u32x4*)(src + dim);
      q[s] = __builtin_bit_cast(bf16x8, w);
    }
  }

  const int row_bytes = p.D * kElem;
  const uint32_t row_stride = 2u * p.Hkv * row_bytes;
  const global_bytes zero = zero_row(), keys = (global_bytes)(uint64_t)p.kv + 2 * (size_t)h * row_bytes;
  const auto block_of = [&](int v) { return p.width == 1 ? v : (int)__umulhi((uint32_t)v, p.magic); };
  u32x4 k[2][kLoads], v[2][kLoads];
  uint32_t seen[2];  // bit n: key n of the 16 exists
  const auto load = [&](int unit) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int key = unit * 32 + 16 * b + n, block = block_of(key), off = key - block * p.width;
      const int entry = min(block, p.per - 1);
      const bool ok = (block < p.per) & (off < s_len[entry]);
      seen[b] = (uint32_t)__ballot(ok) & 0xffffu;
      const global_bytes key_row = keys + (uint64_t)(uint32_t)(s_row[entry] + off) * row_stride, src = ok ? key_row : zero;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int byte = 64 * i + 16 * j;
        const global_bytes from = FULL || byte < row_bytes ? src : zero;
        k[b][i] = load16(from + byte);
        v[b][i] = load16(from + row_bytes + byte);
      }
    }
  };

  uint8_t* const tile_v = s_v + wave * kWave;
  f32x4 o[DP / 16];
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = kLowest, l = 0.f;
  int unit = wave;
  if (unit < units) load(unit);
  for (; unit < units; unit += kAttendWaves) {
    f32x4 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const u32x4 a = FP8 ? bf16_of_codes(k[b][i / 2][2 * (i % 2)], k[b][i / 2][2 * (i % 2) + 1]) : k[b][FP8 ? 0 : i];
        s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), q[i], s[b], 0, 0, 0);
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
    const bool whole = (seen[0] & seen[1]) == 0xffffu;  // before the next unit's
    const uint32_t here[2] = {seen[0] >> (4 * j), seen[1] >> (4 * j)};
    if (unit + kAttendWaves < units) load(unit + kAttendWaves);

    float vs[2][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float ks[4] = {1.f, 1.f, 1.f, 1.f};
      if (FP8) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int block = min(block_of(unit * 32 + 16 * b + 4 * j + r), p.per - 1);
          ks[r] = s_ks[block], vs[b][r] = s_vs[block];
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) s[b][r] = scaled(s[b][r], FP8 ? p.scale * ks[r] : p.scale);
    }
    if (p.cap != 0.f) cap_scores(s, p.cap);
    if (!whole) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][r] = here[b] >> r & 1 ? s[b][r] : -__builtin_inff();
    }
    float top = max_of(max_of(max_of(s[0][0], s[0][1]), max_of(s[0][2], s[0][3])),
                       max_of(max_of(s[1][0], s[1][1]), max_of(s[1][2], s[1][3])));
    if (__ballot(top > m + kRescale)) {  // of the lane's own keys: any lane's
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
        e[r] = __builtin_amdgcn_exp2f(s[b][r] - m);
        l += e[r];
        if (FP8) e[r] *= vs[b][r];
      }
      const Parts first = split_bf16(e[0], e[1]), second = split_bf16(e[2], e[3]);
#pragma unroll
      for (int i = 0; i < 3; ++i) parts[i][2 * b] = first.of[i], parts[i][2 * b + 1] = second.of[i];
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
  for (int w = 1; w < kAttendWaves; ++w) all = fmaxf(all, s_m[w][n]);
  const float f = __builtin_amdgcn_exp2f(m - all);
  float* const mine = (float*)tile_v + n * kORow;
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) *(f32x4*)(mine + 16 * d + 4 * j) = o[d] * f;
  __syncthreads();
  const int rows = min(p.G - tile * 16, 16), quads = p.D / 4;
  const size_t part = (size_t)blockIdx.x * p.splits + split;
  float* const parts = p.parts + part * (32 + (size_t)min(p.G, 16) * p.D);
  for (int i = tid; i < rows * quads; i += 64 * kAttendWaves) {
    const int r = i / quads, d = i % quads * 4;
    float top = s_m[0][r], sum = 0.f;
#pragma unroll
    for (int w = 1; w < kAttendWaves; ++w) top = fmaxf(top, s_m[w][r]);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kAttendWaves; ++w) {
      sum += s_l[w][r] * __builtin_amdgcn_exp2f(s_m[w][r] - top);
      x += *(const f32x4*)((const float*)(s_v + w * kWave) + r * kORow + d);
    }
    if (p.splits > 1) {
      if (d == 0) parts[2 * r] = top, parts[2 * r + 1] = sum;
      if (sum != 0.f) *(f32x4*)(parts + 32 + r * p.D + d) = x;
      continue;
    }
    const float g = sum == 0.f ? 0.f : p.v_scale / sum;
    *(u32x2*)(p.out + ((size_t)t * p.Hkv * p.G + h * p.G + tile * 16 + r) * p.D + d) =
        sum == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(x[0] * g, x[1] * g), pack_bf16(x[2] * g, x[3] * g)};
  }
}

// The split form's second launch: one workgroup a (row, head tile), a thread for every four dims, the loads of
// kParts parts at once.
__global__ __launch_bounds__(256) void join_kernel(AttendParams p) {
  constexpr int kParts = 8;
  const int tile = blockIdx.x % p.tiles, pair = blockIdx.x / p.tiles, h = pair % p.Hkv, t = pair / p.Hkv;
  const int rows = min(p.G - tile * 16, 16), quads = p.D / 4;
  const size_t stride = 32 + (size_t)min(p.G, 16) * p.D;
  const float* const first = p.parts + (size_t)blockIdx.x * p.splits * stride;
  for (int i = threadIdx.x; i < rows * quads; i += 256) {
    const int r = i / quads, d = i % quads * 4;
    float top = kLowest, sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; s += kParts) {
      float m[kParts], l[kParts];
      f32x4 o[kParts];
#pragma unroll
      for (int u = 0; u < kParts; ++u) {
        const float* part = first + min(s + u, p.splits - 1) * stride;
        m[u] = part[2 * r], l[u] = s + u < p.splits ? part[2 * r + 1] : 0.f;
        o[u] = *(const f32x4*)(part + 32 + r * p.D + d);
      }
#pragma unroll
      for (int u = 0; u < kParts; ++u) {
        if (l[u] == 0.f) continue;  // a part without keys has no O
        const float next = fmaxf(top, m[u]), mine = __builtin_amdgcn_exp2f(top - next), its = __builtin_amdgcn_exp2f(m[u] - next);
        top = next;
        sum = sum * mine + l[u] * its;
        x = x * mine + o[u] * its;
      }
    }
    const float g = sum == 0.f ? 0.f : p.v_scale / sum;
    *(u32x2*)(p.out + ((size_t)t * p.Hkv * p.G + h * p.G + tile * 16 + r) * p.D + d) =
        sum == 0.f ? u32x2{0, 0} : u32x2{pack_bf16(x[0] * g, x[1] * g), pack_bf16(x[2] * g, x[3] * g)};
  }
}

// Prompt chunks: a workgroup takes a tile of up to 64 columns of one sequence -- `tokens` consecutive tokens,
// gp columns each, 16 columns a wave -- and the union of their lists, each page of which is read once, into
// LDS, for all of them.  Neighbouring tokens choose mostly the same pages (in the measured chunk 16 tokens of
// 32 pages each name 44 to 48), so the L2 gives up a tenth of the bytes that rows of their own would ask
// for, and every wave multiplies whole 16-column tiles.  Per 32 keys the four waves read 64 KB of K and V out
// of LDS (512 cycles at 128 B a cycle) beside 512 cycles of MFMA each.  A key counts for a column if its page
// is on the token's own list and it is not past the token's position; a wave passes over 32 keys that none of
// its columns counts.  A page one token lists and another does not may hold infinities or NaN, and P = 0 does
// not silence those: where an output is not finite the tile is done again token by token, each reading its own
// keys only.  Lists that name a page twice are done so at once.
struct TileParams {
  AttendParams a;
  int tokens, gp, shift;      // of a tile; columns of a token and their log2
  uint32_t sub_magic;         // ceil(2^32 / subs)
};

constexpr int kTilePages = 384;        // pages of a union that a workgroup holds at once: two workgroups' LDS fit a CU
constexpr int kTileColumns = 32768;    // page table columns whose bitmaps fit beside them
constexpr int kTileParts = 2048;       // 64-key parts of a page: below it, block / subs by sub_magic is exact

struct alignas(16) TileEntry {
  int row, base, mask, unused;  // the page's first pool row, its first position, the tokens that list it
};

// kGroups groups of four waves take every kGroups-th 32 keys and join at the end.  A turn is bound by what a SIMD
// issues (32 MFMA of 16 cycles and, by the counters, 198 VALU and 34 LDS instructions a wave), by its chain of LDS
// reads, products and exponentials and by waiting for the slowest wave, not by memory: 500 tokens of 32 pages of 64 keys
// beside 5 decode rows (32 heads, 8 kv heads, 128 dims; 304 workgroups) take 112 us with 3 groups, one workgroup a CU,
// and 103 with 2 groups of 128 registers, two workgroups a CU; 700 tokens 125 and 111, 1000 125 and 113, 2000 243 and
// 212; of those that do not fill a CU twice, 60 tokens 25 and 28, 250 tokens 65 and 84.  128 bf16 dims do not fit 128
// registers: 36 are spilled, 104 bytes a lane, which writes 9.5 MB of the 13.8 that 505 tokens write.  fp8, which converts
// as well, would spill 69 and keeps 3 groups (123 us); 256 dims fill the LDS with one workgroup.
template <int DP, bool FULL, bool FP8, int kGroups>
__global__ __launch_bounds__(256 * kGroups, DP < 256 && kGroups == 2 ? 4 : kGroups) void attend_tile_kernel(TileParams tp) {
  const AttendParams& p = tp.a;
  constexpr int kThreads = 256 * kGroups;
  constexpr int kKRow = DP * 2 + 16, kVRow = DP * 2 + 32;  // LDS key rows
  constexpr int kBuffer = 32 * (kKRow + kVRow);
  constexpr int kElem = FP8 ? 1 : 2;
  constexpr int kChunks = DP * kElem / 16;                 // 16-byte chunks of a key row
  constexpr int kLoads = (kChunks + 7) / 8;                // of a thread: 8 threads a key
  constexpr int kSteps = DP / 32;
  extern __shared__ __align__(16) uint8_t lds[];
  static_assert(4 * 16 * (DP + 4) * 4 <= 2 * kBuffer, "a group's rows of O fit its buffers");
  TileEntry* const s_entry = (TileEntry*)(lds + kGroups * 2 * kBuffer);
  float* const s_scale = (float*)(s_entry + kTilePages);   // fp8: K and V scales of the entries
  const int words = (p.PPS + 31) / 32;
  uint32_t* const s_bits = (uint32_t*)(s_scale + (FP8 ? 2 * kTilePages : 0));
  uint32_t* const s_before = s_bits + words;
  __shared__ Pair s_scan[kThreads / 64];
  __shared__ int s_flag[2];  // a page listed twice; an output that is not finite
  __shared__ float s_m[kGroups][64], s_l[kGroups][64];
  const int tid = threadIdx.x, lane = tid % 64, n = lane % 16, j = lane / 16;
  const int group = __builtin_amdgcn_readfirstlane(tid / 256), wave = __builtin_amdgcn_readfirstlane(tid / 64 % 4);
  const int member = tid % 256;
  uint8_t* const s_kv = lds + group * 2 * kBuffer;  // two buffers of the group's own
  const int h = blockIdx.x % p.Hkv;
  const Tile tile = tile_of(p.cu, p.num_seqs, p.kv_lens, p.N, p.T, tp.tokens, blockIdx.x / p.Hkv);
  if (tile.count == 0) return;  // uniform
  const int split = blockIdx.y;
  const auto part_of = [&](int t) {  // of a token: as join_kernel reads it
    return p.parts + (((size_t)(tile.first + t) * p.Hkv + h) * p.splits + split) * (32 + (size_t)p.G * p.D);
  };
  if (tile.seq < 0 || tile.pos + tile.count <= 0) {
    if (p.splits > 1) {
      for (int i = tid; i < tile.count * p.G; i += kThreads) part_of(i / p.G)[2 * (i % p.G) + 1] = 0.f;
      return;
    }
    for (int i = tid; i < tile.count * p.G * p.D / 8; i += kThreads) {
      const int t = i / (p.G * p.D / 8), c = i % (p.G * p.D / 8);
      *(u32x4*)(p.out + ((size_t)(tile.first + t) * p.Hkv + h) * p.G * p.D + 8 * c) = u32x4{0, 0, 0, 0};
    }
    return;
  }
  const int32_t* const table = p.table + (size_t)tile.seq * p.PPS;
  const int32_t* const lists = p.picked + ((size_t)tile.first * p.Hkv + h) * p.K;
  const size_t list_stride = (size_t)p.Hkv * p.K;

  // this lane's column
  const int column = wave * 16 + n, token = column >> tp.shift, head = column & (tp.gp - 1);
  const bool live = token < tile.count && head < p.G;
  const int pos = live ? tile.pos + token : -1;
  bf16x8 q[kSteps];
  {
    const uint16_t* src = p.q + (tile.first + token) * p.q_token + ((long long)h * p.G + head) * p.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int dim = 32 * s + 8 * j;
      u32x4 w = {0, 0, 0, 0};
      if (live && (FULL || dim < p.D)) w = *(const u32x4*)(src + dim);
      q[s] = __builtin_bit_cast(bf16x8, w);
    }
  }

  const int row_bytes = p.D * kElem;
  const uint32_t row_stride = 2u * p.Hkv * row_bytes;
  const global_bytes zero = zero_row(), rows = (global_bytes)(uint64_t)p.kv + 2 * (size_t)h * row_bytes;
  f32x4 o[DP / 16];
  float m, l;
  const auto reset = [&] {
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = kLowest, l = 0.f;
  };

  // Attends to the keys of `pages` entries up to position `last`.
  const auto attend = [&](int pages, int last) {
    const int keys = pages * p.subs * p.width, units = (keys + 31) / 32;
    struct Key {
      int entry, off;  // off: in its page
    };
    const auto locate = [&](int v) {
      const int block = p.width == 1 ? v : (int)__umulhi((uint32_t)v, p.magic);
      const int entry = p.subs == 1 ? block : (int)__umulhi((uint32_t)block, tp.sub_magic);
      const int off = v - block * p.width + (block - entry * p.subs) * p.width;
      return Key{entry, off};
    };
    u32x4 k[kLoads], v[kLoads];
    const auto load = [&](int unit) {  // a thread: key member / 8, chunks member % 8, + 8, ...
      const int at = unit * 32 + member / 8;
      Key x;
      if (p.width % 32 == 0) {  // a page's own 32 keys: found once a wave
        x = locate(unit * 32);
        x.off += member / 8;
      } else {
        x = locate(min(at, keys - 1));
      }
      const TileEntry e = s_entry[x.entry];
      const bool exists = (at < keys) & (e.mask != 0) & (x.off < p.S) & (e.base + x.off <= last);
      const global_bytes key = rows + (uint64_t)(uint32_t)(e.row + x.off) * row_stride, src = exists ? key : zero;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int byte = 16 * (member % 8 + 8 * i);
        if (byte >= DP * kElem) break;
        const global_bytes from = FULL || byte < row_bytes ? src : zero;
        k[i] = load16(from + byte);
        v[i] = load16(from + row_bytes + byte);
      }
    };
    const auto store = [&](int turn) {
      uint8_t* const kt = s_kv + (turn & 1) * kBuffer + member / 8 * kKRow;
      uint8_t* const vt = s_kv + (turn & 1) * kBuffer + 32 * kKRow + member / 8 * kVRow;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int byte = 16 * (member % 8 + 8 * i);
        if (byte >= DP * kElem) break;
        if (FP8) {
          *(u32x4*)(kt + 2 * byte) = bf16_of_codes(k[i][0], k[i][1]);
          *(u32x4*)(kt + 2 * byte + 16) = bf16_of_codes(k[i][2], k[i][3]);
          *(u32x4*)(vt + 2 * byte) = bf16_of_codes(v[i][0], v[i][1]);
          *(u32x4*)(vt + 2 * byte + 16) = bf16_of_codes(v[i][2], v[i][3]);
        } else {
          *(u32x4*)(kt + byte) = k[i];
          *(u32x4*)(vt + byte) = v[i];
        }
      }
    };
    if (group < units) load(group), store(0);
    __syncthreads();
#pragma unroll 1
    for (int turn = 0, unit = group; turn * kGroups < units; ++turn, unit += kGroups) {
      if (unit + kGroups < units) load(unit + kGroups);
      // which of the lane's keys (16 b + 4 j + r) count for its column
      uint32_t counts = 0;
      float ks[2][4], vs[2][4];
      bool inside = false;  // all of the keys lie before the tile's first token
      if (unit >= units) {
      } else if (p.width % 32 == 0) {  // 32 keys lie in one page
        const Key x = locate(unit * 32);
        const TileEntry e = s_entry[x.entry];
        const int base = __builtin_amdgcn_readfirstlane(e.base), mask = __builtin_amdgcn_readfirstlane(e.mask);
        inside = base + x.off + 31 <= tile.pos && x.off + 31 < p.S;
        if (inside) {
          counts = 255;
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int most = min(pos - base, p.S - 1) - x.off - 16 * b - 4 * j;  // of the lane's four, 0 .. most count
            counts |= ((1u << min(max(most + 1, 0), 4)) - 1) << (4 * b);
          }
        }
        counts = mask >> token & 1 ? counts : 0u;
        if (FP8) {
          const float kx = s_scale[2 * x.entry], vx = s_scale[2 * x.entry + 1];
#pragma unroll
          for (int r = 0; r < 8; ++r) ks[r / 4][r % 4] = kx, vs[r / 4][r % 4] = vx;
        }
      } else if (p.width % 16 == 0) {  // 16 keys lie in one page
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int at = unit * 32 + 16 * b;
          const Key x = locate(min(at, keys - 1));
          const TileEntry e = s_entry[x.entry];
          const int most = min(pos - e.base, p.S - 1) - x.off - 4 * j;  // of the lane's four, 0 .. most count
          const uint32_t four = (1u << min(max(most + 1, 0), 4)) - 1;
          counts |= ((at < keys) & (e.mask >> token & 1) ? four : 0u) << (4 * b);
          if (FP8) {
            const float kx = s_scale[2 * x.entry], vx = s_scale[2 * x.entry + 1];
#pragma unroll
            for (int r = 0; r < 4; ++r) ks[b][r] = kx, vs[b][r] = vx;
          }
        }
      } else {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = unit * 32 + 16 * b + 4 * j + r;
            const Key x = locate(min(at, keys - 1));
            const TileEntry e = s_entry[x.entry];
            const bool count = (at < keys) & (e.mask >> token & 1) & (x.off < p.S) & (e.base + x.off <= pos);
            counts |= (uint32_t)count << (4 * b + r);
            if (FP8) ks[b][r] = s_scale[2 * x.entry], vs[b][r] = s_scale[2 * x.entry + 1];
          }
      }
      if (__ballot(counts != 0)) {
        const uint8_t* const kt = s_kv + (turn & 1) * kBuffer;
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const u32x4 a = *(const u32x4*)(kt + (16 * b + n) * kKRow + 64 * i + 16 * j);
            s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), q[i], s[b], 0, 0, 0);
          }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[b][r] = scaled(s[b][r], FP8 ? p.scale * ks[b][r] : p.scale);
        if (p.cap != 0.f) cap_scores(s, p.cap);
        if (__ballot(counts != 255)) {
          if (inside) {
#pragma unroll
            for (int r = 0; r < 8; ++r) s[r / 4][r % 4] = counts ? s[r / 4][r % 4] : -__builtin_inff();
          } else {
#pragma unroll
            for (int r = 0; r < 8; ++r) s[r / 4][r % 4] = counts >> r & 1 ? s[r / 4][r % 4] : -__builtin_inff();
          }
        }
        float top = max_of(max_of(max_of(s[0][0], s[0][1]), max_of(s[0][2], s[0][3])),
                           max_of(max_of(s[1][0], s[1][1]), max_of(s[1][2], s[1][3])));
        if (__ballot(top > m + kRescale)) {  // of the lane's own keys: any lane's
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
            e[r] = __builtin_amdgcn_exp2f(s[b][r] - m);
            l += e[r];
            if (FP8) e[r] *= vs[b][r];
          }
          const Parts first = split_bf16(e[0], e[1]), second = split_bf16(e[2], e[3]);
#pragma unroll
          for (int i = 0; i < 3; ++i) parts[i][2 * b] = first.of[i], parts[i][2 * b + 1] = second.of[i];
        }
        typedef __attribute__((address_space(3))) i16x4* lds_i16x4;
        const uint8_t* const vt = kt + 32 * kKRow + (4 * j + n / 4) * kVRow + 8 * (n % 4);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(vt + 32 * d));
          const i16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(vt + 16 * kVRow + 32 * d));
          const bf16x8 f = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int i = 0; i < 3; ++i)
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, parts[i]), o[d], 0, 0, 0);
        }
      }
      if (unit + kGroups < units) store(turn + 1);
      __syncthreads();
    }
  };
  // The first group's waves take the others' (m, l, O) in.
  const auto join = [&] {
    float* const rows = (float*)(s_kv + wave * 16 * (DP + 4) * 4) + n * (DP + 4);
    if (group) {
      l = swap_sum(l);
      if (j == 0) s_m[group][wave * 16 + n] = m, s_l[group][wave * 16 + n] = l;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) *(f32x4*)(rows + 16 * d + 4 * j) = o[d];
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int g = 1; g < kGroups; ++g) {
        const float other = s_m[g][wave * 16 + n], next = fmaxf(m, other);
        const float mine = __builtin_amdgcn_exp2f(m - next), its = __builtin_amdgcn_exp2f(other - next);
        m = next;
        l = l * mine + (j == 0 ? s_l[g][wave * 16 + n] * its : 0.f);
        const float* const from = rows + g * 2 * kBuffer / 4;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[d] = o[d] * mine + *(const f32x4*)(from + 16 * d + 4 * j) * its;
      }
    }
    __syncthreads();
  };

  const auto finite = [&] {
    bool ok = true;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) ok &= fabsf(o[d][r]) < __builtin_inff();
    return ok;
  };
  // The columns' rows, normalised: those of token `only`, or all (-1).
  const auto write = [&](int only) {
    const float sum = swap_sum(l), g = sum == 0.f ? 0.f : p.v_scale / sum;
    if (!live || group || (only >= 0 && token != only)) return;
    if (p.splits > 1) {
      float* const part = part_of(token);
      if (j == 0) part[2 * head] = m, part[2 * head + 1] = sum;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        if (FULL || 16 * d + 4 * j < p.D) *(f32x4*)(part + 32 + head * p.D + 16 * d + 4 * j) = o[d];
      return;
    }
    uint16_t* const row = p.out + (((size_t)(tile.first + token) * p.Hkv + h) * p.G + head) * p.D;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      const int dim = 16 * d + 4 * j;
      if (FULL || dim < p.D)
        *(u32x2*)(row + dim) = sum == 0.f ? u32x2{0, 0}
                                          : u32x2{pack_bf16(o[d][0] * g, o[d][1] * g), pack_bf16(o[d][2] * g, o[d][3] * g)};
    }
  };
  const auto entry = [&](int i, int page, int mask) {
    const int phys = table[page];
    const bool ok = phys >= 0 && phys < p.P;
    if (!ok) flag_error(RPA_SPARSE_ERR_PAGE);
    s_entry[i] = {ok ? phys * p.S : 0, page * p.S, ok ? mask : 0, 0};
    if (FP8) {
      const float* s = p.scales && ok ? p.scales + ((size_t)phys * p.Hkv + h) * 2 : nullptr;
      s_scale[2 * i] = s ? s[0] : 1.f, s_scale[2 * i + 1] = s ? s[1] : 1.f;
    }
  };

  // the union of the lists, as a bitmap
  const int entries = tile.count * p.K;
  const auto listed = [&](int i, int& t) {  // the page of entry i of all lists, -1: none that its token sees
    t = i / p.K;
    const int page = lists[t * list_stride + (i - t * p.K)];
    return page >= 0 && page <= newest_page(tile.pos + t, p.S, p.PPS) ? page : -1;
  };
  for (int i = tid; i < words; i += kThreads) s_bits[i] = 0;
  if (tid < 2) s_flag[tid] = 0;
  __syncthreads();
  for (int i = tid; i < entries; i += kThreads) {
    int t;
    const int page = listed(i, t);
    if (page >= 0) atomicOr(&s_bits[page / 32], 1u << (page % 32));
  }
  __syncthreads();
  const int each = (words + kThreads - 1) / kThreads;
  Pair found = {0, 0}, total;
  for (int i = tid * each; i < min((tid + 1) * each, words); ++i) found.a += __popc(s_bits[i]);
  uint32_t before = scan_pairs<kThreads / 64>(found, total, s_scan).a;
  for (int i = tid * each; i < min((tid + 1) * each, words); ++i) s_before[i] = before, before += __popc(s_bits[i]);
  const auto rank = [&](int page) { return (int)(s_before[page / 32] + __popc(s_bits[page / 32] & ((1u << (page % 32)) - 1))); };
  // this workgroup's part of the union
  const int each_split = ((int)total.a + p.splits - 1) / p.splits, from = split * each_split;
  const int to = min(from + each_split, (int)total.a);
  reset();
  for (int first = from; first < to; first += kTilePages) {
    const int pages = min(to - first, kTilePages);
    __syncthreads();
    for (int i = tid; i < pages; i += kThreads) s_entry[i].mask = 0;
    __syncthreads();
    for (int i = tid; i < entries; i += kThreads) {
      int t;
      const int page = listed(i, t);
      if (page < 0) continue;
      const int at = rank(page) - first;
      if (at < 0 || at >= pages) continue;
      const int old = atomicOr(&s_entry[at].mask, 1 << t);
      if (old >> t & 1) s_flag[0] = 1;
      s_entry[at].base = page;  // every lister writes the same
    }
    __syncthreads();
    if (s_flag[0]) break;  // uniform: a page listed twice
    for (int i = tid; i < pages; i += kThreads) entry(i, s_entry[i].base, s_entry[i].mask);
    __syncthreads();
    attend(pages, tile.pos + tile.count - 1);
  }
  if (!s_flag[0]) {
    join();
    if (group == 0 && !finite()) s_flag[1] = 1;
    __syncthreads();
  }
  if (!s_flag[0] && !s_flag[1]) {
    write(-1);
    return;
  }
  // token by token
  for (int t = 0; t < tile.count; ++t) {
    reset();
    for (int first = 0; first < p.K; first += kTilePages) {
      const int pages = min(p.K - first, kTilePages);
      __syncthreads();
      for (int i = tid; i < pages; i += kThreads) {
        int own;
        const int page = listed(t * p.K + first + i, own);
        const int at = page >= 0 ? rank(page) : -1;
        if (at >= from && at < to) {
          entry(i, page, 1 << t);
        } else {  // 32 keys may hold some of this entry's: their weights of 0 meet its scales
          s_entry[i] = {0, 0, 0, 0};
          if (FP8) s_scale[2 * i] = s_scale[2 * i + 1] = 1.f;
        }
      }
      __syncthreads();
      attend(pages, tile.pos + t);
    }
    join();
    write(t);
  }
}

// ---- host side ----
int check_attend(const rpa_sparse_shape_t* s) {
  const int rc = check_sparse(s);
  if (rc) return rc;
  const long long subs = s->page_size <= 64 ? 1 : (s->page_size + 63) / 64;
  if (s->num_tokens * (long long)s->num_q_heads > 0x7fffffffll)
    return fail(RPA_E_INVALID, "num_tokens * num_q_heads overflows int32");
  if (s->num_pages * subs > 1 << 24) return fail(RPA_E_UNSUPPORTED, "a list of more than 2^24 pages or 64-key parts of pages");
  return RPA_OK;
}

struct AttendPlan {
  bool chunk;           // tiles of tokens
  int tokens, gp;       // of a tile
  int groups;           // of four waves each
  long long grid;       // its workgroups
  int tiles, width, subs, per, splits;
  long long blocks, rows;
  size_t bytes;
};

constexpr long long kTileFill = 257;   // tiles from which two workgroups share a CU
constexpr int kTileSplits = 8;  // 200 tokens of one kv head take 23 us, 28 with 4, 23 with 16
constexpr long long kAttendFill = 256;  // workgroups below which lists are split: one a CU

AttendPlan plan_attend(const rpa_sparse_shape_t& s) {
  AttendPlan r = {};
  const int G = s.num_q_heads / s.num_kv_heads;
  r.tiles = (G + 15) / 16;
  r.rows = (long long)s.num_tokens * s.num_kv_heads * r.tiles;
  r.width = s.page_size <= 64 ? s.page_size : 64;
  r.subs = (s.page_size + r.width - 1) / r.width;
  r.blocks = (long long)s.num_pages * r.subs;
  // Tiles or rows, by the tokens a table row has: lengths are on the GPU, so rows without tokens count too, and a table
  // with many of them takes rows where tiles would be faster.  A lone token's tile costs as much as sixteen's.  In us, as
  // tiles and as rows (32 heads, 8 kv heads, 128 dims, lists of 32 pages of 64 keys): 64 sequences of 2 tokens 123 and 124,
  // of 3 131 and 179; 64 decode rows beside a chunk of 16 181 and 121, of 66 (two a row) 188 and 174, of 200 208 and 286; 200
  // beside 200 (just below two) 380 and 452; 16 beside 8 72 and 40; 8 sequences of 4 33 and 35.
  if (s.num_tokens > 2 * s.max_num_seqs && G <= 16 && s.pages_per_seq <= kTileColumns && r.subs < kTileParts) {
    r.chunk = true;
    r.gp = G <= 4 ? 4 : G <= 8 ? 8 : 16;
    r.tokens = 64 / r.gp;
    r.grid = (((long long)s.num_tokens + r.tokens - 1) / r.tokens + s.max_num_seqs) * s.num_kv_heads;
    // Few tiles: their unions are split, into parts of at least 256 listed keys, while all parts run at once.  20, 60
    // and 120 tokens of 32 pages of 64 keys (8 kv heads) take 21, 25 and 34 us, unsplit 62, 63 and 64.
    long long splits = kAttendFill / r.grid, most = (long long)s.num_pages * s.page_size / 256;
    splits = splits < most ? splits : most;
    r.splits = splits < 2 ? 1 : splits < kTileSplits ? (int)splits : kTileSplits;
    if (r.splits > 1) r.bytes = (size_t)r.rows * r.splits * (32 + (size_t)G * s.head_dim) * 4;
    r.groups = s.head_dim > 128 || (s.kv_dtype == RPA_KV_BF16 && r.grid * r.splits >= kTileFill) ? 2 : 3;
    return r;
  }
  // a workgroup's part: at least 128 keys, one unit a wave, and at most kMaxBlocks blocks
  const long long least = (128 + r.width - 1) / r.width;
  long long splits = r.rows ? (kAttendFill + r.rows - 1) / r.rows : 1;
  if (splits > (r.blocks + least - 1) / least) splits = (r.blocks + least - 1) / least;
  long long per = (r.blocks + splits - 1) / splits;
  if (per > kMaxBlocks) per = kMaxBlocks;
  r.per = (int)per;
  r.splits = (int)((r.blocks + per - 1) / per);
  if (r.splits > 1) r.bytes = (size_t)r.rows * r.splits * (32 + (size_t)(G < 16 ? G : 16) * s.head_dim) * 4;
  return r;
}

template <int DP, bool FULL, bool FP8>
void launch_attend(const AttendPlan& plan, const AttendParams& p, hipStream_t stream) {
  if (plan.chunk) {
    const TileParams tp = {p, plan.tokens, plan.gp, plan.gp == 4 ? 2 : plan.gp == 8 ? 3 : 4,
                           (uint32_t)(0x100000000ull / plan.subs + 1)};
    const auto launch = [&](auto kernel) {
      const size_t lds = plan.groups * 2 * 32 * (size_t)(DP * 4 + 48) + kTilePages * (sizeof(TileEntry) + (FP8 ? 8 : 0)) +
                         (size_t)((p.PPS + 31) / 32) * 8;
      kernel<<<dim3((unsigned)plan.grid, plan.splits), 256 * plan.groups, lds, stream>>>(tp);
    };
    if constexpr (DP == 256) {
      launch(attend_tile_kernel<DP, FULL, FP8, 2>);
    } else if constexpr (FP8) {
      launch(attend_tile_kernel<DP, FULL, FP8, 3>);
    } else {
      if (plan.groups == 3) launch(attend_tile_kernel<DP, FULL, FP8, 3>);
      else launch(attend_tile_kernel<DP, FULL, FP8, 2>);
    }
    return;
  }
  const size_t lds = ((size_t)plan.per * (FP8 ? 16 : 8) + 15) / 16 * 16 + (size_t)kAttendWaves * 32 * (DP * 2 + 32);
  attend_kernel<DP, FULL, FP8><<<dim3((unsigned)plan.rows, plan.splits), 64 * kAttendWaves, lds, stream>>>(p);
}

}  // namespace
}  // namespace rpa_sparse
