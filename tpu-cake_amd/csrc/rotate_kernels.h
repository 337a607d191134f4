// Norms and position rotation of a step's queries and keys, one pass over both.
//
// Mathematics: x' = w x rsqrt(mean(x^2) + eps) for each head's row, then its first R dims as R / 2 pairs (a, b),
// each turned: (a cos - b sin, b cos + a sin).  The angle at position n is n f, f the pair's frequency.  In
// fp32 n f is off by 2^-24 n f: by 0.06 radians at a position of a million.  So a frequency is held in turns,
// as a whole number F of 2^-64: n F mod 2^64 is the angle without its whole turns, exactly, at any position.
// Its first two bits (rounded) say the quarter turn, the rest, within an eighth of a turn, goes through the
// Taylor sums of sine and cosine to a^9 and a^10 (off by 2^-29 there at most).  No table is read.
//
// HBM bounds long batches: every row is read and written once.  A wave takes a token: its lanes share out the
// pairs' sines and cosines, pass them through LDS, and each then turns the same pairs of every head.  In the
// half layout a lane holds V values of each half, so a pair meets in one lane and nothing is exchanged but
// the norm's sum.
//
// 6750 prompt tokens of 64 + 8 heads of 128, half of each turned: 249 MB, 45 us, 5.5 TB/s (a copy of 4 GiB: 4.6; 39.5 us at
// a plain read's 6.3).  54 us where a lane's two values were not whole lines' parts; rows loaded ahead, nontemporal accesses and
// an unrolled loop over heads changed nothing.  64 decode tokens: 5 us on the GPU, 10.6 a call, of which 3.5 are the two output
// tensors and 3.9 the call into the library.
#pragma once

#include "select_kernels.h"

namespace rpa_sparse {
namespace {

struct RotateParams {
  const uint16_t *q, *k;
  uint16_t *q_out, *k_out;
  const void *q_weight, *k_weight;
  const int32_t *positions, *cu, *num_seqs, *dropped;
  const uint64_t* turns;
  long long q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head, qw_head, kw_head;
  int T, Hq, Hkv, D, R, N;
  int parts;         // waves of a token
  int team;          // lanes of a row: D / (2 V) rounded up to a power of two
  int wide_weight;   // weights are fp32
  int keep;          // in place: rows past the last stay
  float eps, magnitude;
};

// Cosine and sine of `turn` / 2^64 of a full turn.
__device__ __forceinline__ float2 cos_sin(uint64_t turn) {
  const uint32_t top = (uint32_t)((turn + 0x80000000ull) >> 32);  // to 2^-32 of a turn, 1.5e-9 radians
  const uint32_t quarter = (top + 0x20000000u) >> 30;
  const float a = (float)(int32_t)(top - (quarter << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float a2 = a * a;
  const float s = a * (1.f + a2 * (-1.f / 6 + a2 * (1.f / 120 + a2 * (-1.f / 5040 + a2 * (1.f / 362880)))));
  const float c = 1.f + a2 * (-0.5f + a2 * (1.f / 24 + a2 * (-1.f / 720 + a2 * (1.f / 40320 + a2 * (-1.f / 3628800)))));
  const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
  return {(quarter + 1) & 2 ? -x : x, quarter & 2 ? -y : y};
}

template <int V>
struct Values;  // V bf16 values as they are loaded
template <>
struct Values<8> {
  typedef u32x4 type;
};
template <>
struct Values<4> {
  typedef u32x2 type;
};

__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

template <int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotate_kernel(RotateParams p) {
  typedef typename Values<V>::type Word;
  extern __shared__ __align__(16) float2 s_turned[];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const long long item = (long long)blockIdx.x * 4 + wave;
  const int t = (int)(item / p.parts), part = (int)(item - (long long)t * p.parts);
  if (t >= p.T) return;
  const int pairs = p.R / 2, rows = p.Hq + p.Hkv;
  const int teams = 64 / p.team, mine = lane / p.team, c = lane % p.team;
  long long at = p.positions[t];
  bool live = true;
  if (p.cu) {
    const Place place = place_of(p.cu, p.num_seqs, p.dropped ? p.dropped : p.cu, p.N, t);
    live = place.seq >= 0;
    if (live && p.dropped) at += p.dropped[place.seq];
  }
  if (!live && p.keep) return;
  float2* const turned = s_turned + wave * pairs;
  for (int i = lane; i < pairs; i += 64) {
    float2 x = cos_sin(p.turns[i] * (uint64_t)at);
    x.x *= p.magnitude, x.y *= p.magnitude;
    turned[i] = x;
  }
  wave_fence();
  // This lane's values: V from `a` on and V from `b` on, both in order over the lanes, so that a load takes whole lines.  In the
  // half layout they are pairs' two sides, interleaved each holds V / 2 pairs.
  const int half = p.D / 2, plain = c - pairs / V;  // plain: of the lanes that hold what is not turned
  const bool inside = c < p.D / (2 * V), turns = INTERLEAVED || c * V < pairs;
  const int a = turns ? V * c : p.R + V * plain;
  const int b = INTERLEAVED ? half + V * c : turns ? pairs + V * c : p.R + (p.D - p.R) / 2 + V * plain;
  float cosine[V], sine[V];
  bool turn[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int pair = INTERLEAVED ? (i < V / 2 ? a / 2 + i : b / 2 + i - V / 2) : c * V + i;
    turn[i] = pair < pairs;
    const float2 x = turn[i] ? turned[pair] : float2{1.f, 0.f};
    cosine[i] = x.x, sine[i] = x.y;
  }
  for (int base = part * teams; base < rows; base += p.parts * teams) {
    const int row = base + mine;
    const bool ok = inside && row < rows, query = row < p.Hq;
    const int head = query ? row : row - p.Hq;
    const uint16_t* const src = query ? p.q + t * p.q_token + head * p.q_head : p.k + t * p.k_token + head * p.k_head;
    Word wa = {}, wb = {};
    if (ok && live) wa = *(const Word*)(src + a), wb = *(const Word*)(src + b);
    float x[V], y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = i % 2 ? bf16_hi(wa[i / 2]) : bf16_lo(wa[i / 2]);
      y[i] = i % 2 ? bf16_hi(wb[i / 2]) : bf16_lo(wb[i / 2]);
    }
    const void* const weight = query ? p.q_weight : p.k_weight;
    if (p.q_weight || p.k_weight) {  // uniform: rows of both kinds go through the sums
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) sum += x[i] * x[i] + y[i] * y[i];
      for (int d = p.team / 2; d; d /= 2) sum += __shfl_xor(sum, d);
      if (weight && ok) {
        const float inv = 1.f / sqrtf(sum / p.D + p.eps);
        const long long from = head * (query ? p.qw_head : p.kw_head);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float u, v;
          if (p.wide_weight) {
            u = ((const float*)weight)[from + a + i], v = ((const float*)weight)[from + b + i];
          } else {
            u = bf16_lo(((const uint16_t*)weight)[from + a + i]), v = bf16_lo(((const uint16_t*)weight)[from + b + i]);
          }
          x[i] *= inv * u, y[i] *= inv * v;
        }
      }
    }
    if (!ok) continue;
    if (INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float* const z = i < V / 2 ? x + 2 * i : y + 2 * i - V;
        const float u = z[0], v = z[1];
        // others keep infinities that a product with 0 would not
        z[0] = turn[i] ? u * cosine[i] - v * sine[i] : u, z[1] = turn[i] ? v * cosine[i] + u * sine[i] : v;
      }
    } else if (turns) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = x[i], v = y[i];
        x[i] = u * cosine[i] - v * sine[i], y[i] = v * cosine[i] + u * sine[i];
      }
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) wa[i] = two_bf16(x[2 * i], x[2 * i + 1]), wb[i] = two_bf16(y[2 * i], y[2 * i + 1]);
    if (!live) wa = Word{}, wb = Word{};
    uint16_t* const dst = query ? p.q_out + t * p.qo_token + head * p.qo_head : p.k_out + t * p.ko_token + head * p.ko_head;
    *(Word*)(dst + a) = wa, *(Word*)(dst + b) = wb;
  }
}

// ---- host side ----
int check_rotate(const rpa_rotate_shape_t* s) {
  if (!s) return fail(RPA_E_INVALID, "shape is NULL");
  if (s->num_tokens < 0) return fail(RPA_E_INVALID, "negative num_tokens");
  if (s->num_tokens >= 1 << 30) return fail(RPA_E_INVALID, "num_tokens must be below 2^30");
  if (s->num_q_heads <= 0) return fail(RPA_E_INVALID, "non-positive dimension in shape");
  if (s->num_q_heads > 1 << 24) return fail(RPA_E_UNSUPPORTED, "more than 2^24 query heads");
  const int rc = check_heads(s->num_kv_heads, s->head_dim, RPA_KV_BF16);
  if (rc) return rc;
  if (s->interleaved != 0 && s->interleaved != 1) return fail(RPA_E_INVALID, "interleaved must be 0 or 1");
  if (s->rotated < 0 || s->rotated > s->head_dim || s->rotated % (s->interleaved ? 2 : 8))
    return fail(RPA_E_INVALID, "rotated=%d must be a multiple of %d in [0, %d]", s->rotated, s->interleaved ? 2 : 8, s->head_dim);
  if (s->weight_bytes != 2 && s->weight_bytes != 4) return fail(RPA_E_INVALID, "weight_bytes must be 2 or 4");
  return RPA_OK;
}

// Whether rows of a may lie in rows of b: not if both are blocks at the same distance and a's lie between b's.
bool rows_meet(const Memory& a, const Memory& b) {
  const auto end = [](const Memory& m) { return (uintptr_t)m.at + (m.outer - 1) * m.step + m.bytes; };
  if (a.bytes <= 0 || b.bytes <= 0 || a.outer <= 0 || b.outer <= 0) return false;
  if (end(a) <= (uintptr_t)b.at || end(b) <= (uintptr_t)a.at) return false;
  if (a.step != b.step || a.step <= 0) return true;
  long long off = ((long long)((uintptr_t)b.at - (uintptr_t)a.at)) % a.step;
  if (off < 0) off += a.step;
  return off < a.bytes || off + b.bytes > a.step;
}

}  // namespace
}  // namespace rpa_sparse
