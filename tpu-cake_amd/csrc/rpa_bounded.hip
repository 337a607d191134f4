// librpa_bounded: the C ABI of include/rpa_bounded.h over its kernels.
#include <float.h>
#include <limits.h>
#include <stdarg.h>
#include <stdio.h>

#include "rpa_bounded.h"

#include "evict_kernels.h"
#include "rotate_kernels.h"
#include "weigh_tiles.h"

using namespace rpa_sparse;

extern "C" {

int rpa_bounded_abi_version(void) { return RPA_BOUNDED_ABI_VERSION; }

const char* rpa_bounded_last_error(void) { return g_last_error; }

int rpa_bounded_read_error_word(int32_t* host_word, int32_t clear, void* stream) {
  if (!host_word) return fail(RPA_E_INVALID, "host_word is NULL");
  const hipStream_t s = (hipStream_t)stream;
  if (hipMemcpyFromSymbolAsync(host_word, HIP_SYMBOL(g_error_word), sizeof(int32_t), 0, hipMemcpyDeviceToHost, s) !=
          hipSuccess ||
      hipStreamSynchronize(s) != hipSuccess)
    return fail(RPA_E_HIP, "reading the error word failed");
  if (clear && *host_word) {
    clear_error_kernel<<<1, 1, 0, s>>>(*host_word);
    if (hipGetLastError() != hipSuccess || hipStreamSynchronize(s) != hipSuccess)
      return fail(RPA_E_HIP, "clearing the error word failed");
  }
  return RPA_OK;
}

int rpa_rotate_heads(const rpa_rotate_shape_t* shape, float eps, float magnitude, const void* q, const void* k,
                     const int32_t* positions, const uint64_t* turns, const void* q_weight, const void* k_weight,
                     const int32_t* cu_q_lens, const int32_t* num_seqs, const int32_t* dropped, void* q_out,
                     void* k_out, void* stream) {
  int rc = check_rotate(shape);
  if (rc) return rc;
  const rpa_rotate_shape_t& s = *shape;
  if (s.num_tokens == 0) return RPA_OK;
  if (!q || !k || !positions || (s.rotated && !turns) || !q_out || !k_out || !cu_q_lens != !num_seqs)
    return fail(RPA_E_INVALID, "NULL tensor pointer");
  if (dropped && !cu_q_lens) return fail(RPA_E_INVALID, "dropped needs cu_q_lens");
  if (cu_q_lens && (s.max_num_seqs <= 0 || s.max_num_seqs > kMostIndex))
    return fail(RPA_E_INVALID, "max_num_seqs must be in [1, 2^31 - 2^16 - 1]");
  if ((rc = check_strides("q", q, s.q_token_stride, s.q_head_stride)) ||
      (rc = check_strides("k", k, s.k_token_stride, s.k_head_stride)) ||
      (rc = check_strides("q_out", q_out, s.q_out_token_stride, s.q_out_head_stride)) ||
      (rc = check_strides("k_out", k_out, s.k_out_token_stride, s.k_out_head_stride)))
    return rc;
  for (long long x : {s.q_token_stride, s.q_head_stride, s.k_token_stride, s.k_head_stride, s.q_out_token_stride,
                      s.q_out_head_stride, s.k_out_token_stride, s.k_out_head_stride, s.q_weight_stride, s.k_weight_stride})
    if (x < 0) return fail(RPA_E_INVALID, "negative stride");
  const long long T = s.num_tokens, D = s.head_dim, N = cu_q_lens ? s.max_num_seqs : 0;
  const bool q_here = q_out == q && s.q_out_token_stride == s.q_token_stride && s.q_out_head_stride == s.q_head_stride;
  const bool k_here = k_out == k && s.k_out_token_stride == s.k_token_stride && s.k_out_head_stride == s.k_head_stride;
  if (q_here != k_here) return fail(RPA_E_INVALID, "q_out and k_out must both be in place or both have memory of their own");
  const auto weight = [&](const char* name, const void* at, long long heads, long long stride) {
    return Memory{name, at, s.weight_bytes * ((heads - 1) * stride + D)};
  };
  const Memory in[] = {rows_of("q", q, T, s.num_q_heads, D, s.q_token_stride, s.q_head_stride),
                       rows_of("k", k, T, s.num_kv_heads, D, s.k_token_stride, s.k_head_stride),
                       {"positions", positions, 4 * T}, {"turns", turns, 4ll * s.rotated},
                       weight("q_weight", q_weight, s.num_q_heads, s.q_weight_stride),
                       weight("k_weight", k_weight, s.num_kv_heads, s.k_weight_stride),
                       {"cu_q_lens", cu_q_lens, 4 * (N + 1)}, {"num_seqs", num_seqs, 4}, {"dropped", dropped, 4 * N}};
  const Memory out[] = {rows_of("q_out", q_out, T, s.num_q_heads, D, s.q_out_token_stride, s.q_out_head_stride),
                        rows_of("k_out", k_out, T, s.num_kv_heads, D, s.k_out_token_stride, s.k_out_head_stride)};
  for (int o = 0; o < 2; ++o)
    for (int i = 0; i < 9; ++i)
      if (in[i].at && !(q_here && o == i) && rows_meet(in[i], out[o]))
        return fail(RPA_E_INVALID, "%s overlaps %s: outputs need memory of their own", out[o].name, in[i].name);
  for (const Memory& o : out)  // its own rows have to differ
    if (o.outer > 1 && o.step < o.bytes) return fail(RPA_E_INVALID, "rows of %s overlap", o.name);
  const bool by_token = s.q_out_token_stride >= s.q_out_head_stride, k_by_token = s.k_out_token_stride >= s.k_out_head_stride;
  if (((by_token ? s.num_q_heads : T) > 1 && (by_token ? s.q_out_head_stride : s.q_out_token_stride) < D) ||
      ((k_by_token ? s.num_kv_heads : T) > 1 && (k_by_token ? s.k_out_head_stride : s.k_out_token_stride) < D))
    return fail(RPA_E_INVALID, "rows of an output overlap");
  if (rows_meet(out[0], out[1])) return fail(RPA_E_INVALID, "k_out overlaps q_out: outputs need memory of their own");

  const bool eight = D % 16 == 0 && (s.interleaved || s.rotated % 16 == 0);
  const int lanes = (int)D / (eight ? 16 : 8), rows = s.num_q_heads + s.num_kv_heads;
  int team = 1;
  while (team < lanes) team *= 2;
  const long long turns_of_wave = (rows + 64 / team - 1) / (64 / team);
  long long parts = 2048 / T;  // few tokens: their heads over several waves
  parts = parts < 1 ? 1 : parts > turns_of_wave ? turns_of_wave : parts;
  const long long grid = (T * parts + 3) / 4;
  if ((rc = check_launch(grid, 256))) return rc;
  const RotateParams p = {(const uint16_t*)q, (const uint16_t*)k, (uint16_t*)q_out, (uint16_t*)k_out, q_weight, k_weight, positions,
                          cu_q_lens, num_seqs, dropped, turns, s.q_token_stride, s.q_head_stride, s.k_token_stride, s.k_head_stride,
                          s.q_out_token_stride, s.q_out_head_stride, s.k_out_token_stride, s.k_out_head_stride, s.q_weight_stride,
                          s.k_weight_stride, s.num_tokens, s.num_q_heads, s.num_kv_heads, s.head_dim, s.rotated, (int)N, (int)parts,
                          team, s.weight_bytes == 4, q_here, eps, magnitude};
  const size_t lds = 4 * (size_t)(s.rotated / 2) * sizeof(float2);
  const auto kernel = eight ? (s.interleaved ? rotate_kernel<8, true> : rotate_kernel<8, false>)
                            : (s.interleaved ? rotate_kernel<4, true> : rotate_kernel<4, false>);
  kernel<<<(unsigned)grid, 256, lds, (hipStream_t)stream>>>(p);
  return launched("rotate_heads");
}

size_t rpa_weigh_workspace_size(const rpa_weigh_shape_t* shape) {
  return check_weigh(shape) == RPA_OK ? plan_weigh(*shape).bytes : 0;
}

int rpa_weighed_attention(const rpa_weigh_shape_t* shape, const rpa_weigh_options_t* options, const void* q,
                          const void* kv_pages, const float* kv_scales, const int32_t* kv_lens,
                          const int32_t* page_indices, const int32_t* cu_q_lens, const int32_t* num_seqs,
                          const int32_t* dropped, float* weights, int32_t* positions, void* out, void* workspace,
                          size_t workspace_bytes, void* stream) {
  int rc = check_weigh(shape);
  if (rc) return rc;
  if (!options) return fail(RPA_E_INVALID, "options is NULL");
  if (!(options->decay >= 0.f && options->decay <= FLT_MAX)) return fail(RPA_E_INVALID, "decay must not be negative, and finite");
  if (shape->num_tokens == 0) return RPA_OK;
  if (!q || !kv_pages || !kv_lens || !page_indices || !cu_q_lens || !num_seqs || !weights || !positions || !out)
    return fail(RPA_E_INVALID, "NULL tensor pointer");
  const rpa_weigh_shape_t& s = *shape;
  const bool fp8 = s.kv_dtype == RPA_KV_FP8_E4M3;
  if (kv_scales && !fp8) return fail(RPA_E_INVALID, "kv_scales requires fp8 kv_pages");
  if ((rc = check_strides("q", q, s.q_token_stride, s.q_head_stride))) return rc;
  if (!aligned16(kv_pages) || !aligned16(out)) return fail(RPA_E_INVALID, "kv_pages and out must be 16-byte aligned");
  const WeighPlan plan = plan_weigh(s);
  if (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace))
    return fail(RPA_E_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  const long long T = s.num_tokens, Hq = s.num_q_heads, Hkv = s.num_kv_heads, D = s.head_dim;
  const long long N = s.max_num_seqs, pool = (long long)s.total_pages * s.page_size;
  const Memory in[] = {rows_of("q", q, T, Hq, D, s.q_token_stride, s.q_head_stride),
                       {"kv_pages", kv_pages, pool * 2 * Hkv * D * (fp8 ? 1 : 2)}, {"kv_scales", kv_scales, 8ll * s.total_pages * Hkv},
                       {"kv_lens", kv_lens, 4 * N}, {"page_indices", page_indices, 4 * N * s.pages_per_seq},
                       {"cu_q_lens", cu_q_lens, 4 * (N + 1)}, {"num_seqs", num_seqs, 4}, {"dropped", dropped, 4 * N},
                       {"workspace", workspace, (long long)plan.bytes}};
  const Memory rows = {"out", out, 2 * T * Hq * D}, sums = {"weights", weights, 4 * pool * Hkv};
  const Memory places = {"positions", positions, 4 * pool * Hkv};
  if ((rc = check_separate(rows, in)) || (rc = check_separate(sums, in)) || (rc = check_separate(places, in)) ||
      (rc = check_separate(rows, {sums, places})) || (rc = check_separate(sums, {places})))
    return rc;
  const float cap = options->soft_cap < 0.f ? -options->soft_cap : options->soft_cap;
  WeighParams p = {};
  p.q = (const uint16_t*)q, p.kv = (const uint8_t*)kv_pages, p.scales = kv_scales;
  p.kv_lens = kv_lens, p.table = page_indices, p.cu = cu_q_lens, p.num_seqs = num_seqs, p.dropped = dropped;
  p.weights = weights, p.positions = positions, p.out = (uint16_t*)out;
  p.stats = (float2*)workspace, p.parts = (float*)((uint8_t*)workspace + plan.stats);
  p.q_token = s.q_token_stride, p.q_head = s.q_head_stride;
  p.T = s.num_tokens, p.Hkv = s.num_kv_heads, p.G = s.num_q_heads / s.num_kv_heads, p.D = s.head_dim;
  p.P = s.total_pages, p.S = s.page_size, p.N = s.max_num_seqs, p.PPS = s.pages_per_seq;
  p.near = plan.near, p.ways = plan.ways, p.block_shift = plan.block_shift, p.one_page = s.page_size % 32 == 0, p.few = plan.few;
  p.rows_grid = plan.rows_grid, p.tiles_grid = plan.tiles_grid;
  p.joins = (JoinOf*)((uint8_t*)workspace + plan.joins);
  p.quads = s.page_size % 4 == 0 && aligned16(weights);
  p.chunk = plan.tiles_grid > 0, p.score_room = plan.score_room;
  p.scores = (float*)((uint8_t*)workspace + plan.stats + plan.parts);
  p.tile_parts = (float*)((uint8_t*)workspace + plan.stats + plan.parts + plan.scores);
  p.tiles = plan.tiles, p.page = divisor(s.page_size), p.group = divisor(p.G);
  p.scale = options->sm_scale * options->k_scale * (cap != 0.f ? 1.f : kLog2e), p.cap = cap;
  p.v_scale = options->v_scale, p.decay = options->decay;
  const hipStream_t stream_ = (hipStream_t)stream;
  if (fp8) {
    if (D == 256) return launch_weigh<256, true, true>(plan, p, stream_);
    if (D == 128) return launch_weigh<128, true, true>(plan, p, stream_);
    if (D == 64) return launch_weigh<64, true, true>(plan, p, stream_);
    return launch_weigh<128, false, true>(plan, p, stream_);
  }
  if (D == 256) return launch_weigh<256, true, false>(plan, p, stream_);
  if (D == 128) return launch_weigh<128, true, false>(plan, p, stream_);
  if (D == 64) return launch_weigh<64, true, false>(plan, p, stream_);
  if (D < 64) return launch_weigh<64, false, false>(plan, p, stream_);
  return launch_weigh<128, false, false>(plan, p, stream_);
}

size_t rpa_choose_workspace_size(const rpa_choose_shape_t* shape) {
  return check_choose(shape) == RPA_OK ? plan_choose(*shape).bytes : 0;
}

int rpa_choose_moves(const rpa_choose_shape_t* shape, const float* weights, const int32_t* positions,
                     const int32_t* kv_lens, const int32_t* page_indices, const int32_t* num_seqs,
                     const int32_t* dropped, int32_t* moves, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_choose(shape);
  if (rc) return rc;
  if (!weights || !positions || !kv_lens || !page_indices || !num_seqs || !moves)
    return fail(RPA_E_INVALID, "NULL tensor pointer");
  const rpa_choose_shape_t& s = *shape;
  const ChoosePlan plan = plan_choose(s);
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace)))
    return fail(RPA_E_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  const long long N = s.max_num_seqs, slots = (long long)s.total_pages * s.page_size * s.num_kv_heads;
  const Memory in[] = {{"weights", weights, 4 * slots}, {"positions", positions, 4 * slots}, {"kv_lens", kv_lens, 4 * N},
                       {"page_indices", page_indices, 4 * N * s.pages_per_seq}, {"num_seqs", num_seqs, 4},
                       {"dropped", dropped, 4 * N}, {"workspace", workspace, (long long)plan.bytes}};
  if ((rc = check_separate({"moves", moves, 8 * N * s.num_kv_heads * s.max_moves}, in))) return rc;
  ChooseParams p = {};
  p.weights = weights, p.positions = positions, p.kv_lens = kv_lens, p.table = page_indices, p.num_seqs = num_seqs;
  p.dropped = dropped, p.moves = moves;
  uint8_t* const base = (uint8_t*)workspace;
  p.found = (uint32_t*)base, p.longs = (Long*)(base + plan.longs), p.keys = (uint32_t*)(base + plan.keys);
  p.near = (uint32_t*)(base + plan.near), p.held = (uint32_t*)(base + plan.held), p.counts = (uint32_t*)(base + plan.counts);
  p.tallies = (uint32_t*)(base + plan.tallies);
  p.N = s.max_num_seqs, p.PPS = s.pages_per_seq, p.Hkv = s.num_kv_heads, p.P = s.total_pages, p.S = s.page_size;
  p.budget = s.budget, p.limit = s.limit, p.sinks = s.sinks, p.recent = s.recent, p.M = s.max_moves;
  p.room = plan.room, p.block_room = plan.block_room, p.quads = s.page_size % 4 == 0 && aligned16(weights) && aligned16(positions);
  const unsigned lists = (unsigned)(N * s.num_kv_heads);
  const hipStream_t stream_ = (hipStream_t)stream;
  // a launch of long sequences' blocks: at most 65535 lists
  const auto by_blocks = [&](auto kernel, const char* name) {
    const unsigned step = 65535 / s.num_kv_heads * s.num_kv_heads;
    for (unsigned first = 0; first < lists; first += step) {
      ChooseParams part = p;
      part.first = (int)(first / s.num_kv_heads);
      kernel<<<dim3(plan.blocks, lists - first < step ? lists - first : step), 256, 0, stream_>>>(part);
      if (const int bad = launched(name)) return bad;
    }
    return (int)RPA_OK;
  };
  const size_t lds = (size_t)plan.room * 4;
  if (plan.block_room && (rc = by_blocks(choose_keys_kernel, "choose_moves (keys)"))) return rc;
  if (plan.threads == 256) choose_rows_kernel<256><<<lists, 256, lds, stream_>>>(p);
  else choose_rows_kernel<1024><<<lists, 1024, lds, stream_>>>(p);
  if ((rc = launched("choose_moves")) || !plan.block_room) return rc;
  if ((rc = by_blocks(choose_near_kernel, "choose_moves (near keys)"))) return rc;
  choose_last_kernel<<<lists, 1024, 0, stream_>>>(p);
  if ((rc = launched("choose_moves (digits)")) || (rc = by_blocks(choose_list_kernel<false>, "choose_moves (tallies)"))) return rc;
  return by_blocks(choose_list_kernel<true>, "choose_moves (list)");
}

int rpa_move_rows(const rpa_move_shape_t* shape, const int32_t* moves, const float* kv_scales, void* kv_pages,
                  float* weights, int32_t* positions, void* stream) {
  int rc = check_move(shape);
  if (rc) return rc;
  const rpa_move_shape_t& s = *shape;
  if (s.num_lists == 0) return RPA_OK;
  if (!moves || !kv_pages || !weights || !positions) return fail(RPA_E_INVALID, "NULL tensor pointer");
  const bool fp8 = s.kv_dtype == RPA_KV_FP8_E4M3;
  if (kv_scales && !fp8) return fail(RPA_E_INVALID, "kv_scales requires fp8 kv_pages");
  if (!aligned16(kv_pages)) return fail(RPA_E_INVALID, "kv_pages must be 16-byte aligned");
  const long long entries = (long long)s.num_lists * s.num_kv_heads * s.max_moves, pool = (long long)s.total_pages * s.page_size;
  const long long row = 2ll * s.head_dim * (fp8 ? 1 : 2);
  const Memory in[] = {{"moves", moves, 8 * entries}, {"kv_scales", kv_scales, 8ll * s.total_pages * s.num_kv_heads}};
  const Memory rows = {"kv_pages", kv_pages, pool * s.num_kv_heads * row}, sums = {"weights", weights, 4 * pool * s.num_kv_heads};
  const Memory places = {"positions", positions, 4 * pool * s.num_kv_heads};
  if ((rc = check_separate(rows, in)) || (rc = check_separate(sums, in)) || (rc = check_separate(places, in)) ||
      (rc = check_separate(rows, {sums, places})) || (rc = check_separate(sums, {places})))
    return rc;
  const MoveParams p = {moves, kv_scales, (uint8_t*)kv_pages, weights, positions, pool, (int)entries, s.max_moves, s.num_kv_heads,
                        s.page_size, (int)(row / 16)};
  const unsigned grid = (unsigned)move_groups(entries);
  const auto kernel = fp8 ? (p.chunks <= 16 ? move_kernel<true, 16> : move_kernel<true, 32>)
                          : (p.chunks <= 16 ? move_kernel<false, 16> : p.chunks <= 32 ? move_kernel<false, 32> : move_kernel<false, 64>);
  kernel<<<grid, 256, 0, (hipStream_t)stream>>>(p);
  return launched("move_rows");
}

}  // extern "C"
