// librpa_sparse: the C ABI of include/rpa_sparse.h over its kernels.
#include <float.h>
#include <stdarg.h>
#include <stdio.h>

#include <type_traits>

#include "attend_kernels.h"
#include "page_index.h"
#include "paging_kernels.h"
#include "select_kernels.h"

using namespace rpa_sparse;

extern "C" {

int rpa_sparse_abi_version(void) { return RPA_SPARSE_ABI_VERSION; }

const char* rpa_sparse_last_error(void) { return g_last_error; }

int rpa_sparse_read_error_word(int32_t* host_word, int32_t clear, void* stream) {
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

int rpa_assign_pages(const rpa_paging_shape_t* shape, const int32_t* cached_lens, const int32_t* new_tokens,
                     int32_t* page_table, const int32_t* free_pages, const int32_t* free_count, int32_t* kv_lens,
                     int32_t* cu_q_lens, int32_t* num_seqs, int32_t* slot_mapping, int32_t* positions,
                     int32_t* free_count_out, void* stream) {
  const int rc = check_paging(shape);
  if (rc) return rc;
  if (!cached_lens || !new_tokens || !page_table || !free_count || !kv_lens || !cu_q_lens || !num_seqs ||
      !free_count_out || (shape->free_capacity && !free_pages) ||
      (shape->max_tokens && (!slot_mapping || !positions)))
    return fail(RPA_E_INVALID, "NULL tensor pointer");
  const long long N = shape->num_requests, most = shape->max_tokens;
  const Memory in[] = {{"cached_lens", cached_lens, 4 * N}, {"new_tokens", new_tokens, 4 * N},
                       {"page_table", page_table, 4 * N * shape->pages_per_seq},
                       {"free_pages", free_pages, 4ll * shape->free_capacity}, {"free_count", free_count, 4}};
  const Memory out[] = {{"kv_lens", kv_lens, 4 * N}, {"cu_q_lens", cu_q_lens, 4 * (N + 1)}, {"num_seqs", num_seqs, 4},
                        {"slot_mapping", slot_mapping, 4 * most}, {"positions", positions, 4 * most},
                        {"free_count_out", free_count_out, 4}};
  for (const Memory& o : out) {
    if (const int bad = check_separate(o, in)) return bad;
    for (const Memory* other = out; other != &o; ++other)
      if (meets(*other, o)) return fail(RPA_E_INVALID, "%s overlaps %s: outputs need memory of their own", o.name, other->name);
  }
  const AssignParams p = {cached_lens, new_tokens, page_table, free_pages, free_count, kv_lens, cu_q_lens, num_seqs,
                          slot_mapping, positions, free_count_out, shape->num_requests, shape->pages_per_seq,
                          shape->page_size, shape->free_capacity, shape->max_tokens};
  // small batches take small workgroups: their scans' barriers cost less
  const int threads = shape->num_requests <= kSmallBatch ? 256 : 1024;
  const int grid = shape->max_tokens > 0 ? (shape->max_tokens - 1) / threads + 1 : 1;
  if (threads == 256) assign_kernel<256><<<grid, threads, 0, (hipStream_t)stream>>>(p);
  else assign_kernel<1024><<<grid, threads, 0, (hipStream_t)stream>>>(p);
  return launched("assign_pages");
}

int rpa_release_pages(const rpa_paging_shape_t* shape, const int32_t* cached_lens, const uint8_t* finished,
                      const int32_t* page_table, int32_t* free_pages, const int32_t* free_count,
                      int32_t* cached_lens_out, int32_t* free_count_out, void* stream) {
  const int rc = check_paging(shape);
  if (rc) return rc;
  if (!cached_lens || !finished || !page_table || !free_count || !cached_lens_out || !free_count_out ||
      (shape->free_capacity && !free_pages))
    return fail(RPA_E_INVALID, "NULL tensor pointer");
  const long long N = shape->num_requests;
  const Memory in[] = {{"cached_lens", cached_lens, 4 * N}, {"finished", finished, N},
                       {"page_table", page_table, 4 * N * shape->pages_per_seq},
                       {"free_pages", free_pages, 4ll * shape->free_capacity}, {"free_count", free_count, 4}};
  const Memory lens = {"cached_lens_out", cached_lens_out, 4 * N}, count = {"free_count_out", free_count_out, 4};
  int bad = check_separate(lens, in);
  if (bad || (bad = check_separate(count, in)) || (bad = check_separate(count, {lens}))) return bad;
  const ReleaseParams p = {cached_lens, finished, page_table, free_pages, free_count, cached_lens_out, free_count_out,
                           shape->num_requests, shape->pages_per_seq, shape->page_size, shape->free_capacity};
  const int grid = (shape->num_requests - 1) / kReleaseSlice + 1;
  if (const int many = check_launch(grid, kReleaseThreads)) return many;
  release_kernel<<<grid, kReleaseThreads, 0, (hipStream_t)stream>>>(p);
  return launched("release_pages");
}

int rpa_append_kv(const rpa_append_shape_t* shape, const void* keys, const void* values, const int32_t* slot_mapping,
                  void* kv_pages, const float* kv_scales, float k_scale, float v_scale, int8_t* bounds,
                  int8_t* exponents, void* stream) {
  int rc = check_append(shape);
  if (rc) return rc;
  if (shape->num_tokens == 0) return RPA_OK;
  if (!keys || !values || !slot_mapping || !kv_pages || !bounds != !exponents)
    return fail(RPA_E_INVALID, "NULL tensor pointer");
  if ((rc = check_strides("keys", keys, shape->k_token_stride, shape->k_head_stride))) return rc;
  if ((rc = check_strides("values", values, shape->v_token_stride, shape->v_head_stride))) return rc;
  if (!aligned16(kv_pages) || !aligned16(bounds)) return fail(RPA_E_INVALID, "kv_pages and bounds must be 16-byte aligned");
  const auto usable = [](float x) { return x > 0.f && x <= FLT_MAX; };
  if (shape->kv_dtype == RPA_KV_FP8_E4M3 && !kv_scales && !(usable(k_scale) && usable(v_scale)))
    return fail(RPA_E_INVALID, "k_scale and v_scale must be positive and finite");
  const int chunks = shape->head_dim / 8, tokens = shape->num_tokens > kAppendLong ? kAppendTokens : 1;
  const int ahead = 64 / chunks * (tokens > 1 ? kAppendRounds : 1);  // tokens of a workgroup that widens bounds
  const int wide = bounds ? (shape->num_tokens - 1) / ahead + 1 : 0;
  const AppendParams p = {(const uint16_t*)keys, (const uint16_t*)values, slot_mapping, (uint8_t*)kv_pages, kv_scales, k_scale,
                          v_scale, bounds, exponents, shape->k_token_stride, shape->k_head_stride, shape->v_token_stride,
                          shape->v_head_stride, (long long)shape->total_pages * shape->page_size, shape->num_tokens,
                          shape->num_kv_heads, shape->head_dim, shape->page_size, wide,
                          (uint32_t)(0x100000000ull / chunks + 1), (uint32_t)(0x100000000ull / (2 * chunks) + 1)};
  const int threads = 64 * (shape->num_kv_heads < 8 ? shape->num_kv_heads : 8);
  const int grid = wide + (shape->num_tokens - 1) / tokens + 1;
  if ((rc = check_launch(grid, threads))) return rc;
  const auto kernel = shape->kv_dtype == RPA_KV_FP8_E4M3
                          ? (tokens > 1 ? append_kernel<true, kAppendTokens> : append_kernel<true, 1>)
                          : (tokens > 1 ? append_kernel<false, kAppendTokens> : append_kernel<false, 1>);
  kernel<<<grid, threads, 0, (hipStream_t)stream>>>(p);
  return launched("append_kv");
}

size_t rpa_select_workspace_size(const rpa_sparse_shape_t* shape) {
  return check_sparse(shape) == RPA_OK ? plan_select(*shape).bytes : 0;
}

int rpa_select_pages(const rpa_sparse_shape_t* shape, int32_t sink_pages, int32_t recent_pages, const void* q,
                     const int8_t* bounds, const int8_t* exponents, const int32_t* kv_lens,
                     const int32_t* page_indices, const int32_t* cu_q_lens, const int32_t* num_seqs,
                     int32_t* selected_pages, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_sparse(shape);
  if (rc) return rc;
  if (sink_pages < 0 || recent_pages < 0 || (long long)sink_pages + recent_pages > shape->num_pages)
    return fail(RPA_E_INVALID, "sink_pages and recent_pages must not be negative nor more than num_pages together");
  if (shape->num_tokens == 0) return RPA_OK;
  if (!q || !bounds || !exponents || !kv_lens || !page_indices || !cu_q_lens || !num_seqs || !selected_pages)
    return fail(RPA_E_INVALID, "NULL tensor pointer");
  if ((rc = check_strides("q", q, shape->q_token_stride, shape->q_head_stride))) return rc;
  if (!aligned16(bounds)) return fail(RPA_E_INVALID, "bounds must be 16-byte aligned");
  const SelectPlan plan = plan_select(*shape);
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace)))
    return fail(RPA_E_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  const long long T = shape->num_tokens, Hkv = shape->num_kv_heads, D = shape->head_dim, N = shape->max_num_seqs;
  const Memory in[] = {rows_of("q", q, T, shape->num_q_heads, D, shape->q_token_stride, shape->q_head_stride),
                       {"bounds", bounds, shape->total_pages * Hkv * 2 * D}, {"exponents", exponents, shape->total_pages * Hkv},
                       {"kv_lens", kv_lens, 4 * N}, {"page_indices", page_indices, 4 * N * shape->pages_per_seq},
                       {"cu_q_lens", cu_q_lens, 4 * (N + 1)}, {"num_seqs", num_seqs, 4},
                       {"workspace", workspace, (long long)plan.bytes}};
  if ((rc = check_separate({"selected_pages", selected_pages, 4 * T * Hkv * shape->num_pages}, in))) return rc;
  const SelectParams p = {(const uint16_t*)q, bounds, exponents, kv_lens, page_indices, cu_q_lens, num_seqs, selected_pages,
                          (uint32_t*)workspace, shape->q_token_stride, shape->q_head_stride, shape->num_tokens,
                          shape->num_kv_heads, shape->num_q_heads / shape->num_kv_heads, shape->head_dim,
                          shape->total_pages, shape->page_size, shape->max_num_seqs, shape->pages_per_seq,
                          shape->num_pages, sink_pages, recent_pages, plan.gp, plan.gp == 4 ? 2 : plan.gp == 8 ? 3 : 4, plan.tokens, plan.stride, 0,
                          (uint32_t)(0x100000000ull / (shape->head_dim / 8) + 1)};
  const hipStream_t s = (hipStream_t)stream;
  return plan.steps == 2 ? launch_select<2>(plan, p, s) : plan.steps == 4 ? launch_select<4>(plan, p, s)
                                                                          : launch_select<8>(plan, p, s);
}

size_t rpa_sparse_workspace_size(const rpa_sparse_shape_t* shape) {
  return check_attend(shape) == RPA_OK ? plan_attend(*shape).bytes : 0;
}

int rpa_sparse_paged_attention(const rpa_sparse_shape_t* shape, const rpa_sparse_options_t* options, const void* q,
                               const void* kv_pages, const float* kv_scales, const int32_t* selected_pages,
                               const int32_t* kv_lens, const int32_t* page_indices, const int32_t* cu_q_lens,
                               const int32_t* num_seqs, void* out, void* workspace, size_t workspace_bytes,
                               void* stream) {
  int rc = check_attend(shape);
  if (rc) return rc;
  if (!options) return fail(RPA_E_INVALID, "options is NULL");
  if (shape->num_tokens == 0) return RPA_OK;
  if (!q || !kv_pages || !selected_pages || !kv_lens || !page_indices || !cu_q_lens || !num_seqs || !out)
    return fail(RPA_E_INVALID, "NULL tensor pointer");
  const bool fp8 = shape->kv_dtype == RPA_KV_FP8_E4M3;
  if (kv_scales && !fp8) return fail(RPA_E_INVALID, "kv_scales requires fp8 kv_pages");
  if ((rc = check_strides("q", q, shape->q_token_stride, shape->q_head_stride))) return rc;
  if (!aligned16(kv_pages) || !aligned16(out)) return fail(RPA_E_INVALID, "kv_pages and out must be 16-byte aligned");
  const AttendPlan plan = plan_attend(*shape);
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace)))
    return fail(RPA_E_WORKSPACE, "workspace missing, too small or not 16-byte aligned");
  const long long T = shape->num_tokens, Hq = shape->num_q_heads, Hkv = shape->num_kv_heads, D = shape->head_dim;
  const long long N = shape->max_num_seqs, pool = (long long)shape->total_pages * shape->page_size;
  const Memory in[] = {rows_of("q", q, T, Hq, D, shape->q_token_stride, shape->q_head_stride),
                       {"kv_pages", kv_pages, pool * 2 * Hkv * D * (fp8 ? 1 : 2)},
                       {"kv_scales", kv_scales, 8 * shape->total_pages * Hkv},
                       {"selected_pages", selected_pages, 4 * T * Hkv * shape->num_pages}, {"kv_lens", kv_lens, 4 * N},
                       {"page_indices", page_indices, 4 * N * shape->pages_per_seq}, {"cu_q_lens", cu_q_lens, 4 * (N + 1)},
                       {"num_seqs", num_seqs, 4}, {"workspace", workspace, (long long)plan.bytes}};
  if ((rc = check_separate({"out", out, 2 * T * Hq * D}, in))) return rc;
  if ((rc = check_launch(plan.chunk ? plan.grid : plan.rows, plan.chunk ? 256 * plan.groups : 64 * kAttendWaves)) ||
      (plan.splits > 1 && (rc = check_launch(plan.rows, 256))))
    return rc;
  const float cap = options->soft_cap < 0.f ? -options->soft_cap : options->soft_cap;
  AttendParams p = {};
  p.q = (const uint16_t*)q, p.kv = (const uint8_t*)kv_pages, p.scales = kv_scales;
  p.picked = selected_pages, p.kv_lens = kv_lens, p.table = page_indices, p.cu = cu_q_lens, p.num_seqs = num_seqs;
  p.out = (uint16_t*)out, p.parts = (float*)workspace;
  p.q_token = shape->q_token_stride, p.q_head = shape->q_head_stride;
  p.T = shape->num_tokens, p.Hkv = shape->num_kv_heads, p.G = shape->num_q_heads / shape->num_kv_heads;
  p.D = shape->head_dim, p.P = shape->total_pages, p.S = shape->page_size, p.N = shape->max_num_seqs;
  p.PPS = shape->pages_per_seq, p.K = shape->num_pages;
  p.tiles = plan.tiles, p.width = plan.width, p.subs = plan.subs, p.blocks = (int)plan.blocks;
  p.magic = plan.width > 1 ? (uint32_t)((0x100000000ull + plan.width - 1) / plan.width) : 0;
  p.per = plan.per, p.splits = plan.splits;
  p.scale = options->sm_scale * options->k_scale * (cap != 0.f ? 1.f : kLog2e), p.cap = cap;
  p.v_scale = options->v_scale;
  const hipStream_t s = (hipStream_t)stream;
  if (fp8) {
    if (D == 256) launch_attend<256, true, true>(plan, p, s);
    else if (D == 128) launch_attend<128, true, true>(plan, p, s);
    else if (D == 64) launch_attend<64, true, true>(plan, p, s);
    else launch_attend<128, false, true>(plan, p, s);
  } else {
    if (D == 256) launch_attend<256, true, false>(plan, p, s);
    else if (D == 128) launch_attend<128, true, false>(plan, p, s);
    else if (D == 64) launch_attend<64, true, false>(plan, p, s);
    else if (D < 64) launch_attend<64, false, false>(plan, p, s);
    else launch_attend<128, false, false>(plan, p, s);
  }
  if ((rc = launched("sparse_paged_attention"))) return rc;
  if (plan.splits > 1) {
    join_kernel<<<(unsigned)plan.rows, 256, 0, s>>>(p);
    return launched("sparse_paged_attention (join)");
  }
  return RPA_OK;
}

}  // extern "C"
