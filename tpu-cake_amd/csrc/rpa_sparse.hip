// librpa_sparse: the C ABI of include/rpa_sparse.h over its kernels.
#include <stdarg.h>
#include <stdio.h>

#include "paging_kernels.h"

using namespace rpa_sparse;

extern "C" {

int rpa_sparse_abi_version(void) { return RPA_SPARSE_ABI_VERSION; }

const char* rpa_sparse_last_error(void) { return g_last_error; }

int rpa_sparse_read_error_word(int32_t* host_word, int32_t clear, void* stream) {
  if (!host_word) return fail(RPA_E_INVALID, "host_word is NULL");
  const hipStream_t s = (hipStream_t)stream;
  const int32_t zero = 0;
  if (hipMemcpyFromSymbolAsync(host_word, HIP_SYMBOL(g_error_word), sizeof(int32_t), 0, hipMemcpyDeviceToHost, s) !=
          hipSuccess ||
      hipStreamSynchronize(s) != hipSuccess)
    return fail(RPA_E_HIP, "reading the error word failed");
  if (clear && (hipMemcpyToSymbolAsync(HIP_SYMBOL(g_error_word), &zero, sizeof zero, 0, hipMemcpyHostToDevice, s) !=
                    hipSuccess ||
                hipStreamSynchronize(s) != hipSuccess))
    return fail(RPA_E_HIP, "clearing the error word failed");
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
  if (kv_lens == cached_lens || kv_lens == new_tokens || free_count_out == free_count)
    return fail(RPA_E_INVALID, "outputs must not overlap the inputs");
  const AssignParams p = {cached_lens, new_tokens, page_table, free_pages, free_count, kv_lens, cu_q_lens, num_seqs,
                          slot_mapping, positions, free_count_out, shape->num_requests, shape->pages_per_seq,
                          shape->page_size, shape->free_capacity, shape->max_tokens};
  constexpr int kThreads = 1024;
  const int grid = shape->max_tokens > 0 ? (shape->max_tokens + kThreads - 1) / kThreads : 1;
  assign_kernel<kThreads><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
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
  if (cached_lens_out == cached_lens || free_count_out == free_count)
    return fail(RPA_E_INVALID, "outputs must not overlap the inputs");
  const ReleaseParams p = {cached_lens, finished, page_table, free_pages, free_count, cached_lens_out, free_count_out,
                           shape->num_requests, shape->pages_per_seq, shape->page_size, shape->free_capacity};
  const int grid = (shape->num_requests - 1) / kReleaseSlice + 1;
  release_kernel<<<grid, kReleaseThreads, 0, (hipStream_t)stream>>>(p);
  return launched("release_pages");
}

}  // extern "C"
