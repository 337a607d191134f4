/*
 * librpa_sparse -- page allocation, K/V append and sparse paged attention for AMD Instinct MI355X
 * (gfx950), beside the operator of rpa.h: the same pool layout, the same metadata tensors.
 *
 * C ABI as in rpa.h: plain pointers and sizes, DEVICE pointers owned by the caller, no allocation
 * on the call path, stream-ordered, 0 or a negative RPA_E* code with a thread-local message
 * (rpa_sparse_last_error).  No entry point throws.  All of them may be captured into a graph: they
 * record kernel launches only.
 *
 * Out-of-range metadata (page ids, slots, lengths) is never dereferenced; the kernels set a bit of
 * the device's error word for it (rpa_sparse_read_error_word).
 * Offsets (cu_q_lens) that decrease or lie outside [0, num_tokens] set none: the calls stay within
 * their tensors, and which rows get a result is not defined.
 */
#ifndef RPA_SPARSE_H_
#define RPA_SPARSE_H_

#include <stddef.h>
#include <stdint.h>

#include "rpa.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RPA_SPARSE_ABI_VERSION 1

/* Bits of the error word. */
enum {
  RPA_SPARSE_ERR_PAGE = 1,  /* a page id outside the pool */
  RPA_SPARSE_ERR_SLOT = 2,  /* a slot outside the pool (not -1, which means: no row) */
  RPA_SPARSE_ERR_LEN = 4,   /* a length past the page table; given to the paging calls, also a negative one */
  RPA_SPARSE_ERR_FREE = 8   /* the free stack's count or capacity exceeded */
};

int rpa_sparse_abi_version(void);
const char* rpa_sparse_last_error(void);

/* The current device's error word: the bits of every call since they were last cleared.  Waits for
 * the stream; `clear` != 0 takes back the bits it returns, and no others that calls on other streams
 * set meanwhile. */
int rpa_sparse_read_error_word(int32_t* host_word, int32_t clear, void* stream);

/* ---- page allocation -------------------------------------------------------------------------
 * The pool's free pages are a stack: free_pages[0 .. free_count).  A request holds the first
 * ceil(len / page_size) entries of its page_table row. */
typedef struct rpa_paging_shape {
  int32_t num_requests;  /* N = page_table.shape[0], at most 2^31 - 2^16 - 1 */
  int32_t pages_per_seq; /* PPS = page_table.shape[1], at most 2^31 - 2^16 - 1 */
  int32_t page_size;     /* S */
  int32_t free_capacity; /* F = free_pages.shape[0], below 2^30 */
  int32_t max_tokens;    /* rows of slot_mapping and positions, below 2^30 */
} rpa_paging_shape_t;

/* Gives every request the pages of its new tokens and writes the step's metadata.
 *   cached_lens, new_tokens int32 [N]; page_table int32 [N, PPS] (new entries written);
 *   free_pages int32 [F], free_count int32 [1] (read)
 *   kv_lens int32 [N]; cu_q_lens int32 [N + 1]; num_seqs int32 [1] (= N); slot_mapping, positions
 *   int32 [max_tokens] (-1 and 0 past the last token); free_count_out int32 [1]
 * A request is admitted if its lengths are not negative and fit the table, the batch's tokens up to
 * and including its own are at most max_tokens, and it needs no page or the pages needed up to and
 * including its own are at most free_count; both sums run over all requests with valid lengths.
 * One that is not admitted keeps its length and gets no token.  The outputs must not overlap the
 * inputs. */
int rpa_assign_pages(const rpa_paging_shape_t* shape, const int32_t* cached_lens, const int32_t* new_tokens,
                     int32_t* page_table, const int32_t* free_pages, const int32_t* free_count, int32_t* kv_lens,
                     int32_t* cu_q_lens, int32_t* num_seqs, int32_t* slot_mapping, int32_t* positions,
                     int32_t* free_count_out, void* stream);

/* Pushes the pages of finished requests (finished uint8 [N], nonzero = finished) on the free stack,
 * in order, and sets their lengths to 0 in cached_lens_out.  max_tokens of the shape is ignored. */
int rpa_release_pages(const rpa_paging_shape_t* shape, const int32_t* cached_lens, const uint8_t* finished,
                      const int32_t* page_table, int32_t* free_pages, const int32_t* free_count,
                      int32_t* cached_lens_out, int32_t* free_count_out, void* stream);

/* ---- K/V append and the page index ------------------------------------------------------------
 * The page index of a pool: bounds int8 [total_pages, num_kv_heads, 2, head_dim] (of every dimension
 * the largest, then the smallest value of the page's keys) and exponents int8 [total_pages,
 * num_kv_heads]: a bound b stands for b * 2^exponent.  exponent is the smallest whole number in
 * [-100, 100] with 127 * 2^exponent >= the largest magnitude of the page's keys; the largest values
 * are rounded up to that grid and the smallest down, clamped to [-127, 127]; NaN counts as 0.  Keys of
 * an fp8 pool are code * K scale. */
typedef struct rpa_append_shape {
  int32_t num_tokens;  /* below 2^30 */
  int32_t num_kv_heads; /* at most 65535 */
  int32_t head_dim;    /* as rpa_shape_t: 256, or a multiple of 8 in [32, 128] (fp8: of 16 in [64, 128]) */
  int32_t total_pages;
  int32_t page_size;
  int32_t kv_dtype;    /* RPA_KV_BF16 | RPA_KV_FP8_E4M3 */
  int64_t k_token_stride, k_head_stride; /* of keys [num_tokens, num_kv_heads, head_dim], in values */
  int64_t v_token_stride, v_head_stride;
} rpa_append_shape_t;

/* Writes token t's key and value rows (bf16) to row slot_mapping[t] % page_size of page
 * slot_mapping[t] / page_size of kv_pages (rpa.h's layout); -1: no row.  fp8 pools hold
 * e4m3(x / scale), saturated, with the scale of the row's page and head in kv_scales (float
 * [total_pages, num_kv_heads, 2]) or, where that is NULL, k_scale and v_scale, positive and finite
 * (ignored for bf16).
 * keys and values must not lie in the rows that are written.
 * bounds and exponents: the pool's index, or both NULL.  A page whose row 0 is written starts its
 * bounds anew, other pages' widen.  The slots (other than -1) have to differ, and the new rows of one
 * page have to be consecutive tokens at consecutive slots. */
int rpa_append_kv(const rpa_append_shape_t* shape, const void* keys, const void* values, const int32_t* slot_mapping,
                  void* kv_pages, const float* kv_scales, float k_scale, float v_scale, int8_t* bounds,
                  int8_t* exponents, void* stream);

/* ---- sparse attention over chosen pages -------------------------------------------------------
 * q, kv_lens, page_indices, cu_q_lens, num_seqs as in rpa.h: token t of sequence i stands at position
 * kv_lens[i] - (cu_q_lens[i + 1] - t) and sees the keys up to there. */
typedef struct rpa_sparse_shape {
  int32_t num_tokens, num_q_heads, num_kv_heads, head_dim;
  int32_t total_pages, page_size, max_num_seqs;
  int32_t pages_per_seq; /* at most 2^31 - 2^16 - 1, as num_pages */
  int32_t kv_dtype;  /* of the pool; ignored by rpa_select_pages apart from its head dims */
  int32_t num_pages; /* entries of a row of the list */
  int64_t q_token_stride, q_head_stride; /* of q [num_tokens, num_q_heads, head_dim], in values */
} rpa_sparse_shape_t;

/* For each token and kv head the logical pages (indices into its sequence's page table row) whose
 * keys are estimated to score highest, ascending, -1 past the last: int32 [num_tokens, num_kv_heads, num_pages], apart
 * from the inputs.
 * A token sees the pages 0 .. position / page_size.  The first `sink_pages` and the last
 * `recent_pages` of them are always chosen (sink_pages + recent_pages <= num_pages), the others by
 *   score(p) = 2^exponent(p) * max over the group's heads g of sum_d max(qh_gd hi_d, qh_gd lo_d)
 * with the index's integer bounds and qh = q / 2^f rounded to nearest even and clamped to
 * [-127, 127], f as an index exponent over the group's queries (NaN counts as 0); the highest first, of
 * equal scores the earlier page.  Tokens past cu_q_lens[num_seqs] get no page. */
size_t rpa_select_workspace_size(const rpa_sparse_shape_t* shape);
int rpa_select_pages(const rpa_sparse_shape_t* shape, int32_t sink_pages, int32_t recent_pages, const void* q,
                     const int8_t* bounds, const int8_t* exponents, const int32_t* kv_lens,
                     const int32_t* page_indices, const int32_t* cu_q_lens, const int32_t* num_seqs,
                     int32_t* selected_pages, void* workspace, size_t workspace_bytes, void* stream);

typedef struct rpa_sparse_options {
  float sm_scale;
  float soft_cap;         /* 0: none; else scores become soft_cap * tanh(score / soft_cap) */
  float k_scale, v_scale; /* of the whole pool; 1 where kv_scales is given */
} rpa_sparse_options_t;

/* Attention of each token and head over the keys, up to the token's position, of the pages listed for
 * its kv head: selected_pages int32 [num_tokens, num_kv_heads, num_pages], logical pages in any order,
 * entries outside the token's pages (-1) list nothing, a page listed twice counts twice.  Keys and values
 * of an fp8 pool are code * scale, not rounded; kv_scales as in rpa.h or NULL.
 * out bf16 [num_tokens, num_q_heads, head_dim], contiguous, apart from the inputs; rows without a key or without a score
 * above -infinity, and rows at or past cu_q_lens[num_seqs], are zero. */
size_t rpa_sparse_workspace_size(const rpa_sparse_shape_t* shape);
int rpa_sparse_paged_attention(const rpa_sparse_shape_t* shape, const rpa_sparse_options_t* options, const void* q,
                               const void* kv_pages, const float* kv_scales, const int32_t* selected_pages,
                               const int32_t* kv_lens, const int32_t* page_indices, const int32_t* cu_q_lens,
                               const int32_t* num_seqs, void* out, void* workspace, size_t workspace_bytes,
                               void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RPA_SPARSE_H_ */
