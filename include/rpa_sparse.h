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
  RPA_SPARSE_ERR_LEN = 4,   /* a negative length, or one past the page table */
  RPA_SPARSE_ERR_FREE = 8   /* the free stack's count or capacity exceeded */
};

int rpa_sparse_abi_version(void);
const char* rpa_sparse_last_error(void);

/* The current device's error word: the bits of every call since it was last cleared.  Waits for
 * the stream; `clear` != 0 sets it to 0 afterwards. */
int rpa_sparse_read_error_word(int32_t* host_word, int32_t clear, void* stream);

/* ---- page allocation -------------------------------------------------------------------------
 * The pool's free pages are a stack: free_pages[0 .. free_count).  A request holds the first
 * ceil(len / page_size) entries of its page_table row. */
typedef struct rpa_paging_shape {
  int32_t num_requests;  /* N = page_table.shape[0] */
  int32_t pages_per_seq; /* PPS = page_table.shape[1] */
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

#ifdef __cplusplus
}
#endif
#endif /* RPA_SPARSE_H_ */
