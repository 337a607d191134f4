/*
 * librpa_bounded -- a step of serving with a bounded cache for AMD Instinct MI355X (gfx950), beside
 * rpa.h and rpa_sparse.h and over their tensors: norms and position rotation of a step's queries and
 * keys, attention that accounts for the weight each cached key got, the choice of the keys that go
 * when a sequence outgrows its budget, and the moves that close the gaps.
 *
 * C ABI as in rpa_sparse.h: plain pointers and sizes, DEVICE pointers owned by the caller, no
 * allocation on the call path, stream-ordered, 0 or a negative RPA_E* code with a thread-local message
 * (rpa_bounded_last_error).  No entry point throws.  All of them may be captured into a graph: they
 * record kernel launches only.
 *
 * Out-of-range metadata (page ids, slots, lengths) is never dereferenced; the kernels set a bit of
 * the device's error word for it (rpa_bounded_read_error_word, RPA_SPARSE_ERR_*).
 * Offsets (cu_q_lens) that decrease or lie outside [0, num_tokens] set none: the calls stay within
 * their tensors, and which rows get a result is not defined.
 */
#ifndef RPA_BOUNDED_H_
#define RPA_BOUNDED_H_

#include <stddef.h>
#include <stdint.h>

#include "rpa_sparse.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RPA_BOUNDED_ABI_VERSION 1

int rpa_bounded_abi_version(void);
const char* rpa_bounded_last_error(void);

/* The current device's error word of this library's calls: as rpa_sparse_read_error_word. */
int rpa_bounded_read_error_word(int32_t* host_word, int32_t clear, void* stream);

/* ---- norms and position rotation of queries and keys -----------------------------------------------
 * For each token t and head: x' = w x / sqrt(mean(x^2) + eps) where a weight is given, else x; then the
 * first `rotated` dims as `rotated / 2` pairs, (x_i, x_{i + rotated/2}) or, interleaved, (x_2i, x_{2i+1}),
 * each turned by turns_i * (positions[t] + dropped[sequence of t]) / 2^64 of a full turn and multiplied
 * by `magnitude`.  The other dims are not turned.  All in fp32, rounded once. */
typedef struct rpa_rotate_shape {
  int32_t num_tokens; /* below 2^30 */
  int32_t num_q_heads, num_kv_heads;
  int32_t head_dim;    /* 256, or a multiple of 8 in [32, 128] */
  int32_t rotated;     /* in [0, head_dim]; a multiple of 8, interleaved: of 2 */
  int32_t interleaved; /* 0 or 1 */
  int32_t max_num_seqs; /* of cu_q_lens and dropped; ignored without them */
  int32_t weight_bytes; /* of a weight's values: 2 (bf16) or 4 (float) */
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride; /* of q and k, in values */
  int64_t q_out_token_stride, q_out_head_stride, k_out_token_stride, k_out_head_stride;
  int64_t q_weight_stride, k_weight_stride; /* from one head's weight to the next; 0: all heads' */
} rpa_rotate_shape_t;

/* q [num_tokens, num_q_heads, head_dim] and k [num_tokens, num_kv_heads, head_dim] bf16, rows 16-byte
 * aligned, as q_out and k_out; positions int32 [num_tokens]; turns uint64 [rotated / 2]; q_weight,
 * k_weight: NULL, or [head_dim] for each head.
 * cu_q_lens int32 [max_num_seqs + 1] with num_seqs int32 [1]: NULL, or as in rpa.h; dropped int32
 * [max_num_seqs]: NULL, or (with cu_q_lens) how many earlier tokens of each sequence its cache has lost.
 * q_out and k_out: q and k themselves with the same strides (in place), or memory of their own.  Rows at or
 * past cu_q_lens[num_seqs] are left as they are in place, and zero otherwise. */
int rpa_rotate_heads(const rpa_rotate_shape_t* shape, float eps, float magnitude, const void* q, const void* k,
                     const int32_t* positions, const uint64_t* turns, const void* q_weight, const void* k_weight,
                     const int32_t* cu_q_lens, const int32_t* num_seqs, const int32_t* dropped, void* q_out,
                     void* k_out, void* stream);

/* ---- attention that accounts for the weight of each key -------------------------------------------
 * The ledger of a pool: weights float [total_pages, num_kv_heads, page_size] and positions int32 of the
 * same shape: for each slot and kv head what the key there got, and where its token stood. */
typedef struct rpa_weigh_shape {
  int32_t num_tokens, num_q_heads, num_kv_heads, head_dim;
  int32_t total_pages, page_size, max_num_seqs, pages_per_seq;
  int32_t kv_dtype; /* RPA_KV_BF16 | RPA_KV_FP8_E4M3 */
  int32_t reserved;
  int64_t q_token_stride, q_head_stride; /* of q, in values */
} rpa_weigh_shape_t;

typedef struct rpa_weigh_options {
  float sm_scale;
  float soft_cap;         /* 0: none; else scores become soft_cap * tanh(score / soft_cap) */
  float k_scale, v_scale; /* of the whole pool; 1 where kv_scales is given */
  float decay;            /* what is left of a key's earlier weight; 0: it is not read */
} rpa_weigh_options_t;

/* Causal attention of each token over its sequence's keys, as rpa_ragged_paged_attention; out bf16
 * [num_tokens, num_q_heads, head_dim], contiguous; rows without a key or without a score above
 * -infinity, and rows at or past cu_q_lens[num_seqs], are zero.  And for each sequence with tokens, of every key
 * and kv head:  weights = decay * weights + the probabilities that the step's tokens and the group's heads
 * gave the key.  The last q_len keys of a sequence are new: their weight starts at 0 and their
 * position is dropped[sequence] (NULL: 0) + the key's row.  The sequences' pages have to differ.
 * Memory of a call's outputs must not overlap its inputs. */
size_t rpa_weigh_workspace_size(const rpa_weigh_shape_t* shape);
int rpa_weighed_attention(const rpa_weigh_shape_t* shape, const rpa_weigh_options_t* options, const void* q,
                          const void* kv_pages, const float* kv_scales, const int32_t* kv_lens,
                          const int32_t* page_indices, const int32_t* cu_q_lens, const int32_t* num_seqs,
                          const int32_t* dropped, float* weights, int32_t* positions, void* out, void* workspace,
                          size_t workspace_bytes, void* stream);

/* ---- eviction -------------------------------------------------------------------------------------- */
typedef struct rpa_choose_shape {
  int32_t max_num_seqs, pages_per_seq, num_kv_heads, total_pages, page_size;
  int32_t budget;        /* rows a sequence keeps, at least 1 */
  int32_t limit;         /* sequences longer than this are cut; at least budget */
  int32_t sinks, recent; /* kept in any case: positions below sinks, and the last `recent`; together at most budget */
  int32_t max_moves;     /* entries of a list */
} rpa_choose_shape_t;

/* For each sequence of more than `limit` keys and each kv head the `budget` rows to keep: those at
 * positions below `sinks` or in the last `recent` of kv_lens + dropped, then those of the highest weight
 * (NaN below all others); of equal ones, and of too many of the former, the lower rows.  The i-th kept row at or past `budget` goes to the i-th
 * row below it that is not kept: moves int32 [max_num_seqs, num_kv_heads, max_moves, 2] holds the two
 * slots (page * page_size + row), to and from, and -1 past the last.  A list that needs more than max_moves
 * entries (never with max_moves >= budget) is cut short and sets RPA_SPARSE_ERR_LEN. */
size_t rpa_choose_workspace_size(const rpa_choose_shape_t* shape);
int rpa_choose_moves(const rpa_choose_shape_t* shape, const float* weights, const int32_t* positions,
                     const int32_t* kv_lens, const int32_t* page_indices, const int32_t* num_seqs,
                     const int32_t* dropped, int32_t* moves, void* workspace, size_t workspace_bytes, void* stream);

typedef struct rpa_move_shape {
  int32_t num_lists; /* sequences of the lists */
  int32_t max_moves; /* entries of a list */
  int32_t num_kv_heads, head_dim, total_pages, page_size;
  int32_t kv_dtype;
} rpa_move_shape_t;

/* Copies, for each entry of moves int32 [num_lists, num_kv_heads, max_moves, 2], the head's key and value rows
 * and its ledger entries from slot [1] to slot [0]; negative slots: none.  No slot that is written may be another
 * entry's.  Rows of an fp8 pool that change their scale (kv_scales) are rounded anew: e4m3(code * scale there
 * / scale here), saturated. */
int rpa_move_rows(const rpa_move_shape_t* shape, const int32_t* moves, const float* kv_scales, void* kv_pages,
                  float* weights, int32_t* positions, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RPA_BOUNDED_H_ */
