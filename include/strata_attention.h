/*
 * strata_attention.h — what an attention layer does between its projections,
 * and the scoring of tokens behind the head projection, on device buffers:
 *
 *   kv_append   a call's new keys and values into a paged cache, rotated by
 *               their positions on the way, and the rotated queries
 *   attention   the new tokens' queries over that cache (single tokens when
 *               decoding, chunks of a prompt), causal, optionally within a
 *               sliding window and with first tokens that stay visible
 *   logprobs    the log-probability of a given token of every row of logits,
 *               the row's entropy and its likeliest tokens
 *
 * The reference runs these steps on the host (crates/strata-core/src/qsa.rs).
 * Status codes, contexts, streams and strata_cuda_last_error are
 * strata_cuda.h's; sequences (seq_len or seq_offsets, empty ones among them),
 * capturing and concurrent calls are as strata_sequence.h describes them. The
 * calls allocate nothing and keep nothing between calls.
 */
#ifndef STRATA_ATTENTION_H
#define STRATA_ATTENTION_H

#include "strata_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------ the cache */

/* A paged cache of one layer's keys and values, bf16. Page g holds page_size
 * tokens; the key (or value) of token row i and head h of a page lies at
 *   g * page_stride + i * token_stride + h * head_stride
 * elements from k_dev (v_dev), head_dim elements side by side. Strides of 0 are
 * packed: [page][token][head][dim]; heads may also be outside the tokens, and
 * both pools may be interleaved. Buffers are 16-byte aligned, strides multiples
 * of 8 elements, head_dim a multiple of 8 (8 to 256), page_size a multiple of 16.
 *
 * Sequence i has its pages in row i of the table (device memory, read when the
 * kernels run, so a captured call follows a table that changes): position p
 * lies in page table[i * table_stride + p / page_size], row p mod page_size.
 * len_dev[i] is the number of its tokens in the cache, those of the call
 * included: a sequence of n new tokens has them at positions len - n to
 * len - 1. A position that is negative, or behind the table's max_pages pages,
 * or whose page is outside [0, n_pages) (-1, say, for pages that were given
 * back) has no place: appending there does nothing, and no query sees it.
 * max_pages * page_size stays below 2^31. */
typedef struct {
    void *k_dev;
    void *v_dev;
    const int32_t *table_dev;
    const int32_t *len_dev;
    int64_t n_pages, page_size, n_kv_head, head_dim;
    int64_t page_stride, token_stride, head_stride; /* elements; 0 = packed */
    int64_t max_pages;                              /* entries of a row of the table */
    int64_t table_stride;                           /* from row to row; 0 = max_pages */
} strata_kv_cache;

/* --------------------------------------------------------------- append */

/* For every token of the call, at position p: its keys, rotated, and its values
 * go to their place in the cache (rounded to bf16, nearest even), its queries,
 * rotated, to q_out. The rotation turns each pair (a, b) of the first n_rot
 * elements of a head by the angle p * freq_base^(-2 i / n_rot):
 *   a' = a cos - b sin,  b' = a sin + b cos
 * where pair i is (i, i + n_rot / 2), or (2 i, 2 i + 1) where `neighbours` is
 * set; the other elements stay (n_rot 0: all). Angles are f64, sines and
 * cosines good to 2^-23 at positions below 2^26 with bases of 1 and above (at the
 * farthest, 2^31, an angle's own 53 bits leave 2^-21; bases below 1 turn faster
 * and lose more), products f32, each result rounded once.
 * Buffers of 16-byte alignment, strides of whole 16 bytes and an n_rot that is a
 * multiple of 8 are read in packs, others element by element (three times slower).
 * q, k and v are dtype (STRATA_QUANT_F32 or STRATA_QUANT_BF16), token rows of
 * heads side by side `*_stride` elements apart (0 = packed), so they may be
 * columns of one projection's output; q_out is q_dtype and may be q itself
 * (same type and stride) where nothing else overlaps. n_head 0: there are no
 * queries, and q and q_out may be NULL. Queries of tokens without a place are
 * rotated all the same (a negative position counts as it is). No two tokens of
 * a call may have the same place, and no key's row may share elements with a
 * value's (pools that do are refused). */
typedef struct {
    int64_t n_seq;
    int64_t seq_len;            /* tokens of every sequence when seq_offsets is NULL */
    const int64_t *seq_offsets; /* host memory, n_seq + 1 row numbers, or NULL */
    int64_t n_head, n_rot;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    double freq_base;
    uint32_t dtype, q_dtype;
    int neighbours;
} strata_kv_append;

int strata_cuda_kv_append_dev(strata_ctx *ctx, const strata_kv_append *desc, const strata_kv_cache *cache,
                              const void *q_dev, const void *k_dev, const void *v_dev, void *q_out_dev, void *stream);

/* ------------------------------------------------------------ attention */

/* For every token of the call, at position p, and head h of n_head (a multiple
 * r of n_kv_head; head h reads key head h / r):
 *   o = sum_j softmax_j(scale * q . k_j) v_j
 * over the positions j that it sees: 0 <= j <= p, and where window > 0 only
 * j > p - window or j < sinks. A token that sees none gives zeros. q and o are
 * dtype (STRATA_QUANT_F32 or STRATA_QUANT_BF16), token rows of n_head *
 * head_dim elements `*_stride` elements apart (0 = packed). The call's own keys
 * and values are in the cache already (kv_append). scale is above 0.
 *
 * Scores, maxima, weights' sums and outputs are f32. Where dtype is bf16,
 * weights are rounded to bf16 before they meet the values (relative to the
 * largest so far), as q, k and v are bf16 themselves, and o is rounded once;
 * where it is f32, queries and weights keep 24 bits. NaN and infinities in what
 * a token sees reach its outputs as the formula has them; what it does not see
 * (pages' unused rows, later tokens, keys outside the window) never does.
 *
 * work_dev: strata_cuda_attention_work_bytes bytes, 16-byte aligned; its
 * contents need not be kept between calls, and calls that may overlap need one
 * each. A device wait that expires leaves o undefined and is reported as
 * STRATA_ERR_TIMEOUT by the context's next host wait. o may overlap neither q
 * nor the cache.
 *
 * bf16 chunks of heads up to 128 are computed in tiles of 128 rows where q and o
 * are 16-byte aligned and their strides multiples of 8; otherwise 16 rows at a
 * time, as f32 and larger heads are (16 chunks of 64 tokens, 32 heads on 8 of 128,
 * behind 8000 keys: 155 us in tiles, 1197 so). */
typedef struct {
    int64_t n_seq;
    int64_t seq_len;            /* tokens of every sequence when seq_offsets is NULL */
    const int64_t *seq_offsets; /* host memory, n_seq + 1 row numbers, or NULL */
    int64_t n_head;
    int64_t q_stride, o_stride;
    int64_t window, sinks;      /* window 0: everything up to the token itself */
    double scale;
    uint32_t dtype;
} strata_attention;

int strata_cuda_attention_work_bytes(const strata_attention *desc, const strata_kv_cache *cache, uint64_t *bytes);
int strata_cuda_attention_dev(strata_ctx *ctx, const strata_attention *desc, const strata_kv_cache *cache,
                              const void *q_dev, void *o_dev, void *work_dev, uint64_t work_bytes, void *stream);

/* ---------------------------------------------------- log-probabilities */

/* For every row of logits (rows x vocab f32, rows `stride` floats apart, 0 =
 * vocab; vocab up to 2^22), with p = softmax of the row:
 *   logprobs      log p of targets[row] (int32); 0 where the target is outside
 *                 [0, vocab), so that padded rows add nothing to a sum
 *   entropy       -sum p log p, or NULL
 *   top_ids,      the `top` (0 to 32) likeliest tokens, [rows][top], likeliest
 *   top_logprobs  first, equal logits by index, the lowest first; both NULL
 *                 where top is 0
 * in natural logarithms. As in sample: a NaN counts as -inf; infinite logits
 * share everything; a row with nothing left has log-probabilities of -inf and
 * entropy 0; where fewer than `top` logits are above -inf the rest of the list
 * is id -1 with -inf. targets and logprobs may both be NULL, rows may be 0.
 * Weights are f32 exponentials, their sum f64. A row of which more than 1024
 * logits may be among the likeliest, equal ones in the main, is read once more for
 * each entry of the list: leave tokens out with -inf, not with the lowest f32. */
int strata_cuda_logprobs_dev(strata_ctx *ctx, const float *logits_dev, int64_t rows, int64_t vocab, int64_t stride,
                             const int32_t *targets_dev, float *logprobs_dev, float *entropy_dev, int64_t top,
                             int32_t *top_ids_dev, float *top_logprobs_dev, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* STRATA_ATTENTION_H */
