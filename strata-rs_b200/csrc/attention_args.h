// attention_args.h — the argument checks of strata_attention.h's calls. Host
// only and free of CUDA, as sequence_args.h, whose pieces they use; tested
// without a device (tests/attention_args_check.cpp).
#pragma once
#include "../../include/strata_attention.h"
#include "sequence_args.h"

namespace strata {

// Resolves packed strides in `c`.
inline int check_kv_cache(Why& why, strata_kv_cache& c, int64_t n_seq) {
    if (c.n_kv_head < 1 || c.n_kv_head > 1024) return why.refuse(STRATA_ERR_INVALID, "n_kv_head %lld (1 to 1024)", (long long)c.n_kv_head);
    if (c.head_dim < 8 || c.head_dim > 256 || c.head_dim % 8)
        return why.refuse(STRATA_ERR_INVALID, "head_dim %lld (a multiple of 8 up to 256)", (long long)c.head_dim);
    if (c.page_size < 16 || c.page_size % 16 || c.page_size > kMaxTokens)
        return why.refuse(STRATA_ERR_INVALID, "page_size %lld (a multiple of 16)", (long long)c.page_size);
    if (c.n_pages < 1 || c.n_pages > kMaxTokens) return why.refuse(STRATA_ERR_INVALID, "bad n_pages %lld", (long long)c.n_pages);
    if (c.max_pages < 1 || c.max_pages > kMaxTokens / c.page_size)
        return why.refuse(STRATA_ERR_INVALID, "max_pages %lld of %lld tokens (below 2^31 tokens)", (long long)c.max_pages,
                          (long long)c.page_size);
    if (c.table_stride == 0) c.table_stride = c.max_pages;
    if (c.table_stride < c.max_pages || c.table_stride > kMaxStride)
        return why.refuse(STRATA_ERR_INVALID, "table_stride is %lld for rows of %lld", (long long)c.table_stride, (long long)c.max_pages);
    if (n_seq > kMaxElements / c.table_stride) return why.refuse(STRATA_ERR_INVALID, "table_stride is %lld for %lld sequences", (long long)c.table_stride, (long long)n_seq);
    if (c.head_stride == 0) c.head_stride = c.head_dim;
    if (c.head_stride < c.head_dim || c.head_stride > kMaxElements / c.n_kv_head)
        return why.refuse(STRATA_ERR_INVALID, "head_stride is %lld for heads of %lld", (long long)c.head_stride, (long long)c.head_dim);
    if (c.token_stride == 0) c.token_stride = c.n_kv_head * c.head_stride;
    if (c.token_stride < c.head_dim || c.token_stride > kMaxElements / c.page_size)
        return why.refuse(STRATA_ERR_INVALID, "token_stride is %lld for heads of %lld", (long long)c.token_stride, (long long)c.head_dim);
    // rows of different heads and tokens may not share elements
    const int64_t heads = (c.n_kv_head - 1) * c.head_stride + c.head_dim, tokens = (c.page_size - 1) * c.token_stride + c.head_dim;
    const bool inside = c.token_stride >= heads;  // heads inside tokens
    if (!inside && c.head_stride < tokens)
        return why.refuse(STRATA_ERR_INVALID, "cache strides %lld and %lld overlap", (long long)c.token_stride, (long long)c.head_stride);
    if (c.page_stride == 0) c.page_stride = inside ? c.page_size * c.token_stride : c.n_kv_head * c.head_stride;
    const int64_t page = heads + tokens - c.head_dim;
    if (c.page_stride < page || c.page_stride > kMaxElements / c.n_pages)
        return why.refuse(STRATA_ERR_INVALID, "page_stride is %lld for %lld pages of %lld", (long long)c.page_stride, (long long)c.n_pages, (long long)page);
    if (c.page_stride % 8 || c.token_stride % 8 || c.head_stride % 8)
        return why.refuse(STRATA_ERR_INVALID, "cache strides %lld, %lld, %lld (multiples of 8)", (long long)c.page_stride,
                          (long long)c.token_stride, (long long)c.head_stride);
    return STRATA_OK;
}

// The elements from the first to the last of a pool, as one row.
inline Rows pool_rows(const char* what, const void* base, const strata_kv_cache& c) {
    const int64_t bytes = ((c.n_pages - 1) * c.page_stride + (c.page_size - 1) * c.token_stride + (c.n_kv_head - 1) * c.head_stride + c.head_dim) * 2;
    return {what, base, bytes, bytes, 1};
}

inline int check_kv_cache_buffers(Why& why, const strata_kv_cache& c) {
    if (!c.k_dev || !c.v_dev || !c.table_dev || !c.len_dev) return why.refuse(STRATA_ERR_INVALID, "null cache buffer");
    int rc;
    if ((rc = check_aligned(why, "the keys' pool", c.k_dev, 16)) || (rc = check_aligned(why, "the values' pool", c.v_dev, 16)) ||
        (rc = check_aligned(why, "the table", c.table_dev, 4)) || (rc = check_aligned(why, "the lengths", c.len_dev, 4)))
        return rc;
    if (c.k_dev == c.v_dev) return why.refuse(STRATA_ERR_INVALID, "keys and values in one pool");
    return STRATA_OK;
}

// Whether a key's and a value's row share elements (strides resolved: rows of a pool
// share none). The pools are apart by a number of pages, of rows of the outer stride and
// of the inner one, each known up to one, and a rest below a row.
inline bool pools_share(const strata_kv_cache& c) {
    const int64_t apart = (int64_t)((uintptr_t)c.v_dev - (uintptr_t)c.k_dev) / 2;
    const bool inside = c.token_stride >= (c.n_kv_head - 1) * c.head_stride + c.head_dim;
    const int64_t stride[] = {c.page_stride, inside ? c.token_stride : c.head_stride, inside ? c.head_stride : c.token_stride};
    const int64_t count[] = {c.n_pages, inside ? c.page_size : c.n_kv_head, inside ? c.n_kv_head : c.page_size};
    for (int up = 0; up < 8; ++up) {
        int64_t rest = apart;
        bool near = true;
        for (int i = 0; i < 3; ++i) {
            int64_t n = rest / stride[i] - (rest % stride[i] < 0);  // rounded down
            n += up >> i & 1;
            near &= n > -count[i] && n < count[i];
            rest -= n * stride[i];
        }
        if (near && rest > -c.head_dim && rest < c.head_dim) return true;
    }
    return false;
}

// Resolves packed strides in `d` and `c`.
inline int check_kv_append(Why& why, strata_kv_append& d, strata_kv_cache& c, int64_t* tokens, int64_t* longest) {
    int rc;
    if ((rc = check_dtype(why, d.dtype)) || (rc = check_dtype(why, d.q_dtype))) return rc;
    if ((rc = check_sequences(why, d.n_seq, d.seq_len, d.seq_offsets, tokens, longest))) return rc;
    if ((rc = check_kv_cache(why, c, d.n_seq))) return rc;
    if (d.n_head < 0 || d.n_head > 65536) return why.refuse(STRATA_ERR_INVALID, "bad n_head %lld", (long long)d.n_head);
    if (d.n_rot < 0 || d.n_rot > c.head_dim || d.n_rot % 2)
        return why.refuse(STRATA_ERR_INVALID, "n_rot %lld (even, up to head_dim %lld)", (long long)d.n_rot, (long long)c.head_dim);
    if (d.n_rot && !(std::isfinite(d.freq_base) && d.freq_base > 0)) return why.refuse(STRATA_ERR_INVALID, "freq_base is not above 0");
    const int64_t q = d.n_head * c.head_dim, kv = c.n_kv_head * c.head_dim;
    if (d.n_head && ((rc = check_stride(why, "q_stride", d.q_stride, q, *tokens)) || (rc = check_stride(why, "q_out_stride", d.q_out_stride, q, *tokens)))) return rc;
    if ((rc = check_stride(why, "k_stride", d.k_stride, kv, *tokens)) || (rc = check_stride(why, "v_stride", d.v_stride, kv, *tokens))) return rc;
    return STRATA_OK;
}

inline int check_kv_append_buffers(Why& why, const strata_kv_append& d, const strata_kv_cache& c, int64_t tokens, const void* q,
                                   const void* k, const void* v, const void* q_out) {
    if (!k || !v || (d.n_head && (!q || !q_out))) return why.refuse(STRATA_ERR_INVALID, "null buffer");
    int rc;
    const int64_t b = dtype_bytes(d.dtype), ob = dtype_bytes(d.q_dtype);
    if ((rc = check_kv_cache_buffers(why, c)) || (rc = check_aligned(why, "k", k, b)) || (rc = check_aligned(why, "v", v, b))) return rc;
    if (d.n_head && ((rc = check_aligned(why, "q", q, b)) || (rc = check_aligned(why, "q_out", q_out, ob)))) return rc;
    if (pools_share(c)) return why.refuse(STRATA_ERR_INVALID, "the keys' pool overlaps the values' pool");
    const int64_t qr = d.n_head * c.head_dim, kvr = c.n_kv_head * c.head_dim;
    const Rows in[] = {{"k", k, kvr * b, d.k_stride * b, tokens},
                       {"v", v, kvr * b, d.v_stride * b, tokens},
                       {"the table", c.table_dev, c.max_pages * 4, c.table_stride * 4, d.n_seq},
                       {"the lengths", c.len_dev, d.n_seq * 4, d.n_seq * 4, 1},
                       {"q", d.n_head ? q : nullptr, qr * b, d.q_stride * b, tokens}};
    const Rows out = {"q_out", d.n_head ? q_out : nullptr, qr * ob, d.q_out_stride * ob, tokens};
    const Rows kp = pool_rows("the keys' pool", c.k_dev, c), vp = pool_rows("the values' pool", c.v_dev, c);
    const bool in_place = q == q_out && d.dtype == d.q_dtype && d.q_stride == d.q_out_stride;
    if ((rc = check_overlaps(why, out, in, in_place ? 4 : 5)) || (rc = check_overlaps(why, kp, in, 5)) || (rc = check_overlaps(why, vp, in, 5)) ||
        (rc = check_overlaps(why, out, &kp, 1)))
        return rc;
    return check_overlaps(why, out, &vp, 1);
}

// Resolves packed strides in `d` and `c`.
inline int check_attention(Why& why, strata_attention& d, strata_kv_cache& c, int64_t* tokens, int64_t* longest) {
    int rc;
    if ((rc = check_dtype(why, d.dtype))) return rc;
    if ((rc = check_sequences(why, d.n_seq, d.seq_len, d.seq_offsets, tokens, longest))) return rc;
    if ((rc = check_kv_cache(why, c, d.n_seq))) return rc;
    if (d.n_head < 1 || d.n_head > 65536 || d.n_head % c.n_kv_head)
        return why.refuse(STRATA_ERR_INVALID, "%lld heads on %lld key heads", (long long)d.n_head, (long long)c.n_kv_head);
    if (*longest > kMaxTokens / d.n_head) return why.refuse(STRATA_ERR_INVALID, "%lld tokens of %lld heads", (long long)*longest, (long long)d.n_head);
    if (d.window < 0 || d.sinks < 0) return why.refuse(STRATA_ERR_INVALID, "bad window %lld or sinks %lld", (long long)d.window, (long long)d.sinks);
    if (!(std::isfinite((float)(d.scale * 1.5)) && (float)d.scale > 0))  // in powers of two it is larger
        return why.refuse(STRATA_ERR_INVALID, "scale is not above 0, or too large");
    const int64_t row = d.n_head * c.head_dim;
    if ((rc = check_stride(why, "q_stride", d.q_stride, row, *tokens)) || (rc = check_stride(why, "o_stride", d.o_stride, row, *tokens))) return rc;
    return STRATA_OK;
}

inline int check_attention_buffers(Why& why, const strata_attention& d, const strata_kv_cache& c, int64_t tokens, const void* q,
                                   const void* o, const void* work, uint64_t work_bytes, uint64_t work_needed) {
    if (!q || !o) return why.refuse(STRATA_ERR_INVALID, "null buffer");
    if (work_needed && (!work || work_bytes < work_needed))
        return why.refuse(STRATA_ERR_SCRATCH_LIMIT, "%llu bytes of work, %llu needed", (unsigned long long)(work ? work_bytes : 0),
                          (unsigned long long)work_needed);
    const int64_t b = dtype_bytes(d.dtype), row = d.n_head * c.head_dim * b, wn = (int64_t)work_needed;
    int rc;
    if ((rc = check_kv_cache_buffers(why, c)) || (rc = check_aligned(why, "q", q, b)) || (rc = check_aligned(why, "o", o, b))) return rc;
    if (work_needed && (rc = check_aligned(why, "work", work, 16))) return rc;
    const Rows in[] = {{"q", q, row, d.q_stride * b, tokens},
                       pool_rows("the keys' pool", c.k_dev, c),
                       pool_rows("the values' pool", c.v_dev, c),
                       {"the table", c.table_dev, c.max_pages * 4, c.table_stride * 4, d.n_seq},
                       {"the lengths", c.len_dev, d.n_seq * 4, d.n_seq * 4, 1}};
    const Rows out = {"o", o, row, d.o_stride * b, tokens}, wk = {"work", work_needed ? work : nullptr, wn, wn, 1};
    if ((rc = check_overlaps(why, out, in, 5)) || (rc = check_overlaps(why, wk, in, 5))) return rc;
    return check_overlaps(why, wk, &out, 1);
}

constexpr int64_t kMaxTop = 32;

// Resolves a packed stride.
inline int check_logprobs(Why& why, const float* logits, int64_t rows, int64_t vocab, int64_t& stride, const int32_t* targets,
                          const float* logprobs, const float* entropy, int64_t top, const int32_t* top_ids, const float* top_logprobs) {
    if (rows < 0 || rows > (int64_t(1) << 24)) return why.refuse(STRATA_ERR_INVALID, "bad rows %lld", (long long)rows);
    if (vocab < 1 || vocab > (int64_t(1) << 22)) return why.refuse(STRATA_ERR_INVALID, "vocab %lld (1 to 2^22)", (long long)vocab);
    if (top < 0 || top > kMaxTop) return why.refuse(STRATA_ERR_INVALID, "top %lld (0 to 32)", (long long)top);
    int rc;
    if ((rc = check_stride(why, "stride", stride, vocab, rows))) return rc;
    if (rows == 0) return STRATA_OK;
    if (!logits || !targets != !logprobs || (top && (!top_ids || !top_logprobs))) return why.refuse(STRATA_ERR_INVALID, "null buffer");
    if ((rc = check_aligned(why, "logits", logits, 4)) || (rc = check_aligned(why, "targets", targets, 4)) ||
        (rc = check_aligned(why, "logprobs", logprobs, 4)) || (rc = check_aligned(why, "entropy", entropy, 4)) ||
        (rc = check_aligned(why, "top_ids", top_ids, 4)) || (rc = check_aligned(why, "top_logprobs", top_logprobs, 4)))
        return rc;
    const int64_t r4 = rows * 4, t4 = rows * top * 4;
    const Rows in[] = {{"logits", logits, vocab * 4, stride * 4, rows}, {"targets", targets, r4, r4, 1}};
    const Rows out[] = {{"logprobs", logprobs, r4, r4, 1}, {"entropy", entropy, r4, r4, 1},
                        {"top_ids", top ? top_ids : nullptr, t4, t4, 1}, {"top_logprobs", top ? top_logprobs : nullptr, t4, t4, 1}};
    for (int i = 0; i < 4; ++i)
        if ((rc = check_overlaps(why, out[i], in, 2)) || (rc = check_overlaps(why, out[i], out, i))) return rc;
    return STRATA_OK;
}

}  // namespace strata
