// sequence_args.h — the argument checks of strata_sequence.h's calls. Host
// only and free of CUDA, so they are tested without a device
// (tests/sequence_args_check.cpp). Each check returns a status and, on a
// refusal, leaves the reason in `why`.
#pragma once
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/strata_sequence.h"

namespace strata {

struct Why {
    char text[192] = "";
    int refuse(int code, const char* fmt, ...) __attribute__((format(printf, 3, 4))) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(text, sizeof text, fmt, ap);
        va_end(ap);
        return code;
    }
};

constexpr int64_t kMaxTokens = (int64_t(1) << 31) - 1;
constexpr int64_t kMaxStride = int64_t(1) << 31;
constexpr int64_t kMaxElements = int64_t(1) << 56;  // of a buffer, strides included: byte offsets stay far inside 64 bits

// A buffer as the rows a call touches: `rows` rows of `row` bytes, `pitch`
// bytes apart, from `base`.
struct Rows {
    const char* what;
    const void* base;
    int64_t row, pitch, rows;
};

inline bool overlap(const Rows& a, const Rows& b) {
    if (!a.base || !b.base || a.rows <= 0 || b.rows <= 0 || a.row <= 0 || b.row <= 0) return false;
    const uintptr_t a0 = (uintptr_t)a.base, b0 = (uintptr_t)b.base;
    const uintptr_t a1 = a0 + (uintptr_t)((a.rows - 1) * a.pitch + a.row);
    const uintptr_t b1 = b0 + (uintptr_t)((b.rows - 1) * b.pitch + b.row);
    if (a1 <= b0 || b1 <= a0) return false;
    if (a.pitch != b.pitch || a.pitch <= 0) return true;
    // interleaved rows of one pitch (columns of one buffer) share bytes only
    // where the row extents meet modulo the pitch
    const int64_t shift = (int64_t)((b0 >= a0 ? b0 - a0 : a.pitch - (int64_t)((a0 - b0) % (uintptr_t)a.pitch)) %
                                    (uintptr_t)a.pitch);
    return shift < a.row || shift + b.row > a.pitch;
}

inline int check_overlaps(Why& why, const Rows& out, const Rows* in, int n) {
    for (int i = 0; i < n; ++i)
        if (overlap(out, in[i])) return why.refuse(STRATA_ERR_INVALID, "%s overlaps %s", out.what, in[i].what);
    return STRATA_OK;
}

inline int check_aligned(Why& why, const char* what, const void* p, int64_t bytes) {
    if ((uintptr_t)p % (uintptr_t)bytes)
        return why.refuse(STRATA_ERR_INVALID, "%s is not %lld-byte aligned", what, (long long)bytes);
    return STRATA_OK;
}

inline int64_t dtype_bytes(uint32_t dtype) { return dtype == STRATA_QUANT_BF16 ? 2 : 4; }

// The sequences of a call: `tokens` receives the row behind the last sequence,
// `longest` the largest number of tokens of one.
inline int check_sequences(Why& why, int64_t n_seq, int64_t seq_len, const int64_t* off, int64_t* tokens,
                           int64_t* longest) {
    if (n_seq < 1 || n_seq > kMaxTokens) return why.refuse(STRATA_ERR_INVALID, "bad n_seq %lld", (long long)n_seq);
    *longest = 0;
    if (!off) {
        if (seq_len < 0 || seq_len > kMaxTokens || seq_len * n_seq > kMaxTokens)
            return why.refuse(STRATA_ERR_INVALID, "bad sequence length %lld x %lld", (long long)n_seq,
                              (long long)seq_len);
        *tokens = n_seq * seq_len;
        *longest = seq_len;
        return STRATA_OK;
    }
    if (off[0] < 0) return why.refuse(STRATA_ERR_INVALID, "seq_offsets[0] is %lld", (long long)off[0]);
    for (int64_t i = 0; i < n_seq; ++i) {
        if (off[i + 1] < off[i] || off[i + 1] > kMaxTokens)
            return why.refuse(STRATA_ERR_INVALID, "seq_offsets[%lld] is %lld after %lld", (long long)(i + 1),
                              (long long)off[i + 1], (long long)off[i]);
        if (off[i + 1] - off[i] > *longest) *longest = off[i + 1] - off[i];
    }
    *tokens = off[n_seq];
    return STRATA_OK;
}

// 0 = packed; otherwise at least one row. `rows` rows of it are a buffer.
inline int check_stride(Why& why, const char* what, int64_t& stride, int64_t packed, int64_t rows) {
    if (stride == 0) stride = packed;
    if (stride < packed || stride > kMaxStride)
        return why.refuse(STRATA_ERR_INVALID, "%s is %lld for rows of %lld", what, (long long)stride,
                          (long long)packed);
    if (rows > kMaxElements / stride)
        return why.refuse(STRATA_ERR_INVALID, "%s is %lld for %lld rows", what, (long long)stride, (long long)rows);
    return STRATA_OK;
}

// The states of n sequences, `each` elements long (below 2^40).
inline int check_states(Why& why, int64_t n, int64_t each) {
    if (each > 0 && n > kMaxElements / each)
        return why.refuse(STRATA_ERR_INVALID, "%lld states of %lld elements", (long long)n, (long long)each);
    return STRATA_OK;
}

inline int check_dtype(Why& why, uint32_t dtype) {
    if (dtype != STRATA_QUANT_F32 && dtype != STRATA_QUANT_BF16)
        return why.refuse(STRATA_ERR_UNSUPPORTED_QUANT, "dtype %u (F32 or BF16)", dtype);
    return STRATA_OK;
}

// Resolves packed strides in `d`.
inline int check_short_conv(Why& why, strata_short_conv& d, int64_t* tokens, int64_t* longest) {
    int rc;
    if ((rc = check_dtype(why, d.dtype))) return rc;
    if ((rc = check_sequences(why, d.n_seq, d.seq_len, d.seq_offsets, tokens, longest))) return rc;
    if (d.channels < 1 || d.channels > (int64_t(1) << 30))
        return why.refuse(STRATA_ERR_INVALID, "bad channels %lld", (long long)d.channels);
    if (d.taps < 1 || d.taps > 8) return why.refuse(STRATA_ERR_INVALID, "taps %lld (1 to 8)", (long long)d.taps);
    if ((rc = check_stride(why, "x_stride", d.x_stride, d.channels, *tokens)) ||
        (rc = check_stride(why, "y_stride", d.y_stride, d.channels, *tokens)))
        return rc;
    return check_states(why, d.n_seq, (d.taps - 1) * d.channels);
}

// `d` and `tokens` as check_short_conv left them.
inline int check_short_conv_buffers(Why& why, const strata_short_conv& d, int64_t tokens, const void* x,
                                    const float* w, const float* bias, const float* state, const void* y) {
    if (!x || !w || !y || (!state && d.taps > 1)) return why.refuse(STRATA_ERR_INVALID, "null buffer");
    const int64_t b = dtype_bytes(d.dtype);
    int rc;
    if ((rc = check_aligned(why, "x", x, b)) || (rc = check_aligned(why, "y", y, b)) ||
        (rc = check_aligned(why, "w", w, 4)) || (rc = check_aligned(why, "bias", bias, 4)) ||
        (rc = check_aligned(why, "state", state, 4)))
        return rc;
    const int64_t c = d.channels;
    const Rows in[] = {{"x", x, c * b, d.x_stride * b, tokens}, {"w", w, c * d.taps * 4, c * d.taps * 4, 1},
                       {"bias", bias, c * 4, c * 4, 1}};
    const Rows st = {"state", d.taps > 1 ? state : nullptr, (d.taps - 1) * c * 4, (d.taps - 1) * c * 4, d.n_seq};
    const Rows out = {"y", y, c * b, d.y_stride * b, tokens};
    if ((rc = check_overlaps(why, out, in, 3)) || (rc = check_overlaps(why, out, &st, 1))) return rc;
    return check_overlaps(why, st, in, 3);
}

// Resolves packed strides in `d`.
inline int check_gated_delta(Why& why, strata_gated_delta& d, int64_t* tokens, int64_t* longest) {
    int rc;
    if ((rc = check_dtype(why, d.dtype))) return rc;
    if ((rc = check_sequences(why, d.n_seq, d.seq_len, d.seq_offsets, tokens, longest))) return rc;
    if (d.n_k_head < 1 || d.n_v_head < 1 || d.n_v_head > 65536 || d.n_v_head % d.n_k_head)
        return why.refuse(STRATA_ERR_INVALID, "%lld value heads on %lld key heads", (long long)d.n_v_head,
                          (long long)d.n_k_head);
    if (d.k_dim < 1 || d.k_dim > 256 || d.v_dim < 1 || d.v_dim > 8192)
        return why.refuse(STRATA_ERR_INVALID, "head sizes %lld x %lld (k_dim 1 to 256, v_dim 1 to 8192)",
                          (long long)d.k_dim, (long long)d.v_dim);
    if (!std::isfinite((float)d.scale)) return why.refuse(STRATA_ERR_INVALID, "scale is not finite");
    if (std::isnan(d.l2_eps) || d.l2_eps > 1e30) return why.refuse(STRATA_ERR_INVALID, "bad l2_eps");
    if ((rc = check_stride(why, "q_stride", d.q_stride, d.n_k_head * d.k_dim, *tokens)) ||
        (rc = check_stride(why, "k_stride", d.k_stride, d.n_k_head * d.k_dim, *tokens)) ||
        (rc = check_stride(why, "v_stride", d.v_stride, d.n_v_head * d.v_dim, *tokens)) ||
        (rc = check_stride(why, "o_stride", d.o_stride, d.n_v_head * d.v_dim, *tokens)) ||
        (rc = check_stride(why, "gate_stride", d.gate_stride, d.n_v_head, *tokens)) ||
        (rc = check_stride(why, "beta_stride", d.beta_stride, d.n_v_head, *tokens)))
        return rc;
    return check_states(why, d.n_seq, d.n_v_head * d.k_dim * d.v_dim);
}

inline int check_gated_delta_buffers(Why& why, const strata_gated_delta& d, int64_t tokens, const void* q,
                                     const void* k, const void* v, const float* gate, const float* beta,
                                     const float* coef, const float* shift, const float* state, const void* o,
                                     const void* work, uint64_t work_bytes, uint64_t work_needed) {
    if (!q || !k || !v || !gate || !beta || !state || !o) return why.refuse(STRATA_ERR_INVALID, "null buffer");
    if (d.raw_gates && !coef) return why.refuse(STRATA_ERR_INVALID, "raw gates need coef");
    if (work_needed && (!work || work_bytes < work_needed))
        return why.refuse(STRATA_ERR_SCRATCH_LIMIT, "%llu bytes of work, %llu needed",
                          (unsigned long long)(work ? work_bytes : 0), (unsigned long long)work_needed);
    const int64_t b = dtype_bytes(d.dtype);
    int rc;
    if ((rc = check_aligned(why, "q", q, b)) || (rc = check_aligned(why, "k", k, b)) ||
        (rc = check_aligned(why, "v", v, b)) || (rc = check_aligned(why, "o", o, b)) ||
        (rc = check_aligned(why, "gate", gate, 4)) || (rc = check_aligned(why, "beta", beta, 4)) ||
        (rc = check_aligned(why, "coef", coef, 4)) || (rc = check_aligned(why, "shift", shift, 4)) ||
        (rc = check_aligned(why, "state", state, 4)))
        return rc;
    if (work_needed && (rc = check_aligned(why, "work", work, 16))) return rc;
    const int64_t kr = d.n_k_head * d.k_dim * b, vr = d.n_v_head * d.v_dim * b, gr = d.n_v_head * 4;
    const int64_t sr = d.n_v_head * d.k_dim * d.v_dim * 4;
    const Rows in[] = {{"q", q, kr, d.q_stride * b, tokens},
                       {"k", k, kr, d.k_stride * b, tokens},
                       {"v", v, vr, d.v_stride * b, tokens},
                       {"gate", gate, gr, d.gate_stride * 4, tokens},
                       {"beta", beta, gr, d.beta_stride * 4, tokens},
                       {"coef", d.raw_gates ? coef : nullptr, gr, gr, 1},
                       {"shift", d.raw_gates ? shift : nullptr, gr, gr, 1}};
    const Rows st = {"state", state, sr, sr, d.n_seq};
    const Rows out = {"o", o, vr, d.o_stride * b, tokens};
    const int64_t wn = (int64_t)work_needed;
    const Rows wk = {"work", work_needed ? work : nullptr, wn, wn, 1};
    if ((rc = check_overlaps(why, out, in, 7)) || (rc = check_overlaps(why, st, in, 7)) ||
        (rc = check_overlaps(why, wk, in, 7)) || (rc = check_overlaps(why, out, &st, 1)) ||
        (rc = check_overlaps(why, wk, &st, 1)))
        return rc;
    return check_overlaps(why, wk, &out, 1);
}

// Resolves a packed stride.
inline int check_sample(Why& why, const float* logits, int64_t rows, int64_t vocab, int64_t& stride,
                        const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                        const double* uniform, const int32_t* ids, const float* logprobs) {
    if (!logits || !uniform || !ids) return why.refuse(STRATA_ERR_INVALID, "null buffer");
    if (rows < 1 || rows > (int64_t(1) << 24)) return why.refuse(STRATA_ERR_INVALID, "bad rows %lld", (long long)rows);
    if (vocab < 1 || vocab > (int64_t(1) << 22))
        return why.refuse(STRATA_ERR_INVALID, "vocab %lld (1 to 2^22)", (long long)vocab);
    int rc;
    if ((rc = check_stride(why, "stride", stride, vocab, rows)) || (rc = check_aligned(why, "logits", logits, 4)) ||
        (rc = check_aligned(why, "temperature", temperature, 4)) || (rc = check_aligned(why, "top_k", top_k, 4)) ||
        (rc = check_aligned(why, "top_p", top_p, 4)) || (rc = check_aligned(why, "min_p", min_p, 4)) ||
        (rc = check_aligned(why, "uniform", uniform, 8)) || (rc = check_aligned(why, "ids", ids, 4)) ||
        (rc = check_aligned(why, "logprobs", logprobs, 4)))
        return rc;
    const int64_t r4 = rows * 4;
    const Rows in[] = {{"logits", logits, vocab * 4, stride * 4, rows}, {"temperature", temperature, r4, r4, 1},
                       {"top_k", top_k, r4, r4, 1}, {"top_p", top_p, r4, r4, 1}, {"min_p", min_p, r4, r4, 1},
                       {"uniform", uniform, rows * 8, rows * 8, 1}};
    const Rows id = {"ids", ids, r4, r4, 1}, lp = {"logprobs", logprobs, r4, r4, 1};
    if ((rc = check_overlaps(why, id, in, 6)) || (rc = check_overlaps(why, lp, in, 6))) return rc;
    return check_overlaps(why, id, &lp, 1);
}

}  // namespace strata
