/*
 * strata_sequence.h — the sequence operators of libstrata_cuda: what a
 * recurrent layer does between its projections, and the choice of the next
 * token after the head projection, on device buffers, so that a token step
 * (strata_cuda.h's GEMV / GEMM / MoE / elementwise calls and these) never
 * returns to the host.
 *
 *   short_conv    causal depthwise convolution with its state
 *   gated_delta   the gated delta rule with its matrix state (one token per
 *                 sequence when decoding, whole prompts chunk by chunk)
 *   sample        top-k, top-p, min-p and temperature from given random numbers
 *
 * The reference runs these steps on the host (crates/strata-core/src/gdn.rs,
 * crates/strata-core/src/sampler.rs). Status codes, contexts, streams and
 * strata_cuda_last_error are strata_cuda.h's. All pointers named *_dev are
 * device memory of the context's device; the calls only enqueue work on
 * `stream` (NULL = the context's own stream), allocate nothing, keep nothing
 * between calls, leave the calling thread's current device as it was and can
 * be captured into a graph (the host-side values they are given, sequence
 * lengths among them, are then part of the graph). Calls that share no buffer
 * may run at the same time on different streams.
 *
 * Sequences: the tokens of a call are rows of its buffers. Either every
 * sequence has seq_len tokens (seq_offsets NULL; sequence i holds rows
 * [i * seq_len, (i + 1) * seq_len)), or seq_offsets gives n_seq + 1
 * non-decreasing row numbers in HOST memory, read during the call (sequence i
 * holds rows [seq_offsets[i], seq_offsets[i + 1])). A sequence may be empty:
 * its state stays as it is; where all are, a call does nothing and its buffers
 * may be NULL. Rows outside every sequence are neither read nor written. Below
 * 2^31 rows.
 */
#ifndef STRATA_SEQUENCE_H
#define STRATA_SEQUENCE_H

#include "strata_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------- short convolution */

/* For every token t and channel c of a sequence
 *   y[t][c] = act(bias[c] + sum_{j < taps} w[c][j] * x[t - (taps - 1) + j][c]),
 * act(z) = z / (1 + exp(-z)) where silu is set, else z. The inputs before the
 * sequence's first token are its state: state[i] holds the last taps - 1
 * inputs, oldest first ([n_seq][taps - 1][channels] f32), and is replaced by
 * the last taps - 1 inputs once the call's tokens are through. x and y are
 * dtype (STRATA_QUANT_F32 or STRATA_QUANT_BF16), sums are f32, y is rounded
 * once (nearest even). w is channels x taps f32 (ggml's [taps, channels]),
 * bias channels f32 or NULL; taps 1..8 (state_dev may be NULL when 1).
 * y may not overlap x, the weights or the state. */
typedef struct {
    int64_t n_seq;
    int64_t seq_len;            /* tokens of every sequence when seq_offsets is NULL */
    const int64_t *seq_offsets; /* host memory, n_seq + 1 row numbers, or NULL */
    int64_t channels, taps;
    int64_t x_stride, y_stride; /* elements from one token to the next; 0 = channels */
    uint32_t dtype;
    int silu;
} strata_short_conv;

int strata_cuda_short_conv_dev(strata_ctx *ctx, const strata_short_conv *desc, const void *x_dev, const float *w_dev,
                               const float *bias_dev, float *state_dev, void *y_dev, void *stream);

/* -------------------------------------------------------- gated delta rule */

/* Per sequence and value head h, with the state S (k_dim x v_dim f32, row-major,
 * [n_seq][n_v_head][k_dim][v_dim], updated in place):
 *   S <- exp(g) S
 *   S <- S + k (beta (v - S^T k))^T
 *   o  = scale * S^T q
 * for its tokens in order. q and k have n_k_head heads, v and o n_v_head (a
 * multiple r of n_k_head): value head h reads key head h / r, or h mod n_k_head
 * where `tiled` is set. q, k, v and o are dtype, token rows of n_head * dim
 * elements (heads side by side) `*_stride` elements apart, so they may be
 * columns of one projection's output. gate and beta are f32, n_v_head a token:
 *   raw_gates 0   g = gate (the log of the decay), beta = beta
 *   raw_gates 1   g = coef[h] * log(1 + exp(gate + shift[h])), beta = 1 / (1 + exp(-beta));
 *                 shift may be NULL (zeros)
 * Where l2_eps >= 0, q and k are first divided by sqrt(sum of squares + l2_eps)
 * per head; a negative l2_eps takes them as they are. k_dim 1..256, v_dim 1..8192.
 *
 * Products and sums are f32; o is rounded once. Sequences are read in chunks of
 * 32 tokens on the tensor cores where k_dim is up to 128 and a sequence of the
 * call has 16 tokens or more, 20 where there are few heads and sequences (many
 * shorter ones beside it are still read token by token). There, products over
 * k_dim carry 22 bits of the norms of their vectors (a key, a query, a column of
 * the state; the elements of one that lie 2^18 below its largest carry fewer of
 * their own), and all others 22 bits of themselves: however sizes differ, no
 * column costs another, and no token an earlier one, precision. Either way,
 * squares of q and k are summed in f32, so normalised ones have norms below
 * 1.8e19, and in chunks the decay from one token to another within 32 is one f32
 * factor: gates above 0 may add up to 88 there, and below e^-88 it counts as 0.
 * Chunks need strata_cuda_gated_delta_work_bytes bytes of
 * work_dev (16-byte aligned; its contents need not be kept between calls, and
 * calls that may overlap need one each); where that is 0 work_dev may be NULL.
 * A NaN or infinity among a token's inputs reaches its own and later outputs of
 * its sequence and head and, where it is read in chunks, earlier ones of the
 * same chunk. A device wait that expires leaves o and the state undefined and
 * is reported as STRATA_ERR_TIMEOUT by the context's next host wait
 * (strata_cuda_synchronize). The state may not overlap an input, nor o
 * overlap any input. */
typedef struct {
    int64_t n_seq;
    int64_t seq_len;            /* tokens of every sequence when seq_offsets is NULL */
    const int64_t *seq_offsets; /* host memory, n_seq + 1 row numbers, or NULL */
    int64_t n_k_head, n_v_head, k_dim, v_dim;
    int64_t q_stride, k_stride, v_stride, o_stride; /* elements between tokens; 0 = n_head * dim */
    int64_t gate_stride, beta_stride;               /* floats between tokens; 0 = n_v_head */
    double scale, l2_eps;
    uint32_t dtype;
    int tiled, raw_gates;
} strata_gated_delta;

int strata_cuda_gated_delta_work_bytes(const strata_gated_delta *desc, uint64_t *bytes);
int strata_cuda_gated_delta_dev(strata_ctx *ctx, const strata_gated_delta *desc, const void *q_dev, const void *k_dev,
                                const void *v_dev, const float *gate_dev, const float *beta_dev, const float *coef_dev,
                                const float *shift_dev, float *state_dev, void *o_dev, void *work_dev,
                                uint64_t work_bytes, void *stream);

/* ---------------------------------------------------------------- sampling */

/* One token for every row of logits (rows x vocab f32, rows `stride` floats
 * apart, 0 = vocab; vocab up to 2^22). The reference's sampler applies its
 * penalties first (they need the tokens so far); a caller that has some changes
 * the logits before the call. Per row, in this order:
 *   top_k        keeps the k largest logits; k <= 0 keeps all
 *   top_p        with the kept tokens' softmax in falling order, keeps the
 *                shortest prefix whose sum reaches p (one token at least);
 *                p >= 1 keeps all
 *   min_p        keeps tokens at least m times as likely as the likeliest
 *                (which always stays); m <= 0 keeps all
 *   temperature  p_i ~ exp(logit_i / t) over what is kept; t <= 0 (or NaN) takes
 *                the largest logit
 *   uniform      u in [0, 1): the first kept token, in index order, whose
 *                cumulative probability exceeds u (u outside is clamped)
 * Equal logits rank by index, the lowest first. Sums and exponentials are f64:
 * a p or u that falls on a border between two tokens to within 1e-13 of the
 * total may be taken to either side of it.
 * A logit of -inf or NaN is never taken; infinite ones share everything; a row
 * with nothing left gives id -1 and log-probability -inf. ids_dev receives
 * int32, logprobs_dev (or NULL) the natural log of the taken token's final
 * probability (0 where t <= 0). Each settings array holds one value per row;
 * NULL means off (temperature: 1), and so does a NaN top_p or min_p. */
int strata_cuda_sample_dev(strata_ctx *ctx, const float *logits_dev, int64_t rows, int64_t vocab, int64_t stride,
                           const float *temperature_dev, const int32_t *top_k_dev, const float *top_p_dev,
                           const float *min_p_dev, const double *uniform_dev, int32_t *ids_dev, float *logprobs_dev,
                           void *stream);

#ifdef __cplusplus
}
#endif
#endif /* STRATA_SEQUENCE_H */
