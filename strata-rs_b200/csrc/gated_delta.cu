// gated_delta.cu — the gated delta rule with its matrix state (the recurrence
// of a gated-delta layer; the reference's loop is in
// crates/strata-core/src/gdn.rs). Per sequence and value head, S: k_dim x v_dim,
//
//   u = beta (v - e^g S^T k),  S <- e^g S + k u^T,  o = scale S^T q.
//
// delta_step_kernel reads tokens one after another. Its columns of S are
// independent, so a block owns 32 * VEC columns of one head and holds them in
// registers (32 rows x VEC columns a thread; one warp per 32 rows) from the
// first token to the last: the state is read and written once a call. One pass
// over the registers gives both S^T k and S^T q, because
// S_new^T q = e^g S^T q + (k . q) u, so a token costs one reduction across the
// warps. For one token per sequence it is bound by the state's bytes: 128
// sequences of 32 heads of 128 x 128 take 88 us, 537 MB at 6.2 TB/s. One
// sequence is bound by latency (3.7 us, with a column a thread: four columns,
// a quarter of the blocks, took 5.6).
#include <cuda_runtime.h>

#include "gated_delta.cuh"

namespace strata {
namespace {

template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T* p, float (&d)[VEC]) {
    const Pack<T, VEC> in = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
    for (int v = 0; v < VEC; ++v) d[v] = to_f32(in.v[v]);
}

constexpr int kRows = 32;  // rows of S a thread holds

template <typename T, int WARPS, int VEC>
__global__ void __launch_bounds__(WARPS * 32, VEC == 4 ? (WARPS == 8 ? 1 : 12 / WARPS) : 1)
    delta_step_kernel(const DeltaArgs a, const __grid_constant__ SeqTable tab) {
    __shared__ float2 kq[2][WARPS * kRows];       // (k, q) of a token, as given
    __shared__ float part[2][WARPS][3];           // per warp: k.k, q.q, k.q
    __shared__ float2 red[WARPS][VEC][32];        // per warp: S^T k, S^T q
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int b = blockIdx.x;
    const int cb = b % a.col_blocks;
    b /= a.col_blocks;
    const int h = b % a.v_heads;
    const Seq seq = sequence_at(tab, b / a.v_heads);
    const int row = seq.row, len = seq.len;
    const int hk = key_head(a, h);
    const int c = (cb * 32 + lane) * VEC;
    const bool live = c < a.v_dim;
    float* S = a.state + ((int64_t)seq.slot * a.v_heads + h) * a.k_dim * a.v_dim + c;
    const int r0 = warp * kRows;

    float s[kRows][VEC];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (live && r0 + r < a.k_dim) load_pack<float, VEC>(S + (int64_t)(r0 + r) * a.v_dim, s[r]);
        else
#pragma unroll
            for (int v = 0; v < VEC; ++v) s[r][v] = 0.0f;
    }

    const int i = threadIdx.x;
    const T* kp = static_cast<const T*>(a.k) + (int64_t)row * a.k_stride + (int64_t)hk * a.k_dim + i;
    const T* qp = static_cast<const T*>(a.q) + (int64_t)row * a.q_stride + (int64_t)hk * a.k_dim + i;
    const T* vp = static_cast<const T*>(a.v) + (int64_t)row * a.v_stride + (int64_t)h * a.v_dim + c;
    T* op = static_cast<T*>(a.o) + (int64_t)row * a.o_stride + (int64_t)h * a.v_dim + c;
    const float* gp = a.gate + (int64_t)row * a.gate_stride + h;
    const float* bp = a.beta + (int64_t)row * a.beta_stride + h;
    float kn = 0.0f, qn = 0.0f, vn[VEC] = {}, gn = 0.0f, bn = 0.0f;
    auto fetch = [&] {
        if (i < a.k_dim) kn = to_f32(*kp), qn = to_f32(*qp);
        if (live) load_pack<T, VEC>(vp, vn);
        gn = *gp;
        bn = *bp;
        kp += a.k_stride, qp += a.q_stride, vp += a.v_stride, gp += a.gate_stride, bp += a.beta_stride;
    };
    fetch();
    for (int t = 0; t < len; ++t) {
        const int buf = t & 1;
        float kk = kn * kn, qq = qn * qn, xy = kn * qn;
        kq[buf][i] = make_float2(kn, qn);
        float v[VEC], g = gn, beta = bn;
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = vn[j];
        if (t + 1 < len) fetch();  // the next token's loads fly while this one is worked on
        gates(a, h, g, beta);
        const float decay = expf(g);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            kk += __shfl_xor_sync(0xFFFFFFFFu, kk, o);
            qq += __shfl_xor_sync(0xFFFFFFFFu, qq, o);
            xy += __shfl_xor_sync(0xFFFFFFFFu, xy, o);
        }
        if (lane == 0) part[buf][warp][0] = kk, part[buf][warp][1] = qq, part[buf][warp][2] = xy;
        __syncthreads();
        float sk[VEC] = {}, sq[VEC] = {};
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const float2 x = kq[buf][r0 + r];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                sk[j] = fmaf(x.x, s[r][j], sk[j]);
                sq[j] = fmaf(x.y, s[r][j], sq[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) red[warp][j][lane] = make_float2(sk[j], sq[j]);
        __syncthreads();
        kk = qq = xy = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) kk += part[buf][w][0], qq += part[buf][w][1], xy += part[buf][w][2];
        const float rk = a.norm ? 1.0f / sqrtf(kk + a.eps) : 1.0f;
        const float rq = a.scale * (a.norm ? 1.0f / sqrtf(qq + a.eps) : 1.0f);
        float u[VEC];
        Pack<T, VEC> out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float x = 0.0f, y = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float2 p = red[w][j][lane];
                x += p.x;
                y += p.y;
            }
            u[j] = rk * beta * (v[j] - decay * rk * x);
            from_f32(out.v[j], rq * (decay * y + xy * u[j]));
        }
        if (warp == 0 && live) *reinterpret_cast<Pack<T, VEC>*>(op) = out;
        op += a.o_stride;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const float k = kq[buf][r0 + r].x;
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[r][j] = fmaf(k, u[j], decay * s[r][j]);
        }
    }
    if (!live) return;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (r0 + r >= a.k_dim) break;
        Pack<float, VEC> out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) out.v[j] = s[r][j];
        *reinterpret_cast<Pack<float, VEC>*>(S + (int64_t)(r0 + r) * a.v_dim) = out;
    }
}

template <typename T, int VEC>
void launch_step(const DeltaArgs& a, const SeqTable& t, unsigned grid, cudaStream_t s) {
    if (a.k_dim <= 32) delta_step_kernel<T, 1, VEC><<<grid, 32, 0, s>>>(a, t);
    else if (a.k_dim <= 64) delta_step_kernel<T, 2, VEC><<<grid, 64, 0, s>>>(a, t);
    else if (a.k_dim <= 128) delta_step_kernel<T, 4, VEC><<<grid, 128, 0, s>>>(a, t);
    else delta_step_kernel<T, 8, VEC><<<grid, 256, 0, s>>>(a, t);
}

// The sequences that have tokens: empty ones launch nothing, so no rule counts them.
int64_t live_sequences(const strata_gated_delta& d) {
    if (!d.seq_offsets) return d.n_seq;
    int64_t n = 0;
    for (int64_t i = 0; i < d.n_seq; ++i) n += d.seq_offsets[i + 1] > d.seq_offsets[i];
    return n;
}

// Columns a thread takes: 4 (16-byte state accesses) or 2 where rows and
// pointers allow, 1 otherwise; fewer where that many blocks would leave
// multiprocessors without one.
int columns(const strata_gated_delta& d, const void* v, const float* state, const void* o, int sm_count) {
    const int64_t live = live_sequences(d);
    const int64_t b = dtype_bytes(d.dtype);
    for (int vec = 4; vec > 1; vec >>= 1) {
        if (d.v_dim % vec == 0 && d.v_stride % vec == 0 && d.o_stride % vec == 0 &&
            (uintptr_t)state % (4 * vec) == 0 && (uintptr_t)v % (b * vec) == 0 && (uintptr_t)o % (b * vec) == 0 &&
            d.v_dim > 32 * (vec / 2) && live * d.n_v_head * ((d.v_dim + 32 * vec - 1) / (32 * vec)) >= sm_count)
            return vec;
    }
    return 1;
}

// The tokens from which on a sequence of the call is read in chunks (more than
// `longest`: none is). A chunk takes as long with 16 tokens as with 32; measured
// in replayed graphs, tokens one after another against a chunk:
//   heads   32 of 128 x 128   16 of 64 x 64   64 of 96 x 128   2 of 32 x 32
//   1 seq.  0.70 a token, 12  0.61, 10        0.84, 14         0.61, 9.4 us
//   4       1.0, 24           0.62, 10        1.8, 30          0.61, 9.4
//   64      13, 254           2.1, 41         25, 358          0.63, 9.6
// (and 2 us a call), so they meet at 12 to 19 tokens, or at 21 where a few
// sequences' blocks have a multiprocessor each one way but share it the other.
// Beside long sequences a short
// one costs 3.7 us as a chunk against 0.5 us and 0.18 us a token, unless there
// are so few that they run alongside: 31 single tokens and 500 take 72 us, not
// 160, apart; 3 sequences of 12 tokens and 500 take 53 us, not 59, together.
int64_t chunks_from(const strata_gated_delta& d, int64_t longest) {
    const int64_t blocks = d.n_v_head * ((d.v_dim + 127) / 128), few = 128 / blocks;  // sequences
    if (d.k_dim > 128 || longest < 16 || (longest < 20 && live_sequences(d) <= few)) return longest + 1;
    if (!d.seq_offsets) return 1;
    int64_t n = 0;
    for (int64_t i = 0; i < d.n_seq; ++i) {
        const int64_t len = d.seq_offsets[i + 1] - d.seq_offsets[i];
        n += len > 0 && len < 16;
    }
    return n > few ? 16 : 1;
}

uint64_t work_needed(const strata_gated_delta& d, int64_t longest) {
    const int64_t from = chunks_from(d, longest);
    return from <= longest ? delta_chunk_work(d, from) : 0;
}

}  // namespace
}  // namespace strata

using namespace strata;

extern "C" {

int strata_cuda_gated_delta_work_bytes(const strata_gated_delta* desc, uint64_t* bytes) {
    if (!desc || !bytes) return STRATA_ERR_INVALID;
    *bytes = 0;
    strata_gated_delta d = *desc;
    Why why;
    int64_t tokens = 0, longest = 0;
    const int rc = check_gated_delta(why, d, &tokens, &longest);
    if (rc) return rc;
    *bytes = work_needed(d, longest);
    return STRATA_OK;
}

int strata_cuda_gated_delta_dev(strata_ctx* ctx, const strata_gated_delta* desc, const void* q_dev, const void* k_dev,
                                const void* v_dev, const float* gate_dev, const float* beta_dev, const float* coef_dev,
                                const float* shift_dev, float* state_dev, void* o_dev, void* work_dev,
                                uint64_t work_bytes, void* stream) {
    if (!ctx || !desc) return STRATA_ERR_INVALID;
    STRATA_CALL_RANGE();
    std::lock_guard<std::mutex> g(ctx->mu);
    strata_gated_delta d = *desc;
    Why why;
    int64_t tokens = 0, longest = 0;
    int rc = check_gated_delta(why, d, &tokens, &longest);
    if (!rc && longest > 0)
        rc = check_gated_delta_buffers(why, d, tokens, q_dev, k_dev, v_dev, gate_dev, beta_dev, coef_dev, shift_dev,
                                       state_dev, o_dev, work_dev, work_bytes, work_needed(d, longest));
    if (rc) return fail(ctx, rc, "gated_delta: %s", why.text);
    if (longest == 0) return STRATA_OK;
    const int vec = columns(d, v_dev, state_dev, o_dev, ctx->sm_count);
    const int64_t blocks = (d.v_dim + 32 * vec - 1) / (32 * vec);
    DeltaArgs a{q_dev, k_dev, v_dev, gate_dev, beta_dev, coef_dev, shift_dev, state_dev, o_dev, d.q_stride,
                d.k_stride, d.v_stride, d.o_stride, d.gate_stride, d.beta_stride, (int)d.n_k_head, (int)d.n_v_head,
                (int)d.k_dim, (int)d.v_dim, (int)blocks, d.tiled, d.raw_gates, d.l2_eps >= 0.0, (float)d.scale,
                (float)d.l2_eps};
    DeviceGuard dev(ctx->device);
    const cudaStream_t s = pick_stream(ctx, stream);
    const int64_t from = chunks_from(d, longest);
    if (from <= longest) {
        rc = delta_chunk_enqueue(ctx, d, a, work_dev, from, s);
        if (rc || from == 1) return rc;
    }
    return for_sequence_groups(d.n_seq, d.seq_len, d.seq_offsets, kMaxTokens, from, [&](const SeqTable& t, int64_t) {
        if (t.n * blocks * d.n_v_head > kMaxTokens)
            return fail(ctx, STRATA_ERR_INVALID, "gated_delta: %d sequences of %lld heads", t.n,
                        (long long)d.n_v_head);
        const unsigned grid = (unsigned)(t.n * blocks * d.n_v_head);
        if (d.dtype == STRATA_QUANT_BF16) {
            if (vec == 4) launch_step<__nv_bfloat16, 4>(a, t, grid, s);
            else if (vec == 2) launch_step<__nv_bfloat16, 2>(a, t, grid, s);
            else launch_step<__nv_bfloat16, 1>(a, t, grid, s);
        } else {
            if (vec == 4) launch_step<float, 4>(a, t, grid, s);
            else if (vec == 2) launch_step<float, 2>(a, t, grid, s);
            else launch_step<float, 1>(a, t, grid, s);
        }
        return check_launch(ctx, "gated_delta kernel");
    });
}

}  // extern "C"
