// kv_append.cu — a call's keys and values into a paged cache, the keys and the
// queries turned by their positions (include/strata_attention.h).
//
//   (a, b) -> (a cos x - b sin x, a sin x + b cos x),  x = p base^(-2 i / n)
//
// Bound by memory: each input is read and each result written once, three
// operations an element. A block takes a few tokens, computes their sines and
// cosines once for all heads and their places in the cache (both in shared memory);
// a thread then owns VEC pairs of one head (two packs of VEC elements where pairs are
// halves apart, one of 2 VEC where they are neighbours) and goes through the tokens,
// so that what a unit is takes its divisions once. Small blocks of few tokens, many
// of them side by side, keep loads under way while others compute angles: 8192 tokens
// of 32 + 8 + 8 heads of 128, f32 to bf16, 52 us, 5.8 TB/s (blocks of 256 threads with
// 13 tokens 65; a unit a thread at a time, with its divisions, 71). 64 single tokens 3.1 us.
// Where only single elements fit (20 of 80 elements turned, say) 8192 tokens of 48 heads of
// 80, bf16, take 171 us; with 40 turned, in packs of four, 59.
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"

namespace strata {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxTokensABlock = 6;
constexpr int kMaxTable = 128 * kMaxTokensABlock;  // pairs of sine and cosine in shared memory

struct AppendArgs {
    CacheArgs c;
    __nv_bfloat16* k_out;
    __nv_bfloat16* v_out;
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    int n_head, half;   // half: pairs that are turned
    int neighbours;
    int tokens;         // of a block
    int turners, turn_rows;  // threads that turn: so many pairs at once, for so many tokens
    double rate;        // -2 log2(base) / n_rot
};

// The sine and cosine of `turns` full turns: the whole turns leave in f64, the
// rest goes to f32 as its rounded value and what that lost (at most 2^-26 of a
// turn), whose sine is itself and whose cosine is 1 to below 2^-40.
__device__ __forceinline__ float2 sine_cosine(double turns) {
    const double rest = 2.0 * (turns - rint(turns));  // half turns, -1 to 1
    const float x = (float)rest, lost = (float)(rest - (double)x) * 3.14159274f;
    float s, c;
    sincospif(x, &s, &c);
    return make_float2(fmaf(lost, c, s), fmaf(-lost, s, c));
}

template <typename T, int N>
__device__ __forceinline__ void load(const void* base, int64_t at, float (&x)[N]) {
    const Pack<T, N> p = *reinterpret_cast<const Pack<T, N>*>(static_cast<const T*>(base) + at);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(p.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store(void* base, int64_t at, const float (&x)[N]) {
    Pack<T, N> p;
#pragma unroll
    for (int i = 0; i < N; ++i) from_f32(p.v[i], x[i]);
    *reinterpret_cast<Pack<T, N>*>(static_cast<T*>(base) + at) = p;
}

// TI, TQ: types of q, k, v and of q_out. VEC 8 or 4: rows, halves and buffers allow
// packs of so many elements; 1: element by element.
template <typename TI, typename TQ, int VEC, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads, 5) append_kernel(const AppendArgs a, const __grid_constant__ SeqTable tab) {
    __shared__ float2 turn[kMaxTable];
    __shared__ int64_t places[kMaxTokensABlock];  // of the tokens in the pools, head 0; -1: none
    const Seq seq = sequence_of_tile(tab, blockIdx.x);
    after_previous();
    const int t0 = (blockIdx.x - seq.tile0) * a.tokens, n = min(a.tokens, seq.len - t0);
    const int raw = a.c.len[seq.slot], p0 = (raw > 0 ? raw : 0) - seq.len + t0;  // the first token's position
    const int d = a.c.head_dim, kv = a.c.n_kv_head, reach = a.c.max_pages * a.c.page_size;
    if ((int)threadIdx.x < n) {
        const int p = p0 + threadIdx.x, page = p >= 0 && p < reach ? page_of(a.c, seq.slot, p) : -1;
        places[threadIdx.x] = page >= 0 ? place(a.c, page, p, 0) : -1;
    }
    // a thread its pairs, whose rate takes an f64 power once
    for (int pair = threadIdx.x % a.turners; pair < a.half && (int)threadIdx.x < a.turners * a.turn_rows; pair += a.turners) {
        const double rate = exp2(a.rate * (double)pair) * 0.15915494309189535;
        // a unit's pairs lie apart, neighbouring units' side by side: lanes read different banks
        const int at = pair % VEC * (a.half / VEC) + pair / VEC;
        for (int t = threadIdx.x / a.turners; t < n; t += a.turn_rows) turn[t * a.half + at] = sine_cosine((double)(p0 + t) * rate);
    }
    __syncthreads();
    // units of a head: first the turned pairs, then what stays, in packs; behind the heads of q and k those of v
    const int turned = a.half / VEC, units = turned + (d - 2 * a.half) / VEC, flat = d / VEC, split = (a.n_head + kv) * units;
    const int64_t row0 = seq.row + t0;
    for (int u = blockIdx.y * kThreads + threadIdx.x; u < split + kv * flat; u += kThreads * gridDim.y) {
        const bool is_v = u >= split;
        int head = is_v ? (u - split) / flat : u / units;
        const int unit = is_v ? (u - split) % flat : u % units;
        const bool is_q = !is_v && head < a.n_head, turns = !is_v && unit < turned;
        if (!is_v && !is_q) head -= a.n_head;
        const int64_t stride = is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride;
        const TI* in = static_cast<const TI*>(is_q ? a.q : is_v ? a.v : a.k) + row0 * stride + (int64_t)head * d;
        const int64_t out_stride = is_q ? a.q_out_stride : 0;
        TQ* out = static_cast<TQ*>(a.q_out) + (is_q ? row0 * a.q_out_stride + (int64_t)head * d : 0);
        __nv_bfloat16* const pool = (is_v ? a.v_out : a.k_out) + (int64_t)head * a.c.head_stride;
        // the unit's packs: e, and e2 for the other half
        const int e = is_v ? unit * VEC : !turns ? 2 * a.half + (unit - turned) * VEC : NEIGHBOURS ? unit * 2 * VEC : unit * VEC;
        const int e2 = e + (NEIGHBOURS ? VEC : a.half);
        constexpr int kAtOnce = 2;  // tokens under way
        for (int t = 0; t < n; t += kAtOnce, in += kAtOnce * stride, out += kAtOnce * out_stride) {
            float x[kAtOnce][VEC], y[kAtOnce][VEC];
#pragma unroll
            for (int w = 0; w < kAtOnce; ++w)
                if (t + w < n) {
                    load<TI>(in, w * stride + e, x[w]);
                    if (turns) load<TI>(in, w * stride + e2, y[w]);
                }
#pragma unroll
            for (int w = 0; w < kAtOnce; ++w) {
                if (t + w >= n) continue;
                if (turns) {
                    const float2* sc = turn + (t + w) * a.half + unit;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        // neighbours lie side by side in the two packs taken as one
                        float& f = NEIGHBOURS ? (2 * i < VEC ? x[w][2 * i % VEC] : y[w][2 * i % VEC]) : x[w][i];
                        float& b = NEIGHBOURS ? (2 * i + 1 < VEC ? x[w][(2 * i + 1) % VEC] : y[w][(2 * i + 1) % VEC]) : y[w][i];
                        const float2 r = sc[i * turned];
                        const float p = fmaf(f, r.y, -b * r.x), q = fmaf(f, r.x, b * r.y);
                        f = p, b = q;
                    }
                }
                if (is_q) {
                    store<TQ>(out, w * out_stride + e, x[w]);
                    if (turns) store<TQ>(out, w * out_stride + e2, y[w]);
                } else if (places[t + w] >= 0) {
                    store<__nv_bfloat16>(pool, places[t + w] + e, x[w]);
                    if (turns) store<__nv_bfloat16>(pool, places[t + w] + e2, y[w]);
                }
            }
        }
    }
}

template <typename TI, typename TQ, int VEC>
cudaError_t launch(dim3 grid, const AppendArgs& a, const SeqTable& t, cudaStream_t s) {
    if (a.neighbours) return launch_early(append_kernel<TI, TQ, VEC, true>, grid, kThreads, 0, s, a, t);
    return launch_early(append_kernel<TI, TQ, VEC, false>, grid, kThreads, 0, s, a, t);
}
template <typename TI, typename TQ>
cudaError_t launch(int vec, dim3 grid, const AppendArgs& a, const SeqTable& t, cudaStream_t s) {
    if (vec == 8) return launch<TI, TQ, 8>(grid, a, t, s);
    if (vec == 4) return launch<TI, TQ, 4>(grid, a, t, s);
    return launch<TI, TQ, 1>(grid, a, t, s);
}

}  // namespace
}  // namespace strata

using namespace strata;

extern "C" int strata_cuda_kv_append_dev(strata_ctx* ctx, const strata_kv_append* desc, const strata_kv_cache* cache,
                                         const void* q_dev, const void* k_dev, const void* v_dev, void* q_out_dev, void* stream) {
    if (!ctx || !desc || !cache) return STRATA_ERR_INVALID;
    STRATA_CALL_RANGE();
    std::lock_guard<std::mutex> g(ctx->mu);
    strata_kv_append d = *desc;
    strata_kv_cache c = *cache;
    Why why;
    int64_t tokens = 0, longest = 0;
    int rc = check_kv_append(why, d, c, &tokens, &longest);
    if (!rc && longest) rc = check_kv_append_buffers(why, d, c, tokens, q_dev, k_dev, v_dev, q_out_dev);
    if (rc) return fail(ctx, rc, "kv_append: %s", why.text);
    if (!longest) return STRATA_OK;
    AppendArgs a = {};
    a.c = cache_args(c);
    a.k_out = static_cast<__nv_bfloat16*>(c.k_dev), a.v_out = static_cast<__nv_bfloat16*>(c.v_dev);
    a.q = q_dev, a.k = k_dev, a.v = v_dev, a.q_out = q_out_dev;
    a.q_stride = d.q_stride, a.k_stride = d.k_stride, a.v_stride = d.v_stride, a.q_out_stride = d.q_out_stride;
    a.n_head = (int)d.n_head, a.half = (int)d.n_rot / 2, a.neighbours = d.neighbours;
    a.rate = d.n_rot ? -2.0 * std::log2(d.freq_base) / (double)d.n_rot : 0.0;
    a.turners = std::min(std::max(a.half, 1), kThreads), a.turn_rows = kThreads / a.turners;
    // one token a block where there are few, more (and their sines once) where there are many
    const int64_t fill = 4 * (int64_t)ctx->sm_count;
    a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxTokensABlock, tokens / fill));
    const int64_t size = dtype_bytes(d.dtype), out = dtype_bytes(d.q_dtype);
    const bool wide = ((uintptr_t)k_dev | (uintptr_t)v_dev) % 16 == 0 && (d.k_stride * size) % 16 == 0 && (d.v_stride * size) % 16 == 0 &&
                      (!d.n_head || (((uintptr_t)q_dev | (uintptr_t)q_out_dev) % 16 == 0 && (d.q_stride * size) % 16 == 0 && (d.q_out_stride * out) % 16 == 0));
    const int vec = !wide ? 1 : a.half % 8 == 0 ? 8 : a.half % 4 == 0 ? 4 : 1;
    DeviceGuard dev(ctx->device);
    const cudaStream_t s = pick_stream(ctx, stream);
    const bool bi = d.dtype == STRATA_QUANT_BF16, bq = d.q_dtype == STRATA_QUANT_BF16;
    return for_sequence_groups(d.n_seq, d.seq_len, d.seq_offsets, a.tokens, tokens + 1, [&](const SeqTable& t, int64_t tiles) {
        if (tiles > kMaxTokens) return fail(ctx, STRATA_ERR_INVALID, "kv_append: %lld tiles", (long long)tiles);
        const int64_t share = std::max<int64_t>(1, std::min<int64_t>(4, fill / tiles));
        const dim3 grid((unsigned)tiles, (unsigned)share);
        const cudaError_t e = bi && bq ? launch<__nv_bfloat16, __nv_bfloat16>(vec, grid, a, t, s)
                              : bi     ? launch<__nv_bfloat16, float>(vec, grid, a, t, s)
                              : bq     ? launch<float, __nv_bfloat16>(vec, grid, a, t, s)
                                       : launch<float, float>(vec, grid, a, t, s);
        return e == cudaSuccess ? STRATA_OK : cuda_fail(ctx, e, "kv_append kernel");
    });
}
