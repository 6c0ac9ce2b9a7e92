// kv_append.cu — a call's keys and values into a paged cache, the keys and the
// queries turned by their positions (include/strata_attention.h).
//
//   (a, b) -> (a cos x - b sin x, a sin x + b cos x),  x = p base^(-2 i / n)
//
// Bound by memory: each input is read and each result written once, three
// operations an element. A block takes a few tokens, computes their sines and
// cosines once for all heads (in shared memory), and then walks the tokens'
// heads, VEC pairs of one head a thread: two packs of VEC elements where pairs
// are halves apart, one pack of 2 VEC where they are neighbours.
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"

namespace strata {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTable = 4096;  // pairs of sine and cosine in shared memory

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

// TI, TQ: types of q, k, v and of q_out. VEC 4: rows, halves and buffers allow
// packs of four elements; 1: element by element.
template <typename TI, typename TQ, int VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a, const __grid_constant__ SeqTable tab) {
    __shared__ float2 turn[kMaxTable];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Seq seq = sequence_of_tile(tab, blockIdx.x);
    const int t0 = (blockIdx.x - seq.tile0) * a.tokens, n = min(a.tokens, seq.len - t0);
    const int raw = a.c.len[seq.slot], p0 = (raw > 0 ? raw : 0) - seq.len + t0;  // the first token's position
    const int d = a.c.head_dim, kv = a.c.n_kv_head, reach = a.c.max_pages * a.c.page_size;
    for (int i = threadIdx.x; i < n * a.half; i += kThreads) {
        const int t = i / a.half, pair = i - t * a.half;
        turn[i] = sine_cosine((double)(p0 + t) * exp2(a.rate * (double)pair) * 0.15915494309189535);
    }
    __syncthreads();
    // units of a head: first the turned pairs, then what stays, in packs
    const int turned = a.half / VEC, rest = (d - 2 * a.half) / VEC, units = turned + rest, flat = d / VEC;
    const int per_token = (a.n_head + kv) * units + kv * flat;
    for (int i = blockIdx.y * kThreads + threadIdx.x; i < n * per_token; i += kThreads * gridDim.y) {
        const int t = i / per_token;
        int u = i - t * per_token;
        const int row = seq.row + t0 + t, p = p0 + t;
        const bool is_v = u >= (a.n_head + kv) * units;
        int head, unit;
        if (is_v) {
            u -= (a.n_head + kv) * units;
            head = u / flat, unit = u - head * flat;
        } else {
            head = u / units, unit = u - head * units;
        }
        const bool is_q = !is_v && head < a.n_head;
        int64_t out = 0;
        if (is_q) {
            out = (int64_t)row * a.q_out_stride + (int64_t)head * d;
        } else {
            if (!is_v) head -= a.n_head;
            if (p < 0 || p >= reach) continue;
            const int page = page_of(a.c, seq.slot, p);
            if (page < 0) continue;
            out = place(a.c, page, p, head);
        }
        const void* in = is_q ? a.q : is_v ? a.v : a.k;
        const int64_t at = (int64_t)row * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + (int64_t)head * d;
        auto put = [&](int e, const auto& x) {
            if (is_q) store<TQ>(a.q_out, out + e, x);
            else store<__nv_bfloat16>(is_v ? a.v_out : a.k_out, out + e, x);
        };
        if (is_v || unit >= turned) {
            float x[VEC];
            const int e = is_v ? unit * VEC : 2 * a.half + (unit - turned) * VEC;
            load<TI>(in, at + e, x);
            put(e, x);
            continue;
        }
        const float2* sc = turn + t * a.half + unit * VEC;
        if (a.neighbours) {
            // element by element rows lie anywhere: a pair is then two accesses
            constexpr int kPack = VEC == 1 ? 1 : 2 * VEC;
            float x[2 * VEC / kPack][kPack];
            const int e = unit * 2 * VEC;
#pragma unroll
            for (int w = 0; w < 2 * VEC / kPack; ++w) load<TI>(in, at + e + w, x[w]);
            float* const pairs = &x[0][0];
#pragma unroll
            for (int w = 0; w < VEC; ++w) {
                const float f = pairs[2 * w], b = pairs[2 * w + 1];
                pairs[2 * w] = fmaf(f, sc[w].y, -b * sc[w].x), pairs[2 * w + 1] = fmaf(f, sc[w].x, b * sc[w].y);
            }
#pragma unroll
            for (int w = 0; w < 2 * VEC / kPack; ++w) put(e + w, x[w]);
        } else {
            float x[VEC], y[VEC];
            load<TI>(in, at + unit * VEC, x);
            load<TI>(in, at + a.half + unit * VEC, y);
#pragma unroll
            for (int w = 0; w < VEC; ++w) {
                const float f = x[w], b = y[w];
                x[w] = fmaf(f, sc[w].y, -b * sc[w].x), y[w] = fmaf(f, sc[w].x, b * sc[w].y);
            }
            put(unit * VEC, x);
            put(a.half + unit * VEC, y);
        }
    }
}

template <typename TI, typename TQ>
void launch(bool wide, dim3 grid, const AppendArgs& a, const SeqTable& t, cudaStream_t s) {
    if (wide) append_kernel<TI, TQ, 4><<<grid, kThreads, 0, s>>>(a, t);
    else append_kernel<TI, TQ, 1><<<grid, kThreads, 0, s>>>(a, t);
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
    // one token a block where there are few, more (and their sines once) where there are many
    const int64_t most = a.half ? kMaxTable / a.half : 64;
    const int64_t fill = 4 * (int64_t)ctx->sm_count;
    a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>({most, 16, tokens / fill}));
    const int64_t size = dtype_bytes(d.dtype), out = dtype_bytes(d.q_dtype);
    const bool wide = a.half % 4 == 0 && ((uintptr_t)k_dev | (uintptr_t)v_dev) % 16 == 0 && (d.k_stride * size) % 16 == 0 &&
                      (d.v_stride * size) % 16 == 0 &&
                      (!d.n_head || (((uintptr_t)q_dev | (uintptr_t)q_out_dev) % 16 == 0 && (d.q_stride * size) % 16 == 0 && (d.q_out_stride * out) % 16 == 0));
    DeviceGuard dev(ctx->device);
    const cudaStream_t s = pick_stream(ctx, stream);
    const bool bi = d.dtype == STRATA_QUANT_BF16, bq = d.q_dtype == STRATA_QUANT_BF16;
    return for_sequence_groups(d.n_seq, d.seq_len, d.seq_offsets, a.tokens, tokens + 1, [&](const SeqTable& t, int64_t tiles) {
        if (tiles > kMaxTokens) return fail(ctx, STRATA_ERR_INVALID, "kv_append: %lld tiles", (long long)tiles);
        const int64_t share = std::max<int64_t>(1, std::min<int64_t>(4, fill / tiles));
        const dim3 grid((unsigned)tiles, (unsigned)share);
        if (bi && bq) launch<__nv_bfloat16, __nv_bfloat16>(wide, grid, a, t, s);
        else if (bi) launch<__nv_bfloat16, float>(wide, grid, a, t, s);
        else if (bq) launch<float, __nv_bfloat16>(wide, grid, a, t, s);
        else launch<float, float>(wide, grid, a, t, s);
        return check_launch(ctx, "kv_append kernel");
    });
}
