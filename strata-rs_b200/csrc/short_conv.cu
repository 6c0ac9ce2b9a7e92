// short_conv.cu — causal depthwise convolution of a recurrent layer's
// projected channels, with its state (the step before the gated delta rule;
// the reference's loop is in crates/strata-core/src/gdn.rs).
//
//   y[t][c] = act(bias[c] + sum_j w[c][j] x[t - (K - 1) + j][c])
//
// Bound by memory: each x is read and each y written once, 2 K flops between
// them. A thread owns VEC neighbouring channels (one 16-byte access) and walks
// a tile of tokens with the last K - 1 inputs in registers, so a tile re-reads
// only its K - 1 rows of halo (from L2). Rows come kAhead at a time: 16-byte
// packs by asynchronous copies into shared memory, three batches ahead and
// without holding registers (each lane copies and reads its own packs, so
// nothing has to be waited for but its own copies); odd shapes element-wise
// into registers, one batch ahead. Tiles are as long as a full GPU allows
// (their weights and halo are then a small part), one token where sequences
// have one.
//
// Measured: 8192 tokens of 8192 bf16 channels, 4 taps, 49 us, 5.5 TB/s (the
// asynchronous copies took it from 111 to 65, tiles for two whole rounds of
// blocks from there; SiLU's exponential and reciprocal keep the special-function
// unit 58% busy); 64
// sequences of one token 5.1 us, launch and latency; 3537
// tokens of 8 sequences, 2571 f32 channels element by element, 18 us.
//
// The state of a sequence is read and replaced by the same thread (the one
// that has its first tile; the new state is the sequence's last K - 1 inputs,
// read again from x), so no other block has to be waited for.
#include <cuda_runtime.h>

#include "sequence.cuh"

namespace strata {
namespace {

constexpr int kMinTile = 8, kMaxTile = 64;  // tokens of a tile; at least the longest halo
constexpr int kThreads = 128;
constexpr int kRingBatches = 4;

struct ConvArgs {
    const void* x;
    const float* w;
    const float* bias;
    float* state;
    void* y;
    int64_t x_stride, y_stride;
    int channels, blocks;  // blocks of channels
    int tile;
    int silu;
    int wide_w;            // w can be read in 16-byte packs
};

// z / (1 + exp(-z)). For bf16 outputs the approximate exponential (its
// argument rounds, 2^-24 |z| of the result) and reciprocal (1 ulp) are far below
// the rounding; f32 outputs take the accurate exponential. The quick division
// is good to 2 ulp, and gives 0 where exp(-z) > 2^126 (the true value is below
// 1e-36).
template <typename T>
__device__ __forceinline__ float silu(float z) {
    if (sizeof(T) == 2) {
        float e, r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
        return z * r;
    }
    return __fdividef(z, 1.0f + expf(-z));
}

// Blocks a multiprocessor runs side by side (up to four taps), as their registers
// allow without spilling: a fifth of eight channels for a few tokens costs 128
// bytes of them a thread (64 single bf16 tokens of 8192 channels 8.1 us, not 7.4,
// 512 of them 45, not 40).
constexpr int resident(int vec, bool few) { return vec == 8 ? 4 : vec == 4 && !few ? 6 : 8; }

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& p, float (&d)[VEC]) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) d[v] = to_f32(p.v[v]);
}

// SHORT: for sequences of a few tokens, where registers spent on reading ahead
// would only keep blocks from running side by side.
template <typename T, int K, int VEC, bool SHORT>
__global__ void __launch_bounds__(kThreads, K <= 4 ? resident(VEC, SHORT) : 1)
    conv_kernel(const ConvArgs a, const __grid_constant__ SeqTable tab) {
    constexpr int kAhead = SHORT ? 1 : VEC == 1 ? 8 : 4;
    const int block = blockIdx.x / a.blocks;
    const int c = ((blockIdx.x - block * a.blocks) * kThreads + threadIdx.x) * VEC;
    if (c >= a.channels) return;
    const Seq seq = sequence_of_tile(tab, block);
    const int row = seq.row, len = seq.len, t0 = (block - seq.tile0) * a.tile;
    const int n = len - t0 < a.tile ? len - t0 : a.tile;
    const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.x_stride + c;
    T* y = static_cast<T*>(a.y) + (int64_t)(row + t0) * a.y_stride + c;
    using P = Pack<T, VEC>;
    using F = Pack<float, VEC>;

    constexpr bool kRing = VEC > 1 && !SHORT;
    __shared__ P ring[kRing ? kRingBatches * kAhead : 1][kRing ? kThreads : 1];
    P now[kAhead], next[kAhead];
    // Brings in the rows from t on: into `in`, or batch t / kAhead of the ring.
    auto load = [&](P(&in)[kAhead], int t) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const T* p = x + (int64_t)(t0 + t + u) * a.x_stride;
            if (t + u < n) {
                if (kRing)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((uint32_t)__cvta_generic_to_shared(
                                     &ring[kRing ? (t + u) % (kRingBatches * kAhead) : 0][kRing ? threadIdx.x : 0])),
                                 "l"(p)
                                 : "memory");
                else
                    in[u] = *reinterpret_cast<const P*>(p);
            }
        }
        if (kRing) asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    load(now, 0);
    if (kRing)
#pragma unroll
        for (int q = 1; q < kRingBatches - 1; ++q) load(now, q * kAhead);
    float w[K][VEC], past[K][VEC];  // past[0 .. K-2]: the inputs before the tile (one spare row keeps K = 1 legal)
    if (K == 4 && a.wide_w) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float4 q = *reinterpret_cast<const float4*>(a.w + (int64_t)(c + v) * 4);
            w[0][v] = q.x, w[K > 1 ? 1 : 0][v] = q.y, w[K > 2 ? 2 : 0][v] = q.z, w[K > 3 ? 3 : 0][v] = q.w;
        }
    } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
#pragma unroll
            for (int j = 0; j < K; ++j) w[j][v] = a.w[(int64_t)(c + v) * K + j];
    }
    float bias[VEC] = {};
    if (a.bias) unpack<float, VEC>(*reinterpret_cast<const F*>(a.bias + c), bias);
    if (K > 1) {
        float* st = a.state + (int64_t)seq.slot * (K - 1) * a.channels + c;
        if (t0 == 0) {
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
                unpack<float, VEC>(*reinterpret_cast<const F*>(st + (int64_t)j * a.channels), past[j]);
            // the new state: input len - (K - 1) + j, or where that is before the
            // call, old row len + j, which lies behind row j and is not yet replaced
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                const int p = len - (K - 1) + j;
                F out;
                if (p >= 0) unpack<T, VEC>(*reinterpret_cast<const P*>(x + (int64_t)p * a.x_stride), out.v);
                else out = *reinterpret_cast<const F*>(st + (int64_t)(len + j) * a.channels);
                *reinterpret_cast<F*>(st + (int64_t)j * a.channels) = out;
            }
        } else {  // t0 >= kMinTile > K - 1: the halo lies inside the sequence
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
                unpack<T, VEC>(*reinterpret_cast<const P*>(x + (int64_t)(t0 - (K - 1) + j) * a.x_stride), past[j]);
        }
    }
    for (int t = 0; t < n; t += kAhead) {
        load(next, t + (kRing ? kRingBatches - 1 : 1) * kAhead);
        if (kRing) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(kRingBatches - 1) : "memory");
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                now[u] = ring[kRing ? (t + u) % (kRingBatches * kAhead) : 0][kRing ? threadIdx.x : 0];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            P out;
            float in[VEC];
            unpack<T, VEC>(now[u], in);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float z = bias[v];
#pragma unroll
                for (int j = 0; j < K - 1; ++j) z = fmaf(w[j][v], past[j][v], z);
                z = fmaf(w[K - 1][v], in[v], z);
#pragma unroll
                for (int j = 0; j + 1 < K - 1; ++j) past[j][v] = past[j + 1][v];
                if (K > 1) past[K >= 2 ? K - 2 : 0][v] = in[v];
                from_f32(out.v[v], a.silu ? silu<T>(z) : z);
            }
            if (t + u < n) *reinterpret_cast<P*>(y + u * a.y_stride) = out;
        }
        y += kAhead * a.y_stride;
        if (!kRing)
#pragma unroll
            for (int u = 0; u < kAhead; ++u) now[u] = next[u];
    }
}

template <typename T, int VEC, bool SHORT>
void launch_conv(int taps, const ConvArgs& a, const SeqTable& t, unsigned grid, cudaStream_t s) {
    switch (taps) {
        case 1: conv_kernel<T, 1, VEC, SHORT><<<grid, kThreads, 0, s>>>(a, t); break;
        case 2: conv_kernel<T, 2, VEC, SHORT><<<grid, kThreads, 0, s>>>(a, t); break;
        case 3: conv_kernel<T, 3, VEC, SHORT><<<grid, kThreads, 0, s>>>(a, t); break;
        case 4: conv_kernel<T, 4, VEC, SHORT><<<grid, kThreads, 0, s>>>(a, t); break;
        case 5: conv_kernel<T, 5, VEC, SHORT><<<grid, kThreads, 0, s>>>(a, t); break;
        case 6: conv_kernel<T, 6, VEC, SHORT><<<grid, kThreads, 0, s>>>(a, t); break;
        case 7: conv_kernel<T, 7, VEC, SHORT><<<grid, kThreads, 0, s>>>(a, t); break;
        default: conv_kernel<T, 8, VEC, SHORT><<<grid, kThreads, 0, s>>>(a, t); break;
    }
}
template <typename T, int VEC>
void launch_conv(bool few, int taps, const ConvArgs& a, const SeqTable& t, unsigned grid, cudaStream_t s) {
    if (few) launch_conv<T, VEC, true>(taps, a, t, grid, s);
    else launch_conv<T, VEC, false>(taps, a, t, grid, s);
}

// The 16-byte form needs whole packs in every row and 16-byte rows.
bool packs(const strata_short_conv& d, const void* x, const void* y, const float* bias, const float* state) {
    const int64_t vec = 16 / dtype_bytes(d.dtype);
    return d.channels % vec == 0 && d.x_stride % vec == 0 && d.y_stride % vec == 0 &&
           ((uintptr_t)x | (uintptr_t)y | (uintptr_t)bias | (uintptr_t)state) % 16 == 0;
}

}  // namespace
}  // namespace strata

using namespace strata;

extern "C" int strata_cuda_short_conv_dev(strata_ctx* ctx, const strata_short_conv* desc, const void* x_dev,
                                          const float* w_dev, const float* bias_dev, float* state_dev, void* y_dev,
                                          void* stream) {
    if (!ctx || !desc) return STRATA_ERR_INVALID;
    STRATA_CALL_RANGE();
    std::lock_guard<std::mutex> g(ctx->mu);
    strata_short_conv d = *desc;
    Why why;
    int64_t tokens = 0, longest = 0;
    int rc = check_short_conv(why, d, &tokens, &longest);
    if (!rc && longest > 0) rc = check_short_conv_buffers(why, d, tokens, x_dev, w_dev, bias_dev, state_dev, y_dev);
    if (rc) return fail(ctx, rc, "short_conv: %s", why.text);
    if (longest == 0) return STRATA_OK;
    const bool bf16 = d.dtype == STRATA_QUANT_BF16, vec = packs(d, x_dev, y_dev, bias_dev, state_dev);
    const int64_t per = (int64_t)kThreads * (vec ? (bf16 ? 8 : 4) : 1);
    const int64_t blocks = (d.channels + per - 1) / per;
    // tiles for two whole rounds of the blocks that run side by side
    const int64_t at_once = 2 * (int64_t)ctx->sm_count * resident(vec ? (bf16 ? 8 : 4) : 1, false);
    const int64_t share = at_once / blocks > 0 ? at_once / blocks : 1;
    const int64_t fit = (tokens + share - 1) / share;
    const bool few = longest <= 4;
    const int64_t tile = fit < kMinTile ? kMinTile : fit > kMaxTile ? kMaxTile : fit;
    const ConvArgs a{x_dev, w_dev, bias_dev, state_dev, y_dev, d.x_stride, d.y_stride, (int)d.channels, (int)blocks,
                     (int)tile, d.silu, (uintptr_t)w_dev % 16 == 0};
    DeviceGuard dev(ctx->device);
    const cudaStream_t s = pick_stream(ctx, stream);
    return for_sequence_groups(d.n_seq, d.seq_len, d.seq_offsets, tile, tokens + 1, [&](const SeqTable& t, int64_t tiles) {
        if (tiles * a.blocks > kMaxTokens)
            return fail(ctx, STRATA_ERR_INVALID, "short_conv: %lld tiles of %d channel blocks", (long long)tiles,
                        a.blocks);
        const unsigned grid = (unsigned)(tiles * a.blocks);
        if (bf16 && vec) launch_conv<__nv_bfloat16, 8>(few, (int)d.taps, a, t, grid, s);
        else if (bf16) launch_conv<__nv_bfloat16, 1>(few, (int)d.taps, a, t, grid, s);
        else if (vec) launch_conv<float, 4>(few, (int)d.taps, a, t, grid, s);
        else launch_conv<float, 1>(few, (int)d.taps, a, t, grid, s);
        return check_launch(ctx, "short_conv kernel");
    });
}
