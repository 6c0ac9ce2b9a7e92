// logprobs.cu — log-probabilities of given tokens, entropies and the likeliest
// tokens of rows of logits (include/strata_attention.h).
//
//   Z = sum_j exp(x_j - M), log p_i = x_i - M - log Z, H = log Z - sum_j e_j (x_j - M) / Z
//
// One pass over the row for M, Z and sum e_j (x_j - M), each thread with a
// running maximum of its own; Z is summed in f64, because next to a certain
// token it is 1 and a little, and log Z is that little. The threads' maxima are
// what the likeliest tokens are found by: the n-th largest of them, T, is a lower
// bound of the n-th largest logit, and only threads whose maximum reaches T can
// have seen one of the n: their logits (one in kThreads each) are read again, and
// those that reach T are ordered by counting.
//
// Bound by memory where rows are many (one block a row); few rows are cut over a
// cluster of blocks, whose results the first one joins.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"

namespace strata {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kTop = (int)kMaxTop;
constexpr int kCand = 1024;     // candidates that are ordered at once
constexpr int kMaxCluster = 8;
constexpr int kAhead = 4;       // 16-byte packs a thread has under way

struct LogprobArgs {
    const float* logits;
    int64_t stride;
    int vocab, top;
    const int* targets;
    float* logprobs;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
};

// What a thread, a block or a row has seen: the largest logit, sum e^(x - max) and sum e^(x - max) (x - max).
struct Sum {
    float max;
    double z, zd;
};
__device__ __forceinline__ void rescale(Sum& s, float max) {  // max >= s.max
    if (s.max == max) return;
    if (s.max == -INFINITY) {
        s.z = s.zd = 0.0;
    } else {
        const double down = (double)s.max - (double)max, f = exp(down);
        s.zd = f * (s.zd + down * s.z);
        s.z *= f;
    }
    s.max = max;
}
__device__ __forceinline__ void join(Sum& a, Sum b) {
    const float max = fmaxf(a.max, b.max);
    rescale(a, max), rescale(b, max);
    a.z += b.z, a.zd += b.zd;
}
__device__ __forceinline__ Sum shuffled(const Sum& s, int w) {
    return {__shfl_xor_sync(0xFFFFFFFFu, s.max, w), __shfl_xor_sync(0xFFFFFFFFu, s.z, w), __shfl_xor_sync(0xFFFFFFFFu, s.zd, w)};
}

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }  // a NaN counts as -inf
__device__ __forceinline__ float exp_of(float d) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * 1.4426950408889634f));
    return y;
}
// N logits more. zd is summed in f32 within them: its terms never meet the 1 of the largest.
template <int N>
__device__ __forceinline__ void add(Sum& s, const float (&x)[N]) {
    float max = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) max = fmaxf(max, x[i]);
    if (max > s.max) rescale(s, max);
    if (s.max == -INFINITY) return;
    float zd = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = fmaxf(x[i] - s.max, -200.0f);  // below e^-200 is nothing, and -inf * 0 is none
        const float e = exp_of(d);
        s.z += (double)e;
        zd = fmaf(e, d, zd);
    }
    s.zd += (double)zd;
}

struct Cand {
    float x;
    int id;
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.x > b.x || (a.x == b.x && a.id < b.id); }

// The first n of m candidates in order, into out (all threads; m up to kCand).
__device__ void order_by_counting(const Cand* in, int m, int n, Cand* out) {
    for (int i = threadIdx.x; i < m; i += kThreads) {
        const Cand c = in[i];
        int rank = 0;
        for (int j = 0; j < m; ++j) rank += before(in[j], c);
        if (rank < n) out[rank] = c;
    }
}

// PACKS: rows are 16-byte aligned and read in packs of four.
template <bool PACKS>
__global__ void __launch_bounds__(kThreads, 2) logprobs_kernel(const LogprobArgs a, int cluster) {
    __shared__ float maxima[kThreads];
    __shared__ Cand cand[kCand];
    __shared__ Cand best[kTop];             // of this block
    __shared__ Cand all[kMaxCluster * kTop], final[kTop];
    __shared__ Sum part[kWarps], sums[kMaxCluster];
    __shared__ int n_cand, infinite;
    __shared__ unsigned long long pick[kWarps];
    const int rank = cluster > 1 ? blockIdx.x % cluster : 0;
    const int64_t row = blockIdx.x / cluster;
    const float* x = a.logits + row * a.stride;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // this block's share, in whole rounds of the block's packs
    constexpr int kStep = kThreads * (PACKS ? 4 : 1);
    const int rounds = (a.vocab + kStep - 1) / kStep;
    const int r0 = (int)((int64_t)rounds * rank / cluster), r1 = (int)((int64_t)rounds * (rank + 1) / cluster);
    const int begin = r0 * kStep, end = min(r1 * kStep, a.vocab);
    // arrive here, wait before the first remote write: the first block then runs
    if (cluster > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    if (threadIdx.x == 0) n_cand = 0, infinite = 0;
    if (threadIdx.x < kTop) best[threadIdx.x] = Cand{-INFINITY, -1}, final[threadIdx.x] = Cand{-INFINITY, -1};

    // ---- the pass
    Sum s = {-INFINITY, 0.0, 0.0};
    if (PACKS) {
        const int whole = end - (end & 3);
        int i = begin + threadIdx.x * 4;
        for (; i + (kAhead - 1) * kStep < whole; i += kAhead * kStep) {
            float v[4 * kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float4 p = __ldcs(reinterpret_cast<const float4*>(x + i + u * kStep));
                v[4 * u] = clean(p.x), v[4 * u + 1] = clean(p.y), v[4 * u + 2] = clean(p.z), v[4 * u + 3] = clean(p.w);
            }
            add(s, v);
        }
        for (; i < whole; i += kStep) {
            const float4 p = __ldcs(reinterpret_cast<const float4*>(x + i));
            const float v[4] = {clean(p.x), clean(p.y), clean(p.z), clean(p.w)};
            add(s, v);
        }
        if (threadIdx.x < end - whole) {  // what is no pack, by the threads of lowest number
            const float v[1] = {clean(x[whole + threadIdx.x])};
            add(s, v);
        }
    } else {
        for (int i = begin + threadIdx.x; i < end; i += kAhead * kStep) {
            float v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) v[u] = i + u * kStep < end ? clean(__ldcs(x + i + u * kStep)) : -INFINITY;
            add(s, v);
        }
    }
    maxima[threadIdx.x] = s.max;
    const float own = s.max;
    for (int w = 16; w; w >>= 1) join(s, shuffled(s, w));
    if (lane == 0) part[warp] = s;
    __syncthreads();

    // ---- this block's likeliest
    if (a.top && begin < end) {
        // how many threads' maxima come before this one's, threads' numbers settling ties
        int ahead = 0;
        for (int j = 0; j < kThreads; ++j) {
            const float m = maxima[j];
            ahead += m > own || (m == own && j < (int)threadIdx.x);
        }
        __shared__ float bound;
        if (ahead == a.top - 1) bound = own;
        __syncthreads();
        const float t = bound;
        auto offer = [&](int i) {
            const float v = clean(x[i]);
            if (v >= t && v > -INFINITY) {
                const int at = atomicAdd(&n_cand, 1);
                if (at < kCand) cand[at] = Cand{v, i};
            }
        };
        if (own >= t && own > -INFINITY) {
            if (PACKS) {
                const int whole = end - (end & 3);
                for (int i = begin + threadIdx.x * 4; i < whole; i += kStep)
                    for (int u = 0; u < 4; ++u) offer(i + u);
                if (threadIdx.x < end - whole) offer(whole + threadIdx.x);
            } else {
                for (int i = begin + threadIdx.x; i < end; i += kStep) offer(i);
            }
        }
        __syncthreads();
        if (n_cand <= kCand) {
            order_by_counting(cand, n_cand, a.top, best);
        } else {
            // more logits reach T than are ordered at once (thousands of equal ones, or large
            // ones all in one thread's share): the best behind the last, one after another
            Cand last = {INFINITY, -1};
            for (int n = 0; n < a.top; ++n) {
                // the order as one number: the float's bits made to rise with it, then the lowest index
                unsigned long long mine = 0;
                for (int i = begin + threadIdx.x; i < end; i += kThreads) {
                    const float v = clean(x[i]);
                    if (v < t || v == -INFINITY) continue;
                    const Cand c = {v, i};
                    if (n && !before(last, c)) continue;
                    const unsigned bits = __float_as_uint(v + 0.0f);
                    const unsigned key = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
                    mine = max(mine, (unsigned long long)key << 32 | (unsigned)~i);
                }
                for (int w = 16; w; w >>= 1) mine = max(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, w));
                __syncthreads();
                if (lane == 0) pick[warp] = mine;
                __syncthreads();
                for (int w = 0; w < kWarps; ++w) mine = max(mine, pick[w]);
                if (!mine) break;
                const int id = (int)~(unsigned)mine;
                last = Cand{clean(x[id]), id};
                if (threadIdx.x == 0) best[n] = last;
            }
        }
        __syncthreads();
    }

    // ---- the blocks of the row joined by the first
    Sum total = {-INFINITY, 0.0, 0.0};
    if (warp == 0) {
        Sum v = lane < kWarps ? part[lane] : Sum{-INFINITY, 0.0, 0.0};
        for (int w = 16; w; w >>= 1) join(v, shuffled(v, w));
        total = v;
    }
    const Cand* list = best;
    if (cluster > 1) {
        cg::cluster_group cl = cg::this_cluster();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (threadIdx.x == 0) *cl.map_shared_rank(&sums[rank], 0) = total;
        if ((int)threadIdx.x < a.top) cl.map_shared_rank(all, 0)[rank * a.top + threadIdx.x] = best[threadIdx.x];
        cl.sync();
        if (rank) return;
        if (warp == 0) {
            Sum v = lane < cluster ? sums[lane] : Sum{-INFINITY, 0.0, 0.0};
            for (int w = 16; w; w >>= 1) join(v, shuffled(v, w));
            total = v;
        }
        // the blanks' ids of -1 would come first among equals: none of -inf is taken
        if (a.top) {
            for (int i = threadIdx.x; i < cluster * a.top; i += kThreads) {
                const Cand c = all[i];
                int place = 0;
                for (int j = 0; j < cluster * a.top; ++j) place += before(all[j], c);
                if (place < a.top && c.x > -INFINITY) final[place] = c;
            }
            list = final;
        }
        __syncthreads();
    }
    __shared__ Sum result;
    if (threadIdx.x == 0) result = total;
    __syncthreads();
    total = result;
    if (total.max == INFINITY) {  // infinite logits share everything: counted
        int n = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) n += x[i] == INFINITY;
        atomicAdd(&infinite, n);
        __syncthreads();
        total.z = infinite, total.zd = 0.0;
    }
    const double logz = total.z > 0.0 ? log(total.z) : 0.0;
    auto log_p = [&](float v) -> float {
        if (total.max == -INFINITY || v == -INFINITY) return -INFINITY;
        if (total.max == INFINITY) return v == INFINITY ? (float)-logz : -INFINITY;
        return (float)((double)v - (double)total.max - logz);
    };
    if (threadIdx.x == 0) {
        if (a.logprobs) {
            const int id = a.targets[row];
            a.logprobs[row] = id >= 0 && id < a.vocab ? log_p(clean(x[id])) : 0.0f;
        }
        if (a.entropy) a.entropy[row] = total.max == -INFINITY ? 0.0f : (float)(logz - total.zd / total.z);
    }
    if ((int)threadIdx.x < a.top) {
        const Cand c = list[threadIdx.x];
        const bool none = c.x == -INFINITY;
        a.top_ids[row * a.top + threadIdx.x] = none ? -1 : c.id;
        a.top_logprobs[row * a.top + threadIdx.x] = none ? -INFINITY : log_p(c.x);
    }
}

}  // namespace
}  // namespace strata

using namespace strata;

extern "C" int strata_cuda_logprobs_dev(strata_ctx* ctx, const float* logits_dev, int64_t rows, int64_t vocab, int64_t stride,
                                        const int32_t* targets_dev, float* logprobs_dev, float* entropy_dev, int64_t top,
                                        int32_t* top_ids_dev, float* top_logprobs_dev, void* stream) {
    if (!ctx) return STRATA_ERR_INVALID;
    STRATA_CALL_RANGE();
    std::lock_guard<std::mutex> g(ctx->mu);
    Why why;
    const int rc = check_logprobs(why, logits_dev, rows, vocab, stride, targets_dev, logprobs_dev, entropy_dev, top, top_ids_dev, top_logprobs_dev);
    if (rc) return fail(ctx, rc, "logprobs: %s", why.text);
    if (rows == 0) return STRATA_OK;
    const LogprobArgs a{logits_dev, stride, (int)vocab, (int)top, targets_dev, logprobs_dev, entropy_dev, top_ids_dev, top_logprobs_dev};
    const bool packs = (uintptr_t)logits_dev % 16 == 0 && stride % 4 == 0;
    // a cluster a row while that leaves multiprocessors to every block, and a share worth a block
    int cluster = 1;
    while (cluster < kMaxCluster && rows * cluster * 2 <= ctx->sm_count && vocab >= (int64_t)cluster * 2 * kThreads * 4) cluster *= 2;
    DeviceGuard dev(ctx->device);
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cluster, at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster)), cfg.blockDim = dim3(kThreads), cfg.stream = pick_stream(ctx, stream);
    cfg.attrs = &at, cfg.numAttrs = cluster > 1 ? 1 : 0;
    const cudaError_t e = packs ? cudaLaunchKernelEx(&cfg, logprobs_kernel<true>, a, cluster) : cudaLaunchKernelEx(&cfg, logprobs_kernel<false>, a, cluster);
    return e == cudaSuccess ? STRATA_OK : cuda_fail(ctx, e, "logprobs kernel");
}
