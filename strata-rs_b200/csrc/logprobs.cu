// logprobs.cu — log-probabilities of given tokens, entropies and the likeliest
// tokens of rows of logits (include/strata_attention.h).
//
//   Z = sum_j exp(x_j - M), log p_i = x_i - M - log Z, H = log Z - sum_j e_j (x_j - M) / Z
//
// One pass over the row for M, Z and sum e_j (x_j - M), each thread with a
// running maximum of its own. Next to a certain token Z is 1 and a little, and
// log Z is that little: so a batch's maximum is found by a tournament, whose
// losers (which never hold the 1) are summed in f32 and whose winner apart, and
// both go to an f64 sum. The threads' maxima are what the likeliest tokens are
// found by: a bound T that at least n of them reach is a lower bound of the n-th
// largest logit, only threads whose maximum reaches T can have seen one of the n,
// and their logits (one in kThreads each) are read again, a warp a thread's. What
// reaches T is ordered by counting.
//
// Bound by memory where rows are many (one block a row): 1024 rows of 151936 120 us,
// 5.2 TB/s. Few rows are cut over a cluster, whose results the first block joins: 32 rows
// 11 us, one row 13 (the pass 4, the rest steps that wait on each other). Before the
// tournament each exponential went to the f64 sum by itself and maxima moved with f64
// exponentials: 264 us for the 1024 rows.
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
constexpr int kMaxCluster = 4;

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
    float zd;
    double z;
};
__device__ __forceinline__ void rescale(Sum& s, float max) {  // max >= s.max
    const float down = fmaxf(s.max - max, -200.0f), f = expf(down);  // below e^-200 is nothing
    const bool none = s.max == -INFINITY, same = s.max == max;
    s.zd = none ? 0.0f : same ? s.zd : f * fmaf(down, (float)s.z, s.zd);
    s.z = none ? 0.0 : same ? s.z : s.z * (double)f;
    s.max = max;
}
// The sums of a warp's lanes, for all of them.
__device__ __forceinline__ Sum warp_sum(Sum s) {
    float max = s.max;
    for (int w = 16; w; w >>= 1) max = fmaxf(max, __shfl_xor_sync(0xFFFFFFFFu, max, w));
    rescale(s, max);
    for (int w = 16; w; w >>= 1) {
        s.z += __shfl_xor_sync(0xFFFFFFFFu, s.z, w);
        s.zd += __shfl_xor_sync(0xFFFFFFFFu, s.zd, w);
    }
    return s;
}

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }  // a NaN counts as -inf
__device__ __forceinline__ float2 exp_of(float2 d) {
    const float2 t = __fmul2_rn(d, make_float2(1.4426950408889634f, 1.4426950408889634f));
    float2 e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    return e;
}
// 16 logits more (-inf where there are fewer).
__device__ __forceinline__ void add(Sum& s, float (&x)[16]) {
    // after this x[0] is the largest, the others are what lost on the way
#pragma unroll
    for (int half = 8; half; half /= 2)
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float a = x[i], b = x[i + half];
            x[i] = fmaxf(a, b), x[i + half] = fminf(a, b);
        }
    if (x[0] > s.max) rescale(s, x[0]);
    const float m = s.max == -INFINITY ? 0.0f : -s.max;
    float2 z = make_float2(0.0f, 0.0f), zd = z;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        float2 d = __fadd2_rn(make_float2(x[i], x[i + 1]), make_float2(m, m));
        d = make_float2(fmaxf(d.x, -200.0f), fmaxf(d.y, -200.0f));  // below e^-200 is nothing, and -inf * 0 is none
        float2 e = exp_of(d);
        zd = __ffma2_rn(e, d, zd);
        if (i == 0) top = e.x, e.x = 0.0f;
        z = __fadd2_rn(z, e);
    }
    s.z += (double)(z.x + z.y);
    s.z += (double)top;
    s.zd += zd.x + zd.y;
}

struct Cand {
    float x;
    int id;
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.x > b.x || (a.x == b.x && a.id < b.id); }

// The first n of m candidates in order, into out (all threads; a warp a candidate).
// Blanks (-inf) are left out.
__device__ __forceinline__ void order_by_counting(const Cand* in, int m, int n, Cand* out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = warp; i < m; i += kWarps) {
        const Cand c = in[i];
        if (c.x == -INFINITY) continue;
        int rank = 0;
        for (int j = lane; j - lane < m; j += 32) rank += __popc(__ballot_sync(0xFFFFFFFFu, j < m && before(in[j], c)));
        if (lane == 0 && rank < n) out[rank] = c;
    }
}

// PACKS: rows are 16-byte aligned and read in packs of four.
template <bool PACKS>
__global__ void __launch_bounds__(kThreads, 2) logprobs_kernel(const LogprobArgs a, int cluster) {
    __shared__ float seconds[kWarps];
    __shared__ short reach[kThreads];       // threads whose maximum reaches T
    __shared__ Cand cand[kCand];
    __shared__ Cand best[kTop];             // of this block
    __shared__ Cand all[kMaxCluster * kTop], final[kTop];
    __shared__ Sum part[kWarps], sums[kMaxCluster], result;
    __shared__ int n_cand, n_reach, infinite;
    __shared__ unsigned long long pick[kWarps];
    const int rank = cluster > 1 ? blockIdx.x % cluster : 0;
    const int64_t row = blockIdx.x / cluster;
    const float* x = a.logits + row * a.stride;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // this block's share, in whole rounds of the block's packs
    constexpr int kPack = PACKS ? 4 : 1, kStep = kThreads * kPack, kBatch = 16 / kPack;
    const int rounds = (a.vocab + kStep - 1) / kStep;
    const int r0 = (int)((int64_t)rounds * rank / cluster), r1 = (int)((int64_t)rounds * (rank + 1) / cluster);
    const int begin = r0 * kStep, end = min(r1 * kStep, a.vocab);
    // arrive here, wait before the first remote write: the first block then runs
    if (cluster > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    if (threadIdx.x == 0) n_cand = n_reach = infinite = 0;
    if (threadIdx.x < kTop) best[threadIdx.x] = Cand{-INFINITY, -1}, final[threadIdx.x] = Cand{-INFINITY, -1};

    after_previous();

    // ---- the pass
    Sum s = {-INFINITY, 0.0f, 0.0};
    auto load = [&](int i, float (&v)[16]) {  // a batch: kBatch packs, kStep apart
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int at = i + u * kStep;
            if (PACKS) {
                float4 p = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (at + 4 <= end) {
                    p = __ldcs(reinterpret_cast<const float4*>(x + at));
                } else {  // the row's end in a pack
                    if (at < end) p.x = x[at];
                    if (at + 1 < end) p.y = x[at + 1];
                    if (at + 2 < end) p.z = x[at + 2];
                }
                v[4 * (u % 4)] = p.x, v[4 * (u % 4) + 1] = p.y, v[4 * (u % 4) + 2] = p.z, v[4 * (u % 4) + 3] = p.w;
            } else {
                v[u] = at < end ? __ldcs(x + at) : -INFINITY;
            }
        }
    };
    float now[16], next[16];
    const int first = begin + threadIdx.x * kPack;
    load(first, now);
    for (int i = first; i < end; i += kBatch * kStep) {
        load(i + kBatch * kStep, next);
#pragma unroll
        for (int u = 0; u < 16; ++u) now[u] = clean(now[u]);
        add(s, now);
#pragma unroll
        for (int u = 0; u < 16; ++u) now[u] = next[u];
    }
    const float own = s.max;
    const Sum w_sum = warp_sum(s);
    if (lane == 0) part[warp] = w_sum;
    // T: of the warps' largest maxima the n-th, or where n is above their number the
    // n/2-th of their second largest (two of a warp's lanes reach it)
    {
        float v = own;
        if (a.top > kWarps) {
            const unsigned at = __ballot_sync(0xFFFFFFFFu, own == w_sum.max);
            if (lane == __ffs(at) - 1) v = -INFINITY;
            for (int w = 16; w; w >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, w));
        } else {
            v = w_sum.max;
        }
        if (lane == 0) seconds[warp] = v;
    }
    __syncthreads();

    // ---- this block's likeliest
    if (a.top && begin < end) {
        const int nth = a.top > kWarps ? (a.top + 1) / 2 : a.top;
        float t;
        {
            const float v = seconds[lane % kWarps];
            int ahead = 0;
#pragma unroll
            for (int j = 0; j < kWarps; ++j) {
                const float other = __shfl_sync(0xFFFFFFFFu, v, j);
                ahead += other > v || (other == v && j < lane % kWarps);
            }
            t = __shfl_sync(0xFFFFFFFFu, v, __ffs(__ballot_sync(0xFFFFFFFFu, ahead == nth - 1)) - 1);
        }
        if (own >= t && own > -INFINITY) reach[atomicAdd(&n_reach, 1)] = (short)threadIdx.x;
        __syncthreads();
        auto offer = [&](int i, float v) {
            if (v >= t && v > -INFINITY) {  // not of a NaN
                const int at = atomicAdd(&n_cand, 1);
                if (at < kCand) cand[at] = Cand{v, i};
            }
        };
        for (int n = warp; n < n_reach; n += kWarps)  // a warp a thread's logits
            for (int i = begin + reach[n] * kPack + lane * kStep; i < end; i += 32 * kStep) {
                if (PACKS && i + 4 <= end) {
                    const float4 p = *reinterpret_cast<const float4*>(x + i);
                    offer(i, p.x), offer(i + 1, p.y), offer(i + 2, p.z), offer(i + 3, p.w);
                } else {
                    for (int u = 0; u < kPack && i + u < end; ++u) offer(i + u, x[i + u]);
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
    Sum total = {-INFINITY, 0.0f, 0.0};
    if (warp == 0) total = warp_sum(lane < kWarps ? part[lane] : total);
    const Cand* list = best;
    if (cluster > 1) {
        cg::cluster_group cl = cg::this_cluster();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (threadIdx.x == 0) *cl.map_shared_rank(&sums[rank], 0) = total;
        if ((int)threadIdx.x < a.top) cl.map_shared_rank(all, 0)[rank * a.top + threadIdx.x] = best[threadIdx.x];
        cl.sync();
        if (rank) return;
        if (warp == 0) total = warp_sum(lane < cluster ? sums[lane] : Sum{-INFINITY, 0.0f, 0.0});
        if (a.top) {
            order_by_counting(all, cluster * a.top, a.top, final);
            list = final;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) result = total;
    __syncthreads();
    total = result;
    if (total.max == INFINITY) {  // infinite logits share everything: counted
        int n = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) n += x[i] == INFINITY;
        atomicAdd(&infinite, n);
        __syncthreads();
        total.z = infinite, total.zd = 0.0f;
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
        if (a.entropy) a.entropy[row] = total.max == -INFINITY ? 0.0f : (float)(logz - (double)total.zd / total.z);
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
    // Blocks a row: two or four while every block has a multiprocessor for itself and a
    // share that is worth it (32 rows of 151936: 18.9, 14.3 and 11.0 us with 1, 2 and 4 blocks,
    // 13.2 with 8; 128 rows: 19.9, 21.4 and 27.6; one row of 32000: 8.4, 8.2 and 7.9)
    int cluster = 1;
    while (cluster < kMaxCluster && rows * cluster * 2 <= ctx->sm_count && vocab >= (int64_t)cluster * 2 * 16384) cluster *= 2;
    DeviceGuard dev(ctx->device);
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster)), cfg.blockDim = dim3(kThreads), cfg.stream = pick_stream(ctx, stream);
    cfg.attrs = at, cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = packs ? cudaLaunchKernelEx(&cfg, logprobs_kernel<true>, a, cluster) : cudaLaunchKernelEx(&cfg, logprobs_kernel<false>, a, cluster);
    return e == cudaSuccess ? STRATA_OK : cuda_fail(ctx, e, "logprobs kernel");
}
