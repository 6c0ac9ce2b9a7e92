// sample.cu — the next token of each row of logits: top-k, top-p, min-p, then
// temperature, drawn with a given random number (the reference's sampler runs
// these steps on the host: crates/strata-core/src/sampler.rs).
//
// Nothing is sorted. What the filters keep is always a prefix of the tokens in
// falling order (equal logits by index), so it is described by its last
// element (Cut: a logit's key and an index), and the draw walks tokens in index
// order. Top-k finds its cut by counting: a histogram of the distance below
// the row's maximum, then of the keys inside the one bin that holds the k-th,
// narrowed until a bin is one key. Top-p does the same with masses: a bin's
// mass is estimated from its count to choose the bin, and the choice is then
// settled by f64 sums over the elements themselves, so that the histogram only
// guides. Sums run over a fixed tree: the result does not depend on the order
// of any atomic (they count integers).
//
// A row is read from memory once: a cluster of blocks holds it in shared
// memory (a slice each) and the passes run there; partial results are
// exchanged through distributed shared memory, one cluster barrier each. All
// blocks of a cluster compute the same decisions from the same partials. Rows
// too long for that are read again from global memory (L2) by each pass.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "sequence.cuh"

namespace cg = cooperative_groups;

namespace strata {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = kThreads;     // a bin a thread
constexpr float kBinsPerNat = 32.0f;  // first histogram: 32 nats below the maximum, the last bin takes the rest
constexpr int kMaxCluster = 8;

struct SampleArgs {
    const float* logits;
    int64_t stride;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const double* uniform;
    int32_t* ids;
    float* logprobs;
    int vocab, slice;
    int resident;  // the slice fits shared memory
};

// Larger key = larger logit; 0 for what is never taken (-inf, NaN). -0 and +0 are equal.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}

// What is kept: keys above `key`, and of those equal to it the indices up to `index`.
struct Cut {
    uint32_t key;
    int index;
    __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
};

// One partial of an exchange between the blocks of a cluster.
struct Part {
    double a, b;
    uint32_t lo, hi;
    int n;
};

struct Shared {
    Part part[2];                  // exchanged, alternating
    uint32_t hist[2][kBins];       // exchanged, alternating
    double wsum[2][kWarps];
    uint32_t wlo[kWarps], whi[kWarps];
    int wn[kWarps];
    int pick_bin;
    uint32_t pick_count;
    double pick_mass;
    int found;
};

struct Row {
    const SampleArgs& a;
    Shared& sh;
    const float* x;  // this block's slice, in shared or global memory
    int base, n;     // its first index and its number of elements
    int seg;         // elements of a warp (contiguous)
    int rank, ranks;
    int turn, hturn;
    cg::cluster_group cluster;

    // every element of this warp's segment, 32 at a time: f(value, index)
    template <typename F>
    __device__ __forceinline__ void each(F f) {
        const int lo = (threadIdx.x >> 5) * seg, hi = min(lo + seg, n);
#pragma unroll 4
        for (int i = lo + (threadIdx.x & 31); i < hi; i += 32) f(x[i], base + i);
    }

    // Sums (a, b, n) and bounds (lo, hi) over the cluster, the same in every thread.
    __device__ Part reduce(Part p) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            p.a += __shfl_xor_sync(0xFFFFFFFFu, p.a, o);
            p.b += __shfl_xor_sync(0xFFFFFFFFu, p.b, o);
            p.n += __shfl_xor_sync(0xFFFFFFFFu, p.n, o);
            p.lo = min(p.lo, __shfl_xor_sync(0xFFFFFFFFu, p.lo, o));
            p.hi = max(p.hi, __shfl_xor_sync(0xFFFFFFFFu, p.hi, o));
        }
        if (lane == 0) {
            sh.wsum[0][warp] = p.a, sh.wsum[1][warp] = p.b;
            sh.wlo[warp] = p.lo, sh.whi[warp] = p.hi, sh.wn[warp] = p.n;
        }
        __syncthreads();
        if (warp == 0) {
            p.a = sh.wsum[0][lane], p.b = sh.wsum[1][lane];
            p.lo = sh.wlo[lane], p.hi = sh.whi[lane], p.n = sh.wn[lane];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                p.a += __shfl_xor_sync(0xFFFFFFFFu, p.a, o);
                p.b += __shfl_xor_sync(0xFFFFFFFFu, p.b, o);
                p.n += __shfl_xor_sync(0xFFFFFFFFu, p.n, o);
                p.lo = min(p.lo, __shfl_xor_sync(0xFFFFFFFFu, p.lo, o));
                p.hi = max(p.hi, __shfl_xor_sync(0xFFFFFFFFu, p.hi, o));
            }
            if (lane == 0) sh.part[turn] = p;
        }
        cluster.sync();  // a slot is written again two exchanges on: every block has read it by then
        Part r = *cluster.map_shared_rank(&sh.part[turn], 0);
        for (int k = 1; k < ranks; ++k) {
            const Part q = *cluster.map_shared_rank(&sh.part[turn], k);
            r.a += q.a, r.b += q.b, r.n += q.n;
            r.lo = min(r.lo, q.lo), r.hi = max(r.hi, q.hi);
        }
        turn ^= 1;
        return r;
    }

    // The cluster's count of this thread's bin. `fill` adds to the block's histogram.
    template <typename F>
    __device__ uint32_t histogram(F fill) {
        uint32_t* h = sh.hist[hturn];
        h[threadIdx.x] = 0;
        __syncthreads();
        fill(h);
        cluster.sync();
        uint32_t c = 0;
        for (int k = 0; k < ranks; ++k) c += cluster.map_shared_rank(h, k)[threadIdx.x];
        hturn ^= 1;
        return c;
    }

    // The first bin whose running sum reaches `target` (the last bin with a
    // count if none does), and the sum before it. W: uint32_t or double.
    template <typename W>
    __device__ int border(uint32_t count, W weight, W target, W& before) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        W incl = weight;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const W up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
            if (lane >= o) incl += up;
        }
        W* tot = reinterpret_cast<W*>(sh.wsum[0]);
        __syncthreads();
        if (lane == 31) tot[warp] = incl;
        if (threadIdx.x == 0) sh.pick_bin = kBins, sh.found = -1;
        __syncthreads();
        W base_sum = 0;
        for (int w = 0; w < warp; ++w) base_sum += tot[w];
        incl += base_sum;
        if (count) {
            atomicMax(&sh.found, (int)threadIdx.x);
            if (incl >= target) atomicMin(&sh.pick_bin, (int)threadIdx.x);
        }
        __syncthreads();
        const int bin = sh.pick_bin < kBins ? sh.pick_bin : sh.found;
        if ((int)threadIdx.x == bin) sh.pick_mass = (double)(incl - weight);
        __syncthreads();
        before = (W)sh.pick_mass;
        return bin;
    }

    // The nearest bin with a count before (dir < 0) or behind `bin`, -1 if none.
    __device__ int neighbour(uint32_t count, int bin, int dir) {
        __syncthreads();
        if (threadIdx.x == 0) sh.found = dir < 0 ? -1 : kBins;
        __syncthreads();
        if (count && dir < 0 && (int)threadIdx.x < bin) atomicMax(&sh.found, (int)threadIdx.x);
        if (count && dir > 0 && (int)threadIdx.x > bin) atomicMin(&sh.found, (int)threadIdx.x);
        __syncthreads();
        return sh.found < kBins ? sh.found : -1;
    }

    // The index of the nth (from 1) element with `key`, in index order.
    __device__ int nth(uint32_t key, int want) {
        int mine = 0;
        each([&](float v, int) { mine += key_of(v) == key; });
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, o);
        __syncthreads();
        if (lane == 0) sh.wn[warp] = mine;
        __syncthreads();
        int before = 0, total = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += sh.wn[w];
            total += sh.wn[w];
        }
        if (threadIdx.x == 0) sh.part[turn].n = total;
        cluster.sync();
        for (int k = 0; k < rank; ++k) before += cluster.map_shared_rank(&sh.part[turn], k)->n;
        turn ^= 1;
        uint32_t found = 0xFFFFFFFFu;
        if (before < want && want <= before + mine) {  // in this warp's segment
            const int lo = warp * seg, hi = min(lo + seg, n);
            int seen = before;
            for (int i = lo; i < hi; i += 32) {
                const bool hit = i + lane < hi && key_of(x[i + lane]) == key;
                const unsigned m = __ballot_sync(0xFFFFFFFFu, hit);
                if (seen + __popc(m) >= want) {
                    if (hit && seen + __popc(m & ((1u << lane) - 1u)) + 1 == want) found = (uint32_t)(base + i + lane);
                    break;
                }
                seen += __popc(m);
            }
        }
        return (int)reduce(Part{0.0, 0.0, found, 0u, 0}).lo;
    }
};

__device__ __forceinline__ double below(float x, float top) {  // x - top, 0 where equal (infinite ones too)
    return x == top ? 0.0 : (double)x - (double)top;
}
__device__ __forceinline__ int first_bin(float x, float top) {
    const float d = x == top ? 0.0f : (top - x) * kBinsPerNat;  // monotone: the subtraction and the product round once
    return (int)fminf(d, (float)(kBins - 1));
}
// Keys lo .. hi cut into kBins ranges of 2^shift, the largest first.
__device__ __forceinline__ int shift_of(uint32_t lo, uint32_t hi) {
    const int bits = 32 - __clz(hi - lo);
    return bits > 10 ? bits - 10 : 0;
}

__device__ Cut cut_top_k(Row& r, float top, uint32_t k) {
    uint32_t count = r.histogram([&](uint32_t* h) {
        r.each([&](float v, int) {
            if (key_of(v)) atomicAdd(&h[first_bin(v, top)], 1u);
        });
    });
    uint32_t before;
    const int bin = r.border<uint32_t>(count, count, k, before);
    uint32_t want = k - before;
    Part p{0.0, 0.0, 0xFFFFFFFFu, 0u, 0};
    r.each([&](float v, int) {
        const uint32_t key = key_of(v);
        if (key && first_bin(v, top) == bin) p.lo = min(p.lo, key), p.hi = max(p.hi, key);
    });
    p = r.reduce(p);
    uint32_t lo = p.lo, hi = p.hi;
    while (true) {
        const int shift = shift_of(lo, hi);
        count = r.histogram([&](uint32_t* h) {
            r.each([&](float v, int) {
                const uint32_t key = key_of(v);
                if (key >= lo && key <= hi) atomicAdd(&h[(hi - key) >> shift], 1u);
            });
        });
        const int j = r.border<uint32_t>(count, count, want, before);
        want -= before;
        const uint32_t upper = hi - ((uint32_t)j << shift), width = (1u << shift) - 1u;
        if (shift == 0) {
            // the keys above `upper` are all kept, and `want` of those equal to it
            __syncthreads();
            if ((int)threadIdx.x == j) r.sh.pick_count = count;
            __syncthreads();
            return Cut{upper, want >= r.sh.pick_count ? INT_MAX : r.nth(upper, (int)want)};
        }
        hi = upper;
        lo = upper - lo < width ? lo : upper - width;
    }
}

__device__ Cut cut_top_p(Row& r, float top, uint32_t top_key, double p, Cut cut) {
    if (p <= 0.0) return Cut{top_key, r.nth(top_key, 1)};
    // the kept tokens' mass, and their histogram
    Part z{0.0, 0.0, 0u, 0u, 0};
    const uint32_t count = r.histogram([&](uint32_t* h) {
        r.each([&](float v, int i) {
            const uint32_t key = key_of(v);
            if (key && cut.keeps(key, i)) {
                z.a += exp(below(v, top));
                atomicAdd(&h[first_bin(v, top)], 1u);
            }
        });
    });
    const double target = p * r.reduce(z).a;
    const double guess = (double)count * exp(-((double)threadIdx.x + 0.5) / (double)kBinsPerNat);
    double before;
    int bin = r.border<double>(count, guess, target, before), way = 0;
    uint32_t lo, hi;
    while (true) {  // until the bin holds the border: mass above < target <= mass above + its own
        Part s{0.0, 0.0, 0xFFFFFFFFu, 0u, 0};
        r.each([&](float v, int i) {
            const uint32_t key = key_of(v);
            if (key && cut.keeps(key, i)) {
                const int b = first_bin(v, top);
                if (b < bin) s.a += exp(below(v, top));
                else if (b == bin) {
                    s.b += exp(below(v, top));
                    s.lo = min(s.lo, key), s.hi = max(s.hi, key);
                }
            }
        });
        s = r.reduce(s);
        lo = s.lo, hi = s.hi, before = s.a;
        const int dir = s.a >= target ? -1 : s.a + s.b < target ? 1 : 0;
        if (dir == 0 || dir == -way) break;  // a turn back: the border lies between two bins
        const int next = r.neighbour(count, bin, dir);
        if (next < 0) {
            if (dir > 0) return cut;  // the sum's last bit: everything is needed
            break;
        }
        bin = next, way = dir;
    }
    while (true) {  // narrow the keys; a range's mass is its count times the middle's
        const int shift = shift_of(lo, hi);
        const uint32_t n = r.histogram([&](uint32_t* h) {
            r.each([&](float v, int i) {
                const uint32_t key = key_of(v);
                if (key >= lo && key <= hi && cut.keeps(key, i)) atomicAdd(&h[(hi - key) >> shift], 1u);
            });
        });
        const uint32_t far = (uint32_t)threadIdx.x << shift, width = (1u << shift) - 1u;
        const uint32_t upper_mine = n ? hi - far : hi;
        const double m = n ? (double)n * exp(below(logit_of(upper_mine - min(width / 2, upper_mine - lo)), top)) : 0.0;
        double above;
        const int j = r.border<double>(n, m, target - before, above);
        before += above;
        const uint32_t upper = hi - ((uint32_t)j << shift);
        hi = upper;
        if (shift == 0) break;
        lo = upper - lo < width ? lo : upper - width;
    }
    uint32_t key = hi;
    int way2 = 0;
    while (true) {  // settle the key by the elements' own sums
        Part s{0.0, 0.0, 0u, 0u, 0};
        uint32_t up = 0xFFFFFFFFu, down = 0u;  // the nearest kept keys above and below
        r.each([&](float v, int i) {
            const uint32_t k = key_of(v);
            if (k && cut.keeps(k, i)) {
                if (k > key) s.a += exp(below(v, top)), up = min(up, k);
                else if (k == key) ++s.n;
                else down = max(down, k);
            }
        });
        s.lo = up, s.hi = down;
        s = r.reduce(s);
        const double e = exp(below(logit_of(key), top));
        const int dir = s.a >= target ? -1 : s.a + (double)s.n * e < target ? 1 : 0;
        const uint32_t next = dir < 0 ? s.lo : s.hi;
        const bool more = dir < 0 ? next != 0xFFFFFFFFu : next != 0u;
        if (dir > 0 && !more) return cut;
        if (dir == 0 || dir == -way2 || !more) {
            double want = ceil((target - s.a) / e);
            if (want > 1.0 && s.a + (want - 1.0) * e >= target) want -= 1.0;
            else if (s.a + want * e < target) want += 1.0;
            if (!(want > 1.0)) want = 1.0;
            if (want < (double)s.n) return Cut{key, r.nth(key, (int)want)};
            return key > cut.key ? Cut{key, INT_MAX} : cut;
        }
        key = next, way2 = dir;
    }
}

__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleArgs a) {
    extern __shared__ float held[];
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int64_t row = blockIdx.x / ranks;
    const float* logits = a.logits + row * a.stride;
    const int base = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - base);
    Row r{a, sh, a.resident ? held : logits + base, base, n, ((n + kThreads - 1) / kThreads) * 32, rank, ranks, 0, 0,
          cluster};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // the row's largest logit, while the slice is brought in
    Part m{0.0, 0.0, 0xFFFFFFFFu, 0u, 0};
    {
        const int lo = warp * r.seg, hi = min(lo + r.seg, n);
#pragma unroll 8
        for (int i = lo + lane; i < hi; i += 32) {
            const float v = logits[base + i];
            if (a.resident) held[i] = v;
            const uint32_t key = key_of(v);
            m.hi = max(m.hi, key);
            m.n += key != 0u;
        }
    }
    m = r.reduce(m);
    const uint32_t top_key = m.hi;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    int id = -1;
    float logp = -INFINITY;
    if (top_key != 0u && !(t > 0.0f)) {
        id = r.nth(top_key, 1);
        logp = 0.0f;
    } else if (top_key != 0u) {
        const float top = logit_of(top_key);
        Cut cut{1u, INT_MAX};  // no element has key 1: everything but the excluded
        const int k = a.top_k ? a.top_k[row] : 0;
        if (k > 0 && k < m.n) cut = cut_top_k(r, top, (uint32_t)k);
        const float p = a.top_p ? a.top_p[row] : 1.0f;
        if (p < 1.0f) cut = cut_top_p(r, top, top_key, (double)p, cut);
        const float mp = a.min_p ? a.min_p[row] : 0.0f;
        if (mp > 1.0f) cut = Cut{top_key, r.nth(top_key, 1)};
        const bool by_min = mp > 0.0f && !(mp > 1.0f);
        const double least = (double)mp, log_least = by_min ? log(least) : 0.0;
        const double inv_t = 1.0 / (double)t;
        auto weight = [&](float v, int i) -> double {
            const uint32_t key = key_of(v);
            if (!key || !cut.keeps(key, i)) return 0.0;
            const double d = below(v, top);
            // the comparison of exponentials, decided by the logs unless they are close
            if (by_min && (d < log_least - 1e-9 || (d < log_least + 1e-9 && exp(d) < least))) return 0.0;
            return d == 0.0 ? 1.0 : d < -1e300 ? 0.0 : exp(d * inv_t);
        };
        double w = 0.0;
        r.each([&](float v, int i) { w += weight(v, i); });
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
        __syncthreads();
        if (lane == 0) sh.wsum[0][warp] = w;
        __syncthreads();
        double before = 0.0, total = 0.0;
        for (int i = 0; i < kWarps; ++i) {
            if (i < warp) before += sh.wsum[0][i];
            total += sh.wsum[0][i];
        }
        if (threadIdx.x == 0) sh.part[r.turn].a = total;
        cluster.sync();
        double all = 0.0, lower = 0.0;
        for (int i = 0; i < ranks; ++i) {
            if (i == rank) lower = all;
            all += cluster.map_shared_rank(&sh.part[r.turn], i)->a;
        }
        r.turn ^= 1;
        double u = a.uniform[row];
        u = u > 0.0 ? u : 0.0;
        const double target = u * all;
        // The first element whose running sum exceeds the target. The sums of
        // blocks, warps and elements are each taken in index order; where
        // their roundings disagree at a border (or u >= 1) the last element
        // with a weight before it is taken.
        // bounds: lo = the first element found, hi = 1 + the last one with a weight
        uint32_t found = 0xFFFFFFFFu, last = 0u;
        const double from = lower + before;
        if (w > 0.0) {
            const int lo = warp * r.seg, hi = min(lo + r.seg, n);
            const bool here = from + w > target;  // uniform in the warp
            // surely before the border, or surely behind it (an earlier warp finds it)
            const bool skip = (!here && u < 1.0 && from + w < target * (1.0 - 1e-9)) || from > target * (1.0 + 1e-9);
            double run = from;
            if (!skip)
                for (int i = lo; i < hi; i += 32) {
                    const double wi = i + lane < hi ? weight(r.x[i + lane], base + i + lane) : 0.0;
                    double incl = wi;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                        if (lane >= o) incl += up;
                    }
                    if (wi > 0.0) {
                        last = max(last, (uint32_t)(base + i + lane) + 1u);
                        if (run + incl > target) found = min(found, (uint32_t)(base + i + lane));
                    }
                    run += __shfl_sync(0xFFFFFFFFu, incl, 31);
                    if (__any_sync(0xFFFFFFFFu, found != 0xFFFFFFFFu)) break;
                }
        }
        const Part q = r.reduce(Part{0.0, 0.0, found, last, 0});
        id = q.lo != 0xFFFFFFFFu ? (int)q.lo : (int)q.hi - 1;
        const float v = logits[id];
        const double d = below(v, top);
        logp = (float)((d == 0.0 ? 0.0 : d * inv_t) - log(all));
    }
    if (rank == 0 && threadIdx.x == 0) {
        a.ids[row] = id;
        if (a.logprobs) a.logprobs[row] = logp;
    }
    cluster.sync();  // no block leaves while another may read its shared memory
}

}  // namespace
}  // namespace strata

using namespace strata;

extern "C" int strata_cuda_sample_dev(strata_ctx* ctx, const float* logits_dev, int64_t rows, int64_t vocab,
                                      int64_t stride, const float* temperature_dev, const int32_t* top_k_dev,
                                      const float* top_p_dev, const float* min_p_dev, const double* uniform_dev,
                                      int32_t* ids_dev, float* logprobs_dev, void* stream) {
    if (!ctx) return STRATA_ERR_INVALID;
    STRATA_CALL_RANGE();
    std::lock_guard<std::mutex> g(ctx->mu);
    Why why;
    const int rc = check_sample(why, logits_dev, rows, vocab, stride, temperature_dev, top_k_dev, top_p_dev, min_p_dev,
                                uniform_dev, ids_dev, logprobs_dev);
    if (rc) return fail(ctx, rc, "sample: %s", why.text);
    DeviceGuard dev(ctx->device);
    // a block takes at least 2048 logits; eight blocks are the portable cluster
    int ranks = 1;
    while (ranks < kMaxCluster && vocab > (int64_t)ranks * 2048) ranks *= 2;
    const int64_t slice = (vocab + ranks - 1) / ranks;
    const int64_t most = 200 * 1024;  // shared memory a block may take for its slice
    const bool resident = slice * 4 <= most;
    SampleArgs a{logits_dev, stride, temperature_dev, top_k_dev, top_p_dev, min_p_dev, uniform_dev, ids_dev,
                 logprobs_dev, (int)vocab, (int)slice, resident};
    cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cudaFuncSetAttribute(sample)");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = resident ? (size_t)slice * 4 : 0;
    cfg.stream = pick_stream(ctx, stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, sample_kernel, a);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "sample kernel");
    return check_launch(ctx, "sample kernel");
}
