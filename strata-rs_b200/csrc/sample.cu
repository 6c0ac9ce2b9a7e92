// sample.cu — the next token of each row of logits: top-k, top-p, min-p, then
// temperature, drawn with a given random number (the reference's sampler runs
// these steps on the host: crates/strata-core/src/sampler.rs).
//
// What the filters keep is always a prefix of the tokens in falling order
// (equal logits by index), so it is described by its last element (Cut: a
// logit's key and an index), and the draw walks tokens in index order.
//
// A cluster of blocks takes a row, a slice of the vocabulary each. One pass
// over the logits finds the maximum and a histogram of the values (and, where
// a filter or the draw needs every token's weight, their f64 sum). The
// histogram says which bins can hold the last kept token: a second pass (from
// shared memory, or L2 where the slice does not fit) gathers the tokens of
// those bins into a list, sums what lies surely above them, and the first
// block settles the cut on the list alone. The histogram only guides: masses
// are compared as f64 sums of the elements themselves, in an order that does
// not depend on any atomic (those count integers). Where the list does not
// hold (nearly flat or clustered rows with a far cut), the same search runs
// over the whole slices, narrowing key ranges pass by pass.
//
// Bound by the logits' bytes for rows whose filters need no sum over the
// vocabulary, and by the f64 pipe (one exponential a token, 8 products and
// sums) where they do.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "sequence.cuh"

namespace cg = cooperative_groups;

namespace strata {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = kThreads;       // a bin a thread
constexpr int kBinBits = 9;
static_assert(kBins == 1 << kBinBits, "a key range is cut into kBins");
constexpr float kBinsPerNat = 16.0f;  // value histograms: 32 nats, the last bin takes the rest
constexpr int kMaxCluster = 8;
constexpr int kList = 4096;           // tokens a list holds
constexpr int kExpTable = 128;

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
    int packs;     // rows and slices are whole 16-byte packs
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

// A block's part of what the first pass finds.
struct First {
    double sum;       // of every token's weight, where the row needs it
    float best;       // largest logit and its first index
    int index, alive; // tokens that can be taken
};

struct Shared {
    First first;                   // exchanged
    double above;                  // exchanged: mass above the list
    double seg[kWarps];            // exchanged: weights of each warp's tokens above the list
    int listed[kWarps];            // exchanged: tokens each warp put into the list
    int block_listed;              // exchanged: their sum
    uint8_t chain[kWarps][kList / 32];  // the pool's groups of 32 that hold them, in order
    int pool_used;
    int offset[kMaxCluster * kWarps + 1];  // of each warp's tokens in the list of the whole row
    double exp2_table[kExpTable];
    int won, id;                   // the draw: its segment (-1: id is the token)
    double won_before, total, weight;
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
    const float* x;    // this block's slice, in shared or global memory; or a list
    const int* index;  // a list's indices (nullptr: x is a slice)
    int base, n;       // its first index and its number of elements
    int seg;         // elements of a warp (contiguous)
    int rank, ranks;
    int turn, hturn;
    cg::cluster_group cluster;

    __device__ __forceinline__ int at(int i) const { return index ? index[i] : base + i; }
    __device__ __forceinline__ void sync() {
        if (ranks == 1) __syncthreads();
        else cluster.sync();
    }
    template <typename T>
    __device__ __forceinline__ const T* of(const T* p, int k) {
        return ranks == 1 ? p : cluster.map_shared_rank(const_cast<T*>(p), k);
    }

    // every element of this warp's segment, 32 at a time: f(value, index)
    template <typename F>
    __device__ __forceinline__ void each(F f) {
        const int lo = (threadIdx.x >> 5) * seg, hi = min(lo + seg, n);
#pragma unroll 4
        for (int i = lo + (threadIdx.x & 31); i < hi; i += 32) f(x[i], at(i));
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
            const int w = lane % kWarps;
            p.a = sh.wsum[0][w], p.b = sh.wsum[1][w];
            p.lo = sh.wlo[w], p.hi = sh.whi[w], p.n = sh.wn[w];
#pragma unroll
            for (int o = kWarps / 2; o > 0; o >>= 1) {
                p.a += __shfl_xor_sync(0xFFFFFFFFu, p.a, o);
                p.b += __shfl_xor_sync(0xFFFFFFFFu, p.b, o);
                p.n += __shfl_xor_sync(0xFFFFFFFFu, p.n, o);
                p.lo = min(p.lo, __shfl_xor_sync(0xFFFFFFFFu, p.lo, o));
                p.hi = max(p.hi, __shfl_xor_sync(0xFFFFFFFFu, p.hi, o));
            }
            if (lane == 0) sh.part[turn] = p;
        }
        sync();  // a slot is written again two exchanges on: every block has read it by then
        Part r = *of(&sh.part[turn], 0);
        for (int k = 1; k < ranks; ++k) {
            const Part q = *of(&sh.part[turn], k);
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
        sync();
        uint32_t c = 0;
        for (int k = 0; k < ranks; ++k) c += of(h, k)[threadIdx.x];
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
        sync();
        for (int k = 0; k < rank; ++k) before += of(&sh.part[turn], k)->n;
        turn ^= 1;
        uint32_t found = 0xFFFFFFFFu;
        if (before < want && want <= before + mine) {  // in this warp's segment
            const int lo = warp * seg, hi = min(lo + seg, n);
            int seen = before;
            for (int i = lo; i < hi; i += 32) {
                const bool hit = i + lane < hi && key_of(x[i + lane]) == key;
                const unsigned m = __ballot_sync(0xFFFFFFFFu, hit);
                if (seen + __popc(m) >= want) {
                    if (hit && seen + __popc(m & ((1u << lane) - 1u)) + 1 == want) found = (uint32_t)at(i + lane);
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
    return bits > kBinBits ? bits - kBinBits : 0;
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

// `above`: the mass of kept tokens larger than all of the view's. total: the
// kept tokens' mass (0: those of the view). `fits` (optional) reports whether
// the border lies in the view; it does not where the view ends above it.
__device__ Cut cut_top_p(Row& r, float top, double p, Cut cut, double above, double total, bool* fits) {
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
    const double mass = r.reduce(z).a;
    const double target = p * (total > 0.0 ? total : above + mass) - above;
    if (fits) {
        *fits = target > 0.0 && target <= mass;
        if (!*fits) return cut;
    }
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
        double more;
        const int j = r.border<double>(n, m, target - before, more);
        before += more;
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

// exp(x) by the table method (Tang, 1989): x = (128 m + j) ln2 / 128 + r,
// exp(x) = 2^m 2^(j/128) exp(r), |r| <= ln2 / 256, four terms of the series.
// Good to a few 1e-15 of the result for |x| < 700 (the cuts compare sums of
// thousands of tokens); 0 below -700, infinity above 700.
__device__ __forceinline__ double exp_table(double x, const double* table) {
    constexpr double kLn2 = 0.69314718055994530942, kMagic = 6755399441055744.0;  // 1.5 * 2^52
    if (!(x > -700.0)) return 0.0;
    if (x > 700.0) return INFINITY;
    const double t = fma(x, kExpTable / kLn2, kMagic);
    const int n = __double2loint(t);
    const double r = fma(t - kMagic, -kLn2 / kExpTable, x);
    const double q = fma(r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0);
    const double b = table[n & (kExpTable - 1)];
    const double y = fma(b * r, q, b);
    return __hiloint2double(__double2hiint(y) + ((n >> 7) << 20), __double2loint(y));
}

// The value histogram of the first pass: `high` falls into bin 0.
__device__ __forceinline__ int value_bin(float v, float high) {
    return (int)fminf(fmaxf((high - v) * kBinsPerNat, 0.0f), (float)(kBins - 1));
}

constexpr int kListBytes = kList * 16;          // the pool of this block's tokens, and the row's list
constexpr int64_t kMaxSlice = 128 * 1024;       // bytes of a slice that is kept in shared memory,
constexpr int64_t kPairSlice = 38 * 1024;       // and that leave room for two blocks a multiprocessor

// Four elements of a lane: neighbours where the row is 16-byte packs, 32 apart otherwise.
template <bool PACKS>
__device__ __forceinline__ int element(int i, int e) {
    const int lane = threadIdx.x & 31;
    return PACKS ? i + lane * 4 + e : i + e * 32 + lane;
}
template <bool PACKS>
__device__ __forceinline__ void load4(const float* x, int i, int hi, float (&v)[4]) {
    if (PACKS) {
        const int at = element<true>(i, 0);
        if (at < hi) {
            const float4 p = *reinterpret_cast<const float4*>(x + at);
            v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w;
        } else {
            v[0] = v[1] = v[2] = v[3] = -INFINITY;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = element<false>(i, e);
            v[e] = at < hi ? x[at] : -INFINITY;
        }
    }
}

// The first element, in index order, of [lo, hi) of the block's slice whose
// running sum of weights exceeds `target` (the last one with a weight if none
// does): the block's warps take a part each, the warp that holds it walks its part.
template <typename W>
__device__ int locate(Row& r, int lo, int hi, double target, double* weight_out, W weight) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = ((hi - lo + kThreads - 1) / kThreads) * 32;
    const int from = min(lo + warp * part, hi), to = min(from + part, hi);
    double w = 0.0;
    for (int i = from + lane; i < to; i += 32) w += weight(r.x[i], r.base + i);
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
    __syncthreads();
    if (lane == 0) r.sh.wsum[0][warp] = w;
    if (threadIdx.x == 0) r.sh.found = -1, r.sh.pick_bin = INT_MAX;
    __syncthreads();
    double run = 0.0;
    bool mine = w > 0.0;  // the first warp whose sum goes past the target, else the last with a weight
    for (int k = 0; k < kWarps; ++k) {
        if (k < warp) run += r.sh.wsum[0][k];
        else if (k > warp && run + w <= target && r.sh.wsum[0][k] > 0.0) mine = false;
    }
    if (run > target) mine = false;
    if (mine) {
        int found = INT_MAX, last = -1;
        for (int i = from; i < to; i += 32) {
            const double wi = i + lane < to ? weight(r.x[i + lane], r.base + i + lane) : 0.0;
            double incl = wi;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                if (lane >= o) incl += up;
            }
            if (wi > 0.0) {
                last = i + lane;
                if (run + incl > target) found = i + lane;
            }
            run += __shfl_sync(0xFFFFFFFFu, incl, 31);
            if (__any_sync(0xFFFFFFFFu, found != INT_MAX)) break;
        }
        if (found != INT_MAX) atomicMin(&r.sh.pick_bin, found);
        if (last >= 0) atomicMax(&r.sh.found, last);
    }
    __syncthreads();
    const int at = r.sh.pick_bin != INT_MAX ? r.sh.pick_bin : r.sh.found;
    *weight_out = at >= 0 ? weight(r.x[at], r.base + at) : 0.0;
    return at >= 0 ? r.base + at : -1;
}

// The search over whole slices: for rows whose cut no list holds.
__device__ void sample_wide(Row& r, const float* logits, float top, int top_index, int alive, float t, int k, float p,
                            float mp, double u_in, int& id, float& logp) {
    Shared& sh = r.sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Cut cut{1u, INT_MAX};  // no element has key 1: everything but the excluded
    if (k > 0 && k < alive) cut = cut_top_k(r, top, (uint32_t)k);
    if (p < 1.0f) cut = cut_top_p(r, top, (double)p, cut, 0.0, 0.0, nullptr);
    const bool by_min = mp > 0.0f;
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
    r.sync();
    double all = 0.0, lower = 0.0;
    for (int i = 0; i < r.ranks; ++i) {
        if (i == r.rank) lower = all;
        all += r.of(&sh.part[r.turn], i)->a;
    }
    r.turn ^= 1;
    const double target = u_in * all;
    // The first element whose running sum exceeds the target. The sums of
    // blocks, warps and elements are each taken in index order; where their
    // roundings disagree at a border (or u >= 1) the last element with a
    // weight before it is taken.
    uint32_t found = 0xFFFFFFFFu, last = 0u;  // the first one past the target; 1 + the last one with a weight
    const double from = lower + before;
    if (w > 0.0) {
        const int lo = warp * r.seg, hi = min(lo + r.seg, r.n);
        const bool here = from + w > target;  // uniform in the warp
        // surely before the border, or surely behind it (an earlier warp finds it)
        const bool skip = (!here && u_in < 1.0 && from + w < target * (1.0 - 1e-9)) || from > target * (1.0 + 1e-9);
        double run = from;
        if (!skip)
            for (int i = lo; i < hi; i += 32) {
                const double wi = i + lane < hi ? weight(r.x[i + lane], r.at(i + lane)) : 0.0;
                double incl = wi;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                    if (lane >= o) incl += up;
                }
                if (wi > 0.0) {
                    last = max(last, (uint32_t)r.at(i + lane) + 1u);
                    if (run + incl > target) found = min(found, (uint32_t)r.at(i + lane));
                }
                run += __shfl_sync(0xFFFFFFFFu, incl, 31);
                if (__any_sync(0xFFFFFFFFu, found != 0xFFFFFFFFu)) break;
            }
    }
    const Part q = r.reduce(Part{0.0, 0.0, found, last, 0});
    id = q.lo != 0xFFFFFFFFu ? (int)q.lo : (int)q.hi - 1;
    const double d = below(logits[id], top);
    logp = (float)((d == 0.0 ? 0.0 : d * inv_t) - log(all));
}

template <bool PACKS>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    float* pool = reinterpret_cast<float*>(dynamic);             // values, then indices
    int* pool_index = reinterpret_cast<int*>(pool + kList);
    float* list = pool + 2 * kList;
    int* list_index = reinterpret_cast<int*>(pool + 3 * kList);
    float* held = pool + 4 * kList;
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int64_t row = blockIdx.x / ranks;
    const float* logits = a.logits + row * a.stride;
    const int base = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - base);
    const int seg = ((n + kWarps * 128 - 1) / (kWarps * 128)) * 128;
    Row r{a, sh, a.resident ? held : logits + base, nullptr, base, n, seg, rank, ranks, 0, 0, cluster};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int lo = warp * seg, hi = min(lo + seg, n);

    const float t = a.temperature ? a.temperature[row] : 1.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    if (k >= a.vocab) k = 0;
    float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f;
    if (!(p < 1.0f)) p = 1.0f;
    if (!(mp > 0.0f)) mp = 0.0f;
    double u = a.uniform[row];
    u = u > 0.0 ? u : 0.0;
    const bool greedy = !(t > 0.0f) || p <= 0.0f || mp > 1.0f || k == 1;
    const double inv_t = 1.0 / (double)t;
    const bool sums_all = !greedy && k <= 0 && (p < 1.0f || mp == 0.0f);  // the first pass sums every weight
    const bool draws_all = sums_all && p >= 1.0f;                         // at the draw's temperature

    // Where the histogram lies and what the sums refer to: the largest of a
    // sample of the row, the same for all its blocks.
    for (int i = threadIdx.x; i < kExpTable; i += kThreads) sh.exp2_table[i] = exp2((double)i / kExpTable);
    if (threadIdx.x == 0) sh.pool_used = 0;
    sh.hist[0][threadIdx.x] = 0;
    float center = logits[(int64_t)threadIdx.x * a.vocab / kThreads];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) center = fmaxf(center, __shfl_xor_sync(0xFFFFFFFFu, center, o));
    if (lane == 0) sh.wlo[warp] = __float_as_uint(center);
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) center = fmaxf(center, __uint_as_float(sh.wlo[w]));
    if (!(fabsf(center) < 1e30f)) center = 0.0f;  // a masked or infinite sample
    const float high = center + 8.0f;
    const double ref = (double)center;

    // first pass
    {
        double sum = 0.0;
        float best = -INFINITY;
        int index = INT_MAX, alive = 0;
        const double f = draws_all ? inv_t : 1.0;
        for (int i = lo; i < hi; i += 128) {
            float v[4];
            load4<PACKS>(logits + base, i, hi, v);
            if (a.resident) {
                if (PACKS) {
                    if (element<true>(i, 0) < hi)
                        *reinterpret_cast<float4*>(held + element<true>(i, 0)) = make_float4(v[0], v[1], v[2], v[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (element<false>(i, e) < hi) held[element<false>(i, e)] = v[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!(v[e] > -INFINITY)) continue;
                ++alive;
                if (v[e] > best) best = v[e], index = base + element<PACKS>(i, e);
                if (greedy) continue;
                if (!draws_all) atomicAdd(&sh.hist[0][value_bin(v[e], high)], 1u);
                if (sums_all) sum += exp_table(((double)v[e] - ref) * f, sh.exp2_table);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float b2 = __shfl_xor_sync(0xFFFFFFFFu, best, o);
            const int i2 = __shfl_xor_sync(0xFFFFFFFFu, index, o);
            if (b2 > best || (b2 == best && i2 < index)) best = b2, index = i2;
            sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            alive += __shfl_xor_sync(0xFFFFFFFFu, alive, o);
        }
        if (lane == 0) {
            sh.wsum[0][warp] = sum, sh.wn[warp] = alive;
            sh.wlo[warp] = __float_as_uint(best), sh.whi[warp] = (uint32_t)index;
            sh.seg[warp] = draws_all ? sum : 0.0;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            First m{0.0, -INFINITY, INT_MAX, 0};
            for (int w = 0; w < kWarps; ++w) {
                const float b2 = __uint_as_float(sh.wlo[w]);
                const int i2 = (int)sh.whi[w];
                if (b2 > m.best || (b2 == m.best && i2 < m.index)) m.best = b2, m.index = i2;
                m.sum += sh.wsum[0][w], m.alive += sh.wn[w];
            }
            sh.first = m;
        }
    }
    r.sync();
    First m{0.0, -INFINITY, INT_MAX, 0};
    uint32_t count = 0;
    for (int i = 0; i < ranks; ++i) {
        const First q = *r.of(&sh.first, i);
        if (q.best > m.best) m.best = q.best, m.index = q.index;  // ranks hold rising indices
        m.sum += q.sum, m.alive += q.alive;
        count += r.of(sh.hist[0], i)[threadIdx.x];
    }
    r.hturn = 1;
    const float top = m.best;

    int id = -1;
    float logp = -INFINITY;
    bool done = true, wide = false;
    if (m.alive > 0 && greedy) {
        id = m.index;
        // the one kept token; at a positive temperature it has all the weight
        logp = 0.0f;
    } else if (m.alive > 0) {
        done = false;
    }

    // Which bins the list takes ([first, last]); bins before it are kept for sure.
    int first = 0, last = -1;
    bool sure = false, by_k = false;
    if (!done) {
        by_k = k > 0 && k < m.alive;
        // a range that the sample misjudged, or infinite logits
        if (sums_all && !(m.sum > 1e-250 && m.sum < 1e250 && top < 1e30f)) wide = true;
        if (wide || draws_all) {
        } else if (k > 0 || mp > 0.0f) {
            // top-p behind top-k needs the mass of all k; otherwise nothing below min-p's bin matters
            const int by_min = mp > 0.0f && !(k > 0 && p < 1.0f)
                                   ? value_bin(__double2float_rd((double)top + log((double)mp) - 1e-4), high)
                                   : kBins - 1;
            last = by_min;
            if (by_k) {
                uint32_t before;
                last = r.border<uint32_t>(count, count, (uint32_t)k, before);
                if (last > by_min) last = by_min, by_k = false;  // what min-p keeps is less than k
            }
        } else {
            // the bins around the estimated border, far enough that the estimate's error cannot matter
            const double guess = (double)count * exp(-((double)threadIdx.x + 0.5) / (double)kBinsPerNat);
            double before, mass = guess;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xFFFFFFFFu, mass, o);
            __syncthreads();
            if (lane == 0) sh.wsum[1][warp] = mass;
            __syncthreads();
            mass = 0.0;
            for (int w = 0; w < kWarps; ++w) mass += sh.wsum[1][w];
            first = r.border<double>(count, guess, (double)p * mass * (1.0 - 1e-3), before);
            last = r.border<double>(count, guess, (double)p * mass * (1.0 + 1e-3), before);
            sure = true;
        }
    }
    auto sure_weight = [&](float v) { return exp_table(((double)v - ref) * inv_t, sh.exp2_table); };

    // second pass: the list's tokens, and the sums of what lies above them
    if (!done && !wide && !draws_all) {
        double above = 0.0, weights = 0.0;
        int mine = 0;
        for (int i = lo; i < hi; i += 128) {
            float v[4];
            load4<PACKS>(r.x, i, hi, v);
            int take = 0, bits = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!(v[e] > -INFINITY)) continue;
                const int b = value_bin(v[e], high);
                if (b > last) continue;
                if (b >= first) {
                    bits |= 1 << e, ++take;
                } else {
                    above += exp_table((double)v[e] - ref, sh.exp2_table);
                    weights += sure_weight(v[e]);
                }
            }
            if (!__any_sync(0xFFFFFFFFu, take)) continue;
            int pos[4], all = 0;  // places of this step's tokens, in index order
            if (PACKS) {
                int incl = take;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                    if (lane >= o) incl += up;
                }
                all = __shfl_sync(0xFFFFFFFFu, incl, 31);
#pragma unroll
                for (int e = 0; e < 4; ++e) pos[e] = incl - take + __popc(bits & ((1 << e) - 1));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned votes = __ballot_sync(0xFFFFFFFFu, bits >> e & 1);
                    pos[e] = all + __popc(votes & ((1u << lane) - 1u));
                    all += __popc(votes);
                }
            }
            if (lane == 0)  // groups of 32 from the pool, up to the last of them
                for (int g = (mine + 31) / 32; g < (mine + all + 31) / 32; ++g) {
                    const int got = atomicAdd(&sh.pool_used, 1);
                    if (g < kList / 32) sh.chain[warp][g] = (uint8_t)min(got, kList / 32 - 1);
                }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int slot = mine + pos[e];
                if ((bits >> e & 1) && slot < kList) {
                    const int to = sh.chain[warp][slot / 32] * 32 + slot % 32;
                    pool[to] = v[e];
                    pool_index[to] = base + element<PACKS>(i, e);
                }
            }
            mine += all;
        }
        for (int o = 16; o > 0; o >>= 1) {
            above += __shfl_xor_sync(0xFFFFFFFFu, above, o);
            weights += __shfl_xor_sync(0xFFFFFFFFu, weights, o);
        }
        if (lane == 0) sh.listed[warp] = mine, sh.seg[warp] = weights, sh.wsum[0][warp] = above;
        __syncthreads();
        if (threadIdx.x == 0) {
            double s = 0.0;
            int c = sh.pool_used > kList / 32 ? kList + 1 : 0;  // more than the pool holds
            for (int w = 0; w < kWarps; ++w) s += sh.wsum[0][w], c += sh.listed[w];
            sh.above = s, sh.block_listed = c;
        }
        r.sync();
    }
    // every block: does the list hold?
    int listed = 0;
    double above = 0.0;
    if (!done && !wide && !draws_all) {
        for (int i = 0; i < ranks; ++i) {
            listed += *r.of(&sh.block_listed, i);
            above += *r.of(&sh.above, i);
        }
        if (listed > kList) wide = true;
    }

    // the first block settles the cut and finds the draw's segment
    Cut cut{1u, INT_MAX};
    if (!done && !wide && rank == 0) {
        const int segs = ranks * kWarps;
        if (threadIdx.x == 0) sh.won = -1, sh.id = -1;
        bool fits = true;
        if (!draws_all) {
            if (warp == 0) {  // where each warp's tokens start in the list
                int before = 0;
                for (int g = 0; g < segs; g += 32) {
                    int c = g + lane < segs ? r.of(sh.listed, (g + lane) / kWarps)[(g + lane) % kWarps] : 0, own_c = c;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int up = __shfl_up_sync(0xFFFFFFFFu, c, o);
                        if (lane >= o) c += up;
                    }
                    if (g + lane < segs) sh.offset[g + lane] = before + c - own_c;
                    before += __shfl_sync(0xFFFFFFFFu, c, 31);
                }
                if (lane == 0) sh.offset[segs] = before;
            }
            __syncthreads();
            for (int g = warp; g < segs; g += kWarps) {
                const int q = g / kWarps, from = sh.offset[g], c = sh.offset[g + 1] - from;
                const uint8_t* chain = r.of(&sh.chain[0][0], q) + (g % kWarps) * (kList / 32);
                const float* pv = r.of(pool, q);
                const int* pi = r.of(pool_index, q);
                for (int i = lane; i < c; i += 32) {
                    const int at = chain[i / 32] * 32 + i % 32;
                    list[from + i] = pv[at];
                    list_index[from + i] = pi[at];
                }
            }
            __syncthreads();
            Row l{a, sh, list, list_index, 0, listed, ((listed + kThreads - 1) / kThreads) * 32, 0, 1, r.turn, r.hturn, cluster};
            if (by_k) cut = cut_top_k(l, top, (uint32_t)k);
            if (p < 1.0f) {
                if (sure) {
                    const double scale = exp(ref - (double)top);
                    cut = cut_top_p(l, top, (double)p, cut, above * scale, m.sum * scale, &fits);
                } else if (k > 0) {
                    cut = cut_top_p(l, top, (double)p, cut, 0.0, 0.0, nullptr);
                } else {
                    // the list ends at min-p's bin: top-p's border may lie behind it, and then cuts nothing here
                    bool inside;
                    cut = cut_top_p(l, top, (double)p, cut, 0.0, m.sum * exp(ref - (double)top), &inside);
                }
            }
            r.turn = l.turn, r.hturn = l.hturn;
        }
        if (!fits) {
            if (threadIdx.x == 0) sh.won = -2;
        } else if (!sure && !draws_all) {
            // the draw is among the list's tokens
            const bool by_min = mp > 0.0f;
            const double least = (double)mp, log_least = by_min ? log(least) : 0.0;
            constexpr int PER = kList / kThreads;
            double w[PER], own = 0.0;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int i = threadIdx.x * PER + e;
                w[e] = 0.0;
                if (i < listed) {
                    const float v = list[i];
                    const double d = below(v, top);
                    const bool small = by_min && (d < log_least - 1e-9 || (d < log_least + 1e-9 && exp(d) < least));
                    if (cut.keeps(key_of(v), list_index[i]) && !small)
                        w[e] = d == 0.0 ? 1.0 : d < -1e300 ? 0.0 : exp(d * inv_t);
                }
                own += w[e];
            }
            double incl = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                if (lane >= o) incl += up;
            }
            __syncthreads();
            if (lane == 31) sh.wsum[0][warp] = incl;
            if (threadIdx.x == 0) sh.pick_bin = INT_MAX, sh.found = -1;
            __syncthreads();
            double before = 0.0, total = 0.0;
            for (int i = 0; i < kWarps; ++i) {
                if (i < warp) before += sh.wsum[0][i];
                total += sh.wsum[0][i];
            }
            const double target = u * total;
            double run = before + (incl - own);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                run += w[e];
                if (w[e] > 0.0) {
                    atomicMax(&sh.found, threadIdx.x * PER + e);
                    if (run > target) atomicMin(&sh.pick_bin, threadIdx.x * PER + e);
                }
            }
            __syncthreads();
            const int at = sh.pick_bin != INT_MAX ? sh.pick_bin : sh.found;
            if (at / PER == (int)threadIdx.x) {
                double mine = 0.0;
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    if (at % PER == e) mine = w[e];
                sh.id = list_index[at], sh.weight = mine, sh.total = total;
            }
        } else {
            // the segment that holds the draw: each one's sure weights and its kept tokens of the list
            double w = 0.0;
            const int g = threadIdx.x;
            if (g < segs) {
                w = r.of(sh.seg, g / kWarps)[g % kWarps];
                if (!draws_all)
                    for (int i = sh.offset[g]; i < sh.offset[g + 1]; ++i)
                        if (cut.keeps(key_of(list[i]), list_index[i])) w += sure_weight(list[i]);
            }
            double incl = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                if (lane >= o) incl += up;
            }
            __syncthreads();
            if (lane == 31) sh.wsum[0][warp] = incl;
            if (threadIdx.x == 0) sh.pick_bin = INT_MAX, sh.found = -1;
            __syncthreads();
            double before = 0.0, total = 0.0;
            for (int i = 0; i < kWarps; ++i) {
                if (i < warp) before += sh.wsum[0][i];
                total += sh.wsum[0][i];
            }
            const double target = u * total;
            if (w > 0.0) {
                atomicMax(&sh.found, g);
                if (before + incl > target) atomicMin(&sh.pick_bin, g);
            }
            __syncthreads();
            const int won = sh.pick_bin != INT_MAX ? sh.pick_bin : sh.found;
            if (!(total > 1e-250 && total < 1e250)) {  // a temperature that takes the weights out of range
                if (threadIdx.x == 0) sh.won = -2;
            } else if (won == g) {
                sh.won = won, sh.won_before = target - (before + (incl - w)), sh.total = total;
                sh.part[0].lo = cut.key, sh.part[0].n = cut.index;
            }
        }
    }
    if (!done && !wide) {
        r.sync();
        const int won = *r.of(&sh.won, 0);
        const double total = *r.of(&sh.total, 0);
        if (won == -2) {
            wide = true;
        } else if (won < 0) {
            id = *r.of(&sh.id, 0);
            logp = (float)log(*r.of(&sh.weight, 0) / total);
        } else {
            const Part* q = r.of(&sh.part[0], 0);
            const Cut c{q->lo, q->n};
            const double target = *r.of(&sh.won_before, 0);
            if (won / kWarps == rank) {
                const int from = (won % kWarps) * seg, to = min(from + seg, n);
                double w;
                const int got = locate(r, from, to, target, &w, [&](float v, int i) -> double {
                    if (!(v > -INFINITY)) return 0.0;
                    if (!draws_all) {
                        const int b = value_bin(v, high);
                        if (b > last || (b >= first && !c.keeps(key_of(v), i))) return 0.0;
                    }
                    return sure_weight(v);
                });
                if (threadIdx.x == 0) {
                    a.ids[row] = got;
                    if (a.logprobs) a.logprobs[row] = (float)log(w / total);
                }
            }
        }
        if (won >= 0) {
            if (ranks > 1) cluster.sync();  // no block leaves while another may read its shared memory
            return;
        }
        r.sync();  // the first block's words have been read
    }
    if (wide) {
        r.turn = 0, r.hturn = 1;  // the same in every block
        sample_wide(r, logits, top, m.index, m.alive, t, k, p, mp, u, id, logp);
    }
    if (rank == 0 && threadIdx.x == 0) {
        a.ids[row] = id;
        if (a.logprobs) a.logprobs[row] = logp;
    }
    if (ranks > 1) cluster.sync();
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
    // blocks a row takes: as many as keep the GPU busy with two a multiprocessor
    // (eight are the portable cluster), each with at least 2048 logits
    int ranks = 1;
    while (ranks < kMaxCluster && vocab > (int64_t)ranks * 2048 && rows * ranks * 2 <= 2 * (int64_t)ctx->sm_count)
        ranks *= 2;
    const int64_t slice = ((vocab + ranks - 1) / ranks + 3) / 4 * 4;
    const bool resident = slice * 4 <= (rows * ranks > ctx->sm_count ? kPairSlice : kMaxSlice);
    const bool packs = stride % 4 == 0 && vocab % 4 == 0 && (uintptr_t)logits_dev % 16 == 0;
    SampleArgs a{logits_dev, stride, temperature_dev, top_k_dev, top_p_dev, min_p_dev, uniform_dev, ids_dev,
                 logprobs_dev, (int)vocab, (int)slice, resident, packs};
    auto kernel = packs ? sample_kernel<true> : sample_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kListBytes + kMaxSlice);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cudaFuncSetAttribute(sample)");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)(kListBytes + (resident ? slice * 4 : 0));
    cfg.stream = pick_stream(ctx, stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "sample kernel");
    return check_launch(ctx, "sample kernel");
}
