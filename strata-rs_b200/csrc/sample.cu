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
// What it measured, and what bounds it: 256 rows of 151,936 logits with top-p
// take 203 us (155 MB from DRAM in each pass). Of the 172,000 cycles of the first
// pass on a multiprocessor with two rows, 87,000 are its exponentials (37 a warp
// for 32 tokens; ten f64 operations of two and a conversion of eight are 28),
// 11,000 the histogram; of the second's 182,000, 37,000 the exponentials of what
// lies above the border, 49,000 queueing them, 30,000 the list. Instruction
// issue is the limit in both. Without a filter 256 rows take 84 us, greedy ones
// 39 us (4.0 TB/s). Few rows are bound by steps that wait for each other, most of
// them for another block's shared memory (700 cycles a read): one row 7 us greedy,
// 18 with a top-k of 20, 30 with top-p.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "sequence.cuh"

namespace cg = cooperative_groups;

namespace strata {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = kThreads;       // of the wide search: a bin a thread
constexpr int kBinBits = 9;
static_assert(kBins == 1 << kBinBits, "a key range is cut into kBins");
constexpr float kBinsPerNat = 16.0f;  // its value histogram: 32 nats, the last bin takes the rest
constexpr int kFine = 2048;           // of the first pass: kPer bins a thread,
constexpr int kPer = kFine / kThreads;
constexpr float kFinePerNat = 64.0f;  // 32 nats
constexpr int kMaxCluster = 8;
constexpr int kList = 4096;           // tokens a list holds
constexpr int kExpTable = 64;
constexpr int kSub = 4;               // parts of a warp's segment whose weights are summed apart

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

// A block's part of what the first pass finds.
struct First {
    double sum;  // of every token's weight, where the row needs it
    float best;  // largest logit and, where the row takes it, its first index
    int index;
};

struct Shared {
    First first;                   // exchanged
    double above;                  // exchanged: mass above the list
    double seg[kWarps * kSub];     // exchanged: weights of the tokens above the list, by part of the slice
    int listed[kWarps];            // exchanged: tokens each warp put into the list (then: crowded bins),
    int listed_part[kWarps * kSub];  // and how many of them by the end of each part
    int block_listed;              // exchanged: their sum
    uint8_t chain[kWarps][kList / 32];  // the pool's groups of 32 that hold them, in order
    int pool_used;
    int offset[kMaxCluster * kWarps + 1];  // of each warp's tokens in the list of the whole row
    int part_end[kMaxCluster * kWarps * kSub];  // and the list's length by the end of each part
    double exp2_table[kExpTable][32];  // a copy a lane: no two lanes meet in a bank
    alignas(16) uint32_t fine[kFine + 32];              // exchanged: the first pass's histogram
    alignas(16) uint32_t share[kFine / 2];  // exchanged: the block's share of the bins, summed over the row (then: the list's counts)
    int won, id;                   // the draw: its segment (-1: id is the token)
    double won_before, total, weight;
    Part part[2];                  // exchanged, alternating
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

    __device__ __forceinline__ void sync() {
        if (ranks == 1) __syncthreads();
        else cluster.sync();
    }
    template <typename T>
    __device__ __forceinline__ const T* of(const T* p, int k) {
        return ranks == 1 ? p : cluster.map_shared_rank(const_cast<T*>(p), k);
    }

    __device__ __forceinline__ int at(int i) const { return index ? index[i] : base + i; }

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
        uint32_t* h = sh.fine + hturn * kBins;  // the first pass is done with its own
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
        const int past = __reduce_min_sync(0xFFFFFFFFu, count && incl >= target ? (int)threadIdx.x : kBins);
        const int last = __reduce_max_sync(0xFFFFFFFFu, count ? (int)threadIdx.x : -1);
        if (lane == 0) atomicMin(&sh.pick_bin, past), atomicMax(&sh.found, last);
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

// above: the mass of kept tokens larger than all of the view's; total: the kept
// tokens' mass (0: above and the view's). Where the border lies outside the view
// the cut stays as it was, and `holds` says so.
__device__ Cut cut_top_p(Row& r, float top, double p, Cut cut, double above = 0.0, double total = 0.0,
                         bool* holds = nullptr) {
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
    if (holds) {
        *holds = target > 0.0 && target <= mass;
        if (!*holds) return cut;
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

// exp by the table method (Tang, 1989): v f + c = (64 m + j) ln2 / 64 + r,
// exp = 2^m 2^(j/64) exp(r), |r| <= ln2 / 128, four terms of exp(r) - 1. Good
// to 4e-14 of the result while |v f + c| < 700. (The whole steps are those of the
// rounded v f + c: from v and c apart they would be off by one where c lies
// between two, and r^5 / 120 thirty times larger.)
struct Exp {
    const double (*table)[32];
    double f, c;
    __device__ Exp(const double (*t)[32], double f_, double c_) : table(t), f(f_), c(c_) {}
    __device__ __forceinline__ double operator()(float v) const {
        constexpr double kLn2 = 0.69314718055994530942, kMagic = 6755399441055744.0;  // 1.5 * 2^52
        const double d = fma((double)v, f, c), t = fma(d, kExpTable / kLn2, kMagic);
        const int n = __double2loint(t);
        const double r = fma(t - kMagic, -kLn2 / kExpTable, d);
        const double b = table[n & (kExpTable - 1)][threadIdx.x & 31];
        const double q = fma(r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0);
        const double y = fma(b * r, q, b);
        return __hiloint2double(__double2hiint(y) + ((n >> 6) << 20), __double2loint(y));
    }
};

// The value histogram of the first pass: bin round(high - v * kFinePerNat), by
// one fused operation whose last bits are the bin, and bounds, all monotone: a
// larger value is never in a later bin. What lies below the last bin has none.
struct Fine {
    float high;  // what falls into bin 0, times kFinePerNat, plus 2^23
    __device__ __forceinline__ unsigned raw(float v) const {
        return __float_as_uint(fmaxf(fmaf(v, -kFinePerNat, high), 8388608.0f)) - 0x4B000000u;
    }
    __device__ __forceinline__ int operator()(float v) const { return (int)min(raw(v), (unsigned)kFine); }
    // The smallest value that falls into bin `b` or an earlier one.
    __device__ float start(int b) const {
        float v = (high - 8388608.0f - (float)b - 0.5f) / kFinePerNat;
        for (int i = 0; i < 64 && (*this)(v) > b; ++i) v = nextafterf(v, INFINITY);
        for (int i = 0; i < 64 && (*this)(nextafterf(v, -INFINITY)) <= b; ++i) v = nextafterf(v, -INFINITY);
        return v;
    }
};

constexpr int kListBytes = kList * 16;     // the pool of this block's tokens, and the row's list
constexpr int64_t kMaxSlice = 124 * 1024;  // bytes of a slice that is kept in shared memory,
constexpr int64_t kPairSlice = 13 * 1024;  // and that leave room for two blocks a multiprocessor

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
        float4 p = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at < hi) p = *reinterpret_cast<const float4*>(x + at);
        v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = element<false>(i, e);
            v[e] = at < hi ? x[at] : -INFINITY;
        }
    }
}

// Inclusive sum over the block's threads, and the total.
__device__ __forceinline__ double block_scan(Shared& sh, double v, double& total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += up;
    }
    __syncthreads();
    if (lane == 31) sh.wsum[0][warp] = v;
    __syncthreads();
    double w = sh.wsum[0][lane % kWarps];
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
        const double up = __shfl_up_sync(0xFFFFFFFFu, w, o, kWarps);
        if (lane % kWarps >= o) w += up;
    }
    total = __shfl_sync(0xFFFFFFFFu, w, kWarps - 1);
    const double before = __shfl_sync(0xFFFFFFFFu, w, warp > 0 ? warp - 1 : 0);
    return (warp > 0 ? before : 0.0) + v;
}

// Among the block's weights w[e] (element threadIdx.x * PER + e), the first
// whose running sum exceeds `target` of the total `u` asks for; the last one
// with a weight where none does (u >= 1, or a border's rounding). -1: none.
template <int PER>
__device__ int pick(Shared& sh, const double (&w)[PER], double u, double offset, double& total, double& weight) {
    double own = 0.0;
#pragma unroll
    for (int e = 0; e < PER; ++e) own += w[e];
    double run = block_scan(sh, own, total) - own;
    const double target = u >= 0.0 ? u * total : offset;
    if (threadIdx.x == 0) sh.pick_bin = INT_MAX, sh.found = -1;
    __syncthreads();
    int past = INT_MAX, last = -1;  // the first past the target, the last with a weight
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        run += w[e];
        if (w[e] > 0.0) {
            last = (int)threadIdx.x * PER + e;
            if (run > target && past == INT_MAX) past = last;
        }
    }
    past = __reduce_min_sync(0xFFFFFFFFu, past), last = __reduce_max_sync(0xFFFFFFFFu, last);
    if ((threadIdx.x & 31) == 0) {
        if (past != INT_MAX) atomicMin(&sh.pick_bin, past);
        if (last >= 0) atomicMax(&sh.found, last);
    }
    __syncthreads();
    const int at = sh.pick_bin != INT_MAX ? sh.pick_bin : sh.found;
    if (at >= 0 && at / PER == (int)threadIdx.x) {
        double upto = run - own;  // the sum up to the element itself
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (e <= at % PER) upto += w[e];
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (at % PER == e) sh.weight = w[e], sh.won_before = upto;
    }
    __syncthreads();
    weight = sh.weight;
    return at;
}

// Sums of two values over the block's threads.
__device__ __forceinline__ void block_sums(Shared& sh, double& a, double& b) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
        b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
    __syncthreads();
    if (lane == 0) sh.wsum[0][warp] = a, sh.wsum[1][warp] = b;
    __syncthreads();
    a = sh.wsum[0][lane % kWarps], b = sh.wsum[1][lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
        b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
    }
}

// The bins of the first pass, kPer a thread: the first ones whose running sums
// reach `low` and `high`; kFine, for what has no bin, if none does.
template <typename W>
__device__ int2 fine_borders(Shared& sh, const W (&weight)[kPer], W low, W high) {
    double own = 0.0, total;
#pragma unroll
    for (int e = 0; e < kPer; ++e) own += (double)weight[e];
    double run = block_scan(sh, own, total) - own;
    if (threadIdx.x == 0) sh.pick_bin = sh.found = kFine;
    __syncthreads();
    int at_low = kFine, at_high = kFine;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        run += (double)weight[e];
        const int bin = (int)threadIdx.x * kPer + e;
        if (weight[e] > 0 && run >= (double)low) at_low = min(at_low, bin);
        if (weight[e] > 0 && run >= (double)high) at_high = min(at_high, bin);
    }
    at_low = __reduce_min_sync(0xFFFFFFFFu, at_low), at_high = __reduce_min_sync(0xFFFFFFFFu, at_high);
    if ((threadIdx.x & 31) == 0) {
        if (at_low < kFine) atomicMin(&sh.pick_bin, at_low);
        if (at_high < kFine) atomicMin(&sh.found, at_high);
    }
    __syncthreads();
    return make_int2(sh.pick_bin, sh.found);
}

// Puts the list's tokens in falling order (equal ones by place): mine[e] is
// token threadIdx.x + e * kThreads on entry and the one of place
// threadIdx.x * PER + e on return; the words order[0 .. listed) are scratch. A
// key is ~key_of(value) << 32 | place, ~0 behind the list. The values' range is
// cut into kFine bins, every token takes a place in its bin, and counts those of
// its bin that precede it. Where a bin has too many for that to be quick they
// are mostly one value (rounded logits), and stay in the list's order. False
// where they are several. (A list of 1000 takes 2 us so; 9 with a bitonic sort.)
template <int PER>
__device__ bool order_list(Shared& sh, unsigned long long (&mine)[PER], const float* list, unsigned long long* order,
                           int listed) {
    constexpr uint32_t kCrowd = 256;
    static_assert(PER * kThreads / kCrowd <= kWarps, "room for the crowded bins' numbers");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t first = 0xFFFFFFFFu, last = 0u;  // keys
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const uint32_t key = ~(uint32_t)(mine[e] >> 32);
        if (e * kThreads + (int)threadIdx.x < listed) first = min(first, key), last = max(last, key);
    }
    first = __reduce_min_sync(0xFFFFFFFFu, first), last = __reduce_max_sync(0xFFFFFFFFu, last);
    if (lane == 0) sh.wlo[warp] = first, sh.whi[warp] = last;
    reinterpret_cast<uint4*>(sh.fine)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const float low = logit_of(__reduce_min_sync(0xFFFFFFFFu, sh.wlo[lane % kWarps]));
    const float high = logit_of(__reduce_max_sync(0xFFFFFFFFu, sh.whi[lane % kWarps]));
    // monotone, whatever the range: infinite ones make it one bin
    const float scale = high > low ? (float)(kFine - 1) / (high - low) : 0.0f;
    auto bin_of = [&](uint32_t key) {
        return (uint32_t)fminf(fmaxf((high - logit_of(key)) * scale, 0.0f), (float)(kFine - 1));
    };
    uint32_t bin[PER], at[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        bin[e] = bin_of(~(uint32_t)(mine[e] >> 32));
        if (e * kThreads + (int)threadIdx.x < listed) at[e] = atomicAdd(&sh.fine[bin[e]], 1u);
    }
    __syncthreads();
    const uint4 c = reinterpret_cast<const uint4*>(sh.fine)[threadIdx.x];
    if (threadIdx.x == 0) sh.pick_bin = 0;
    const bool crowded = __syncthreads_or(max(max(c.x, c.y), max(c.z, c.w)) > kCrowd);
    if (crowded) {
        const uint32_t n[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n[e] > kCrowd) sh.listed[atomicAdd(&sh.pick_bin, 1)] = (int)threadIdx.x * 4 + e;
    }
    const uint32_t own = c.x + c.y + c.z + c.w;
    uint32_t incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) sh.wn[warp] = (int)incl;
    __syncthreads();
    const uint32_t before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? (uint32_t)sh.wn[lane % kWarps] : 0u) + incl - own;
    reinterpret_cast<uint4*>(sh.fine)[threadIdx.x] =
        make_uint4(before, before + c.x, before + c.x + c.y, before + c.x + c.y + c.z);
    if (threadIdx.x == 0) sh.fine[kFine] = (uint32_t)listed;
    __syncthreads();
    uint32_t lone = 0;  // tokens in bins that are not crowded
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const uint32_t from = sh.fine[bin[e]], to = sh.fine[bin[e] + 1];
        if (e * kThreads + (int)threadIdx.x >= listed || to - from > kCrowd) continue;
        lone |= 1u << e;
        order[from + at[e]] = mine[e];
    }
    if (crowded) {
        // every warp has a stretch of the list and counts what it holds of each
        // crowded bin (lane q of bin q), then puts these behind earlier warps'
        const int crowds = sh.pick_bin, stretch = (listed + kWarps * 32 - 1) / (kWarps * 32) * 32;
        const int lo = warp * stretch, hi = min(lo + stretch, listed);
        const uint32_t own_crowd = lane < crowds ? (uint32_t)sh.listed[lane] : kFine;
        uint32_t to = 0;
        for (int i = lo + lane; i - lane < hi; i += 32) {
            const uint32_t b = i < hi ? bin_of(key_of(list[i])) : kFine;
            for (int q = 0; q < crowds; ++q) {
                const unsigned votes = __ballot_sync(0xFFFFFFFFu, b == __shfl_sync(0xFFFFFFFFu, own_crowd, q));
                if (lane == q) to += __popc(votes);
            }
        }
        sh.share[warp * 32 + lane] = to;
        __syncthreads();
        to = lane < crowds ? sh.fine[own_crowd] : 0;
        for (int w = 0; w < warp; ++w) to += sh.share[w * 32 + lane];
        for (int i = lo + lane; i - lane < hi; i += 32) {
            const uint32_t key = i < hi ? key_of(list[i]) : 0u, b = i < hi ? bin_of(key) : kFine;
            for (int q = 0; q < crowds; ++q) {
                const bool in = b == __shfl_sync(0xFFFFFFFFu, own_crowd, q);
                const unsigned votes = __ballot_sync(0xFFFFFFFFu, in);
                const uint32_t start = __shfl_sync(0xFFFFFFFFu, to, q);
                if (in) order[start + __popc(votes & ((1u << lane) - 1u))] = (unsigned long long)~key << 32 | (unsigned)i;
                if (lane == q) to += __popc(votes);
            }
        }
        __syncthreads();
        bool mixed = false;
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (e * kThreads + (int)threadIdx.x < listed && !(lone >> e & 1))
                mixed |= (uint32_t)(order[sh.fine[bin[e]]] >> 32) != (uint32_t)(mine[e] >> 32);
        if (__syncthreads_or(mixed)) return false;
    } else {
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        if (!(lone >> e & 1)) continue;
        const uint32_t from = sh.fine[bin[e]], to = sh.fine[bin[e] + 1];
        at[e] = from;
#pragma unroll 4
        for (uint32_t i = from; i < to; ++i) at[e] += order[i] < mine[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e)
        if (lone >> e & 1) order[at[e]] = mine[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int i = (int)threadIdx.x * PER + e;
        mine[e] = i < listed ? order[i] : ~0ull;
    }
    return true;
}

// The search over whole slices: for rows whose cut no list holds.
__device__ void sample_wide(Row& r, const float* logits, float top, uint32_t k, float p, float mp, float t, double u,
                            int& id, float& logp) {
    Shared& sh = r.sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Cut cut{1u, INT_MAX};  // no element has key 1: everything but the excluded
    if (k > 0) cut = cut_top_k(r, top, k);
    if (p < 1.0f) cut = cut_top_p(r, top, (double)p, cut);
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
    const double target = u * all;
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
        const bool skip = (!here && u < 1.0 && from + w < target * (1.0 - 1e-9)) || from > target * (1.0 + 1e-9);
        double run = from;
        if (!skip)
            for (int i = lo; i < hi; i += 32) {
                const double wi = i + lane < hi ? weight(r.x[i + lane], r.base + i + lane) : 0.0;
                double incl = wi;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                    if (lane >= o) incl += up;
                }
                if (wi > 0.0) {
                    last = max(last, (uint32_t)(r.base + i + lane) + 1u);
                    if (run + incl > target) found = min(found, (uint32_t)(r.base + i + lane));
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

// The first element, in index order, of [lo, hi) of the block's slice whose
// running sum of weights exceeds `target`: the warps sum a part each, then the
// block looks at the one part that holds it.
template <typename W>
__device__ int locate(Row& r, int lo, int hi, double target, double& weight_out, W weight) {
    Shared& sh = r.sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    while (hi - lo > 2 * kThreads) {
        const int part = ((hi - lo + kThreads - 1) / kThreads) * 32;
        const int from = min(lo + warp * part, hi), to = min(from + part, hi);
        double w = 0.0;
        for (int i = from + lane; i < to; i += 32) w += weight(r.x[i], r.base + i);
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
        __syncthreads();
        if (lane == 0) sh.wsum[1][warp] = w;
        __syncthreads();
        double run = 0.0, before = 0.0;
        int at = -1;  // the first part past the target, else the last with a weight
        for (int k = 0; k < kWarps; ++k) {
            const double wk = sh.wsum[1][k];
            if (wk > 0.0) at = k, before = run;
            run += wk;
            if (wk > 0.0 && run > target) break;
        }
        __syncthreads();
        if (at < 0) return -1;
        const int end = hi;
        lo = min(lo + at * part, end), hi = min(lo + part, end);
        target -= before;
    }
    double w[2], total;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = lo + (int)threadIdx.x * 2 + e;
        w[e] = i < hi ? weight(r.x[i], r.base + i) : 0.0;
    }
    const int at = pick<2>(sh, w, -1.0, target, total, weight_out);
    return at < 0 ? -1 : r.base + lo + at;
}

// The list's order and cut. On entry list holds `listed` tokens in index order;
// on return out[i] is token i's weight in the draw (0 where it is not kept).
// above: mass of larger tokens outside the list; all: mass that p refers to
// (0: that of the first k). 0 where the border of p lies outside a list that has
// tokens above it, -1 where too many are nearly equal to be put in order, else 1.
// A thread holds PER neighbours of the order.
template <int PER, typename M, typename D>
__device__ int settle_list(Shared& sh, const float* list, unsigned long long* order, double* out, int listed, int k,
                           float p, double above, double all, bool sure, M mass, D draw) {
    unsigned long long mine[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int i = e * kThreads + threadIdx.x;
        mine[e] = i < listed ? (unsigned long long)~key_of(list[i]) << 32 | (unsigned)i : ~0ull;
    }
    if (!order_list<PER>(sh, mine, list, order, listed)) return -1;
    int kept = k > 0 && k < listed ? k : listed;
    bool holds = true;
    if (p < 1.0f) {
        double m[PER], own = 0.0, total;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            m[e] = (int)threadIdx.x * PER + e < kept ? mass(logit_of(~(uint32_t)(mine[e] >> 32))) : 0.0;
            own += m[e];
        }
        double run = above + (block_scan(sh, own, total) - own);
        const double target = (double)p * (all > 0.0 ? all : total);
        if (sure) holds = target > above && target <= above + total;
        if (threadIdx.x == 0) sh.found = 1;  // the first token always stays
        __syncthreads();
        int last = 0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int r = threadIdx.x * PER + e;
            if (r < kept && run < target) last = r + 1;
            run += m[e];
        }
        last = __reduce_max_sync(0xFFFFFFFFu, last);
        if ((threadIdx.x & 31) == 0) atomicMax(&sh.found, last);
        __syncthreads();
        kept = sh.found;
    }
    __syncthreads();  // every thread holds its part of the order; its place takes the weights
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int r = threadIdx.x * PER + e;
        if (r < listed) out[(uint32_t)mine[e]] = r < kept ? draw(logit_of(~(uint32_t)(mine[e] >> 32))) : 0.0;
    }
    __syncthreads();
    return holds;
}

// Two blocks a multiprocessor hold a thread to 64 registers, which spill (a frame
// of 112 bytes). Where all rows run at once, one block without spills would do
// better (top-p: a row of 32,003 19.8 us against 20.3, 148 rows of 151,936 86
// against 114); where rows queue, two hide each other's steps (1500 rows of 257
// 104 us against 158, 2000 of 32,003 367 against 428).
template <bool PACKS>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    float* pool = reinterpret_cast<float*>(dynamic);  // this block's tokens for the list: values, then indices
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
    const int seg = ((n + kWarps * 256 - 1) / (kWarps * 256)) * 256;
    Row r{a, sh, a.resident ? held : logits + base, nullptr, base, n, seg, rank, ranks, 0, 0, cluster};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int lo = min(warp * seg, n), hi = min(lo + seg, n);
    const int part = ((seg / 256 + kSub - 1) / kSub) * 256;  // elements of a part of the segment

    const float t = a.temperature ? a.temperature[row] : 1.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    if (k < 0 || k >= a.vocab) k = 0;
    float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f;
    if (!(p < 1.0f)) p = 1.0f;
    if (!(mp > 0.0f)) mp = 0.0f;
    double u = a.uniform[row];
    u = u > 0.0 ? u : 0.0;
    // rows that take the largest logit; at a positive temperature it has all the weight
    const bool greedy = !(t > 0.0f) || p <= 0.0f || mp > 1.0f || k == 1;
    const double inv_t = 1.0 / (double)t;
    const bool sums_all = !greedy && k == 0 && (p < 1.0f || mp == 0.0f);  // the first pass sums every weight,
    const bool draws_all = sums_all && p >= 1.0f;                         // at the draw's temperature

    // Where the histogram lies and what the sums refer to: the largest of a
    // sample of the row, the same for all its blocks.
    const bool exps = !greedy && (sums_all || p < 1.0f);
    if (exps && threadIdx.x < kExpTable) reinterpret_cast<double*>(sh.share)[threadIdx.x] = exp2((double)threadIdx.x / kExpTable);
    if (threadIdx.x == 0) sh.pool_used = 0;
    if (threadIdx.x < kWarps * kSub) sh.seg[threadIdx.x] = 0.0, sh.listed_part[threadIdx.x] = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) sh.fine[threadIdx.x * kPer + e] = 0;
    float center = -INFINITY;
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // 32 neighbours from each of 32 places
        const int64_t at = (int64_t)(warp * 2 + e) * a.vocab / (2 * kWarps) + lane;
        if (at < a.vocab) center = fmaxf(center, logits[at]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) center = fmaxf(center, __shfl_xor_sync(0xFFFFFFFFu, center, o));
    if (lane == 0) sh.wlo[warp] = __float_as_uint(center);
    __syncthreads();
    if (exps) {
#pragma unroll
        for (int i = 0; i < kExpTable / kWarps; ++i)
            sh.exp2_table[i * kWarps + warp][lane] = reinterpret_cast<const double*>(sh.share)[i * kWarps + warp];
    }
    center = __uint_as_float(sh.wlo[lane % kWarps]);
    // the fourth largest of the warps' maxima: six in a thousand tokens or so are above it
    int larger = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const float other = __shfl_sync(0xFFFFFFFFu, center, w);
        larger += other > center || (other == center && w < lane % kWarps);
    }
    float upper = __shfl_sync(0xFFFFFFFFu, center, __ffs(__ballot_sync(0xFFFFFFFFu, larger == 3)) - 1);
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) center = fmaxf(center, __shfl_xor_sync(0xFFFFFFFFu, center, o));
    __syncthreads();
    reinterpret_cast<uint2*>(sh.share)[threadIdx.x] = make_uint2(0, 0);
    // a masked sample, or values too large for the bins
    if (!(fabsf(center) < 1e4f)) center = upper = 0.0f;
    if (!(fabsf(upper) < 1e4f)) upper = center;
    // Top-p's border is mostly below the few largest tokens: they share the
    // first bin, whose mass follows from the sum and needs no estimate.
    const bool sure = sums_all && p < 1.0f && mp == 0.0f;  // tokens above the border's bins are not listed
    const Fine bin_of{(sure ? upper : center + 8.0f) * kFinePerNat + 8388608.0f};
    const double ref = (double)center;
    const Exp mass(sh.exp2_table, 1.0, -ref);                  // relative to the sample's maximum
    const Exp draw(sh.exp2_table, inv_t, -ref * inv_t);
    // what lies so far below it that its exponential is zero at either temperature
    auto lowest = [](double x) { return x > -3e38 ? (float)x : -INFINITY; };
    const float mass_floor = (float)(ref - 600.0), draw_floor = lowest(ref - 600.0 * (double)t);

    // first pass
    {
        double sum = 0.0;
        float best = -INFINITY;
        int index = INT_MAX;
        constexpr int STEPS = 2;  // loads in flight, eight elements a lane
        const float floor_of = draws_all ? draw_floor : mass_floor;
        const Exp f(sh.exp2_table, draws_all ? inv_t : 1.0, draws_all ? -ref * inv_t : -ref);
        int next = part;  // where the part ends
        double before = 0.0;
        // The slice comes in by asynchronous copies, kAhead steps ahead, each
        // lane's elements by itself: into place where the slice is kept, else
        // into a ring of the warp's own.
        constexpr int kAhead = 3, kStep = 128 * STEPS;
        float* ring = pool + warp * (4 * kStep);
        auto place = [&](int i, int step) { return a.resident ? held + i : ring + (step & 3) * kStep; };
        auto copy = [&](int i, int step) {
            if (i < hi) {
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(place(i, step));
#pragma unroll
                for (int q = 0; q < STEPS; ++q)
#pragma unroll
                    for (int e = 0; e < (PACKS ? 1 : 4); ++e) {
                        const int at = element<PACKS>(128 * q, e);
                        if (i + at < hi)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(dst + at * 4),
                                         "l"(logits + base + i + at), "n"(PACKS ? 16 : 4)
                                         : "memory");
                    }
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        };
#pragma unroll
        for (int d = 0; d < kAhead; ++d) copy(lo + d * kStep, d);
        float v[STEPS][4];
        for (int i = lo, step = 0; i < hi; i += kStep, ++step) {
            copy(i + kAhead * kStep, step + kAhead);
            asm volatile("cp.async.wait_group %0;\n" ::"n"(kAhead) : "memory");
            const float* in = place(i, step);
#pragma unroll
            for (int q = 0; q < STEPS; ++q) load4<PACKS>(in, 128 * q, hi - i, v[q]);
            if (greedy) {
#pragma unroll
                for (int q = 0; q < STEPS; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (v[q][e] > best) best = v[q][e], index = base + element<PACKS>(i + 128 * q, e);
                continue;
            }
#pragma unroll
            for (int q = 0; q < STEPS; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    best = fmaxf(best, v[q][e]);              // a NaN is passed over,
                    v[q][e] = fmaxf(v[q][e], floor_of);       // and counts, as -inf does, as nothing
                }
            if (!draws_all) {
#pragma unroll
                for (int q = 0; q < STEPS; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e)  // what has no bin goes to a word of the lane's own
                        atomicAdd(&sh.fine[min(bin_of.raw(v[q][e]), (unsigned)(kFine + lane))], 1u);
            }
            if (sums_all) {
#pragma unroll
                for (int q = 0; q < STEPS; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += f(v[q][e]);
                if (draws_all && (i + 128 * STEPS - lo >= next || i + 128 * STEPS >= hi)) {
                    double w = sum - before;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
                    if (lane == 0) sh.seg[warp * kSub + next / part - 1] = w;
                    before = sum, next += part;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float b2 = __shfl_xor_sync(0xFFFFFFFFu, best, o);
            const int i2 = __shfl_xor_sync(0xFFFFFFFFu, index, o);
            if (b2 > best || (b2 == best && i2 < index)) best = b2, index = i2;
            sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        }
        if (lane == 0) {
            sh.wsum[0][warp] = sum;
            sh.wlo[warp] = __float_as_uint(best), sh.whi[warp] = (uint32_t)index;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            First m{0.0, -INFINITY, INT_MAX};
            for (int w = 0; w < kWarps; ++w) {
                const float b2 = __uint_as_float(sh.wlo[w]);
                const int i2 = (int)sh.whi[w];
                if (b2 > m.best || (b2 == m.best && i2 < m.index)) m.best = b2, m.index = i2;
                m.sum += sh.wsum[0][w];
            }
            sh.first = m;
        }
    }
    r.sync();
    First m{0.0, -INFINITY, INT_MAX};
    if (lane < ranks) m = *r.of(&sh.first, lane);
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
        const float b2 = __shfl_xor_sync(0xFFFFFFFFu, m.best, o);
        const int i2 = __shfl_xor_sync(0xFFFFFFFFu, m.index, o);
        if (b2 > m.best || (b2 == m.best && i2 < m.index)) m.best = b2, m.index = i2;
        m.sum += __shfl_xor_sync(0xFFFFFFFFu, m.sum, o);
    }
    m.best = __shfl_sync(0xFFFFFFFFu, m.best, 0), m.index = __shfl_sync(0xFFFFFFFFu, m.index, 0);
    m.sum = __shfl_sync(0xFFFFFFFFu, m.sum, 0);
    const float top = m.best;
    if (!(top > -INFINITY) || greedy) {
        if (rank == 0 && threadIdx.x == 0) {
            a.ids[row] = top > -INFINITY ? m.index : -1;
            if (a.logprobs) a.logprobs[row] = top > -INFINITY ? 0.0f : -INFINITY;
        }
        if (ranks > 1) cluster.sync();  // no block leaves while another may read its shared memory
        return;
    }

    // Which bins the list takes ([first, last]); bins before it are kept for sure.
    int first = 0, last = -1;
    // a range that the sample misjudged, or infinite logits
    bool wide = sums_all && !(m.sum > 1e-100 && m.sum < 1e250 && top < center + 500.0f * fminf(t, 1.0f));
    // or a temperature so small that the rounded floor lies outside the exponential's range, or so large that none is left
    wide |= sums_all && !((ref - (double)draw_floor) * inv_t < 700.0);
    // Excluded tokens have weighed e^-600 each in the sums: nothing, unless the
    // draw asks for the very first or last token with a weight.
    if ((sure || draws_all) && !(u > 1e-100 && u < 1.0 - 1e-9)) wide = true;
    if (!draws_all && !wide) {
        uint4 c;
        if (ranks == 1) {
            c = reinterpret_cast<const uint4*>(sh.fine)[threadIdx.x];
        } else {
            // Each block sums its share of the bins over all blocks, then all
            // read the sums: what crosses between multiprocessors (10 bytes a
            // cycle) is a quarter of all histograms read by all.
            const int quads = kFine / 4 / ranks;  // of a share; as many threads read from each block
            const int quad = threadIdx.x % quads, from = threadIdx.x / quads;
            const uint4 part = reinterpret_cast<const uint4*>(r.of(sh.fine, from))[rank * quads + quad];
            atomicAdd(&sh.share[quad * 4], part.x), atomicAdd(&sh.share[quad * 4 + 1], part.y);
            atomicAdd(&sh.share[quad * 4 + 2], part.z), atomicAdd(&sh.share[quad * 4 + 3], part.w);
            cluster.sync();
            c = reinterpret_cast<const uint4*>(r.of(sh.share, from))[quad];
        }
        const uint32_t count[kPer] = {c.x, c.y, c.z, c.w};
        if (!sure) {
            // top-p behind top-k needs the mass of all k; otherwise nothing below min-p's bin matters
            last = mp > 0.0f && !(k > 0 && p < 1.0f)
                       ? bin_of(__double2float_rd((double)top + log((double)mp) - 1e-4))
                       : kFine;
            if (k > 0) {
                const int by_k = fine_borders<uint32_t>(sh, count, (uint32_t)k, (uint32_t)k).x;
                if (by_k > last) k = 0;  // what min-p keeps is less than k
                else last = by_k;
            }
        } else {
            // The bins around the border. A bin's tokens are estimated at its
            // middle, each off by 1/128 of its mass at most and by independent
            // amounts: six spreads of their sum (a spread of 1/222 each), and
            // 1e-4 for bins on a slope. What has no bin is below e^-24 a token.
            // The first bin takes what the sum has beyond the others. Where
            // that is not enough, the list does not hold the border and the
            // wide search settles the row.
            double guess[kPer], others = 0.0, spread = 0.0;
            double one = exp(((double)bin_of.high - 8388608.0 - (double)(threadIdx.x * kPer)) / kFinePerNat - ref);
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                guess[e] = threadIdx.x * kPer + e ? (double)count[e] * one : 0.0;
                others += guess[e], spread += guess[e] * one;
                one *= 0.98449643700540845;  // exp(-1 / kFinePerNat)
            }
            block_sums(sh, others, spread);
            if (threadIdx.x == 0) guess[0] = fmax(m.sum - others, 0.0);
            const double border = (double)p * m.sum;
            const double none = 3.8e-11 * (double)a.vocab;
            const double off = fmin(m.sum / 125.0, 6.0 / 222.0 * sqrt(spread) + 1e-4 * m.sum) + none;
            const int2 at = fine_borders<double>(sh, guess, border - off, border + off);
            first = at.x, last = at.y;
        }
    }

    // second pass: the list's tokens, and the sums of what lies above them
    int listed = 0;
    double above = 0.0;
    if (!draws_all && !wide) {
        // the bins' borders as values: the list takes v >= from, those above it v >= over
        const float from = last == kFine ? -INFINITY : bin_of.start(last);
        const float over = first == 0 ? INFINITY : bin_of.start(first - 1);
        double sum = 0.0, weights = 0.0;
        int mine = 0, waiting = 0, next = part;
        // Values above the list wait in a column of the lane's own (the list's
        // place, not needed yet), so that their exponentials are computed with
        // most of the warp's lanes at work.
        constexpr int kStep = 256, kDeep = 16;
        float* queue = list + warp * (kDeep * 32) + lane;
        auto drain = [&] {
            for (int d = 0; __any_sync(0xFFFFFFFFu, d < waiting); ++d)
                if (d < waiting) {
                    const float w = queue[d * 32];
                    const double e = mass(w);
                    sum += e;
                    weights += t == 1.0f ? e : draw(fmaxf(w, draw_floor));
                }
            waiting = 0;
        };
        float v[2][4], ahead[2][4];
#pragma unroll
        for (int q = 0; q < 2; ++q) load4<PACKS>(r.x, lo + 128 * q, hi, ahead[q]);
        for (int i = lo; i < hi; i += kStep) {
            bool take = false;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[q][e] = ahead[q][e];
                load4<PACKS>(r.x, i + kStep + 128 * q, hi, ahead[q]);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = v[q][e] >= over;  // over is infinite where nothing is sure
                    if (sure) queue[waiting * 32] = v[q][e];  // the next one overwrites what does not count
                    waiting += in && sure;
                    take |= v[q][e] >= from && v[q][e] > -INFINITY && !(in && sure);
                }
            if (sure && __any_sync(0xFFFFFFFFu, waiting > kDeep - 8)) drain();
            if (__any_sync(0xFFFFFFFFu, take)) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    int bits = 0, pos[4], all = 0;  // places of these tokens, in index order
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        bits |= (v[q][e] >= from && v[q][e] > -INFINITY && !(sure && v[q][e] >= over)) << e;
                    const unsigned some = __ballot_sync(0xFFFFFFFFu, bits);
                    if (!some) continue;
                    if (PACKS) {
                        const int c = __popc(bits);
                        int before = __popc(some & ((1u << lane) - 1u));
                        all = __popc(some);
                        if (__any_sync(0xFFFFFFFFu, c > 1)) {
                            int incl = c;
#pragma unroll
                            for (int o = 1; o < 32; o <<= 1) {
                                const int up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                                if (lane >= o) incl += up;
                            }
                            all = __shfl_sync(0xFFFFFFFFu, incl, 31);
                            before = incl - c;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) pos[e] = before + __popc(bits & ((1 << e) - 1));
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const unsigned votes = __ballot_sync(0xFFFFFFFFu, bits >> e & 1);
                            pos[e] = all + __popc(votes & ((1u << lane) - 1u));
                            all += __popc(votes);
                        }
                    }
                    if ((mine + 31) / 32 < (mine + all + 31) / 32) {
                        if (lane == 0)  // groups of 32 from the pool, up to the last of them
                            for (int g = (mine + 31) / 32; g < (mine + all + 31) / 32; ++g) {
                                const int got = atomicAdd(&sh.pool_used, 1);
                                if (g < kList / 32) sh.chain[warp][g] = (uint8_t)min(got, kList / 32 - 1);
                            }
                        __syncwarp();
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int slot = mine + pos[e];
                        if ((bits >> e & 1) && slot < kList) {
                            const int to = sh.chain[warp][slot / 32] * 32 + slot % 32;
                            pool[to] = v[q][e];
                            pool_index[to] = base + element<PACKS>(i + 128 * q, e);
                        }
                    }
                    mine += all;
                }
            }
            if (sure && (i + kStep - lo >= next || i + kStep >= hi)) {  // a part ends
                drain();
                double w = weights;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
                if (lane == 0) sh.seg[warp * kSub + next / part - 1] = w, sh.listed_part[warp * kSub + next / part - 1] = mine;
                weights = 0.0, next += part;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (lane == 0) sh.listed[warp] = mine, sh.wsum[1][warp] = sum;
        if (lane == 0)
            for (int e = next / part - 1; e < kSub; ++e) sh.listed_part[warp * kSub + e] = mine;
        __syncthreads();
        if (warp == 0) {
            double s = sh.wsum[1][lane % kWarps];
            int c = sh.listed[lane % kWarps];
#pragma unroll
            for (int o = kWarps / 2; o > 0; o >>= 1) {
                s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
                c += __shfl_xor_sync(0xFFFFFFFFu, c, o);
            }
            // more than the pool holds
            if (lane == 0) sh.above = s, sh.block_listed = sh.pool_used > kList / 32 ? kList + 1 : c;
        }
        r.sync();
        if (lane < ranks) listed = *r.of(&sh.block_listed, lane), above = *r.of(&sh.above, lane);
#pragma unroll
        for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
            listed += __shfl_xor_sync(0xFFFFFFFFu, listed, o);
            above += __shfl_xor_sync(0xFFFFFFFFu, above, o);
        }
        listed = __shfl_sync(0xFFFFFFFFu, listed, 0), above = __shfl_sync(0xFFFFFFFFu, above, 0);
        if (listed > kList) wide = true;  // every block sees the same sum
    }

    // The first block settles the cut; the draw is one of the list's tokens,
    // or lies in one warp's segment of the row.
    if (!wide) {
        double* weight_of = reinterpret_cast<double*>(pool);  // of the list's tokens: the pool has been read by then
        if (rank == 0) {
            const int segs = ranks * kWarps;
            bool holds = true;
            if (threadIdx.x == 0) sh.won = -1;
            if (!draws_all) {
                if (warp == 0) {  // where each warp's tokens start in the list
                    int before = 0, c[kMaxCluster * kWarps / 32];
#pragma unroll
                    for (int q = 0; q < kMaxCluster * kWarps / 32; ++q) {
                        const int g = min(q * 32 + lane, segs - 1);
                        c[q] = r.of(sh.listed, g / kWarps)[g % kWarps];
                    }
#pragma unroll
                    for (int q = 0; q < kMaxCluster * kWarps / 32; ++q) {
                        const int g = q * 32 + lane, own = g < segs ? c[q] : 0;
                        int incl = own;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const int up = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                            if (lane >= o) incl += up;
                        }
                        if (g < segs) sh.offset[g] = before + incl - own;
                        before += __shfl_sync(0xFFFFFFFFu, incl, 31);
                    }
                    if (lane == 0) sh.offset[segs] = before;
                }
                __syncthreads();
                for (int i = threadIdx.x; i < listed; i += kThreads) {
                    int g = 0, end = segs;  // the warp that put it there: offset[g] <= i < offset[g + 1]
                    while (end - g > 1) {
                        const int mid = (g + end) >> 1;
                        if (sh.offset[mid] <= i) g = mid;
                        else end = mid;
                    }
                    const int q = g / kWarps, at = i - sh.offset[g];
                    const int from = r.of(&sh.chain[0][0], q)[(g % kWarps) * (kList / 32) + at / 32] * 32 + at % 32;
                    list[i] = r.of(pool, q)[from];
                    list_index[i] = r.of(pool_index, q)[from];
                }
                if (sure)
                    for (int g = threadIdx.x; g < segs * kSub; g += kThreads)
                        sh.part_end[g] = sh.offset[g / kSub] + r.of(sh.listed_part, g / (kWarps * kSub))[g % (kWarps * kSub)];
                __syncthreads();
                const double least = (double)mp, log_least = mp > 0.0f ? log(least) : 0.0;
                auto kept_weight = [&](float v) -> double {
                    const double d = below(v, top);
                    // min-p's comparison of exponentials, decided by the logs unless they are close
                    if (mp > 0.0f && (d < log_least - 1e-9 || (d < log_least + 1e-9 && exp(d) < least))) return 0.0;
                    if (sure) return v > draw_floor ? draw(v) : 0.0;
                    return d == 0.0 ? 1.0 : d < -1e300 ? 0.0 : exp(d * inv_t);
                };
                auto list_mass = [&](float v) -> double {
                    if (sums_all) return v > mass_floor ? mass(v) : 0.0;
                    return exp(below(v, top));
                };
                unsigned long long* order = reinterpret_cast<unsigned long long*>(pool);
                const double all = sums_all ? m.sum : 0.0;
                auto settle = [&](auto per) {
                    return settle_list<decltype(per)::value>(sh, list, order, weight_of, listed, k, p, above, all, sure,
                                                             list_mass, kept_weight);
                };
                int settled = -1;
                if (listed <= kThreads) settled = settle(std::integral_constant<int, 1>());
                else if (listed <= 2 * kThreads) settled = settle(std::integral_constant<int, 2>());
                else if (listed <= 4 * kThreads) settled = settle(std::integral_constant<int, 4>());
                else settled = settle(std::integral_constant<int, 8>());
                holds = settled != 0;
                if (settled < 0) {  // the search by key ranges, on the list
                    Row l{a, sh, list, list_index, 0, listed, ((listed + kThreads - 1) / kThreads) * 32, 0, 1, 0, 0, cluster};
                    Cut cut{1u, INT_MAX};
                    if (k > 0 && k < listed) cut = cut_top_k(l, top, (uint32_t)k);
                    if (p < 1.0f) {
                        const double scale = sums_all ? exp(ref - (double)top) : 1.0;
                        bool inside = true;
                        cut = cut_top_p(l, top, (double)p, cut, above * scale, all * scale, sums_all ? &inside : nullptr);
                        holds = inside || !sure;  // behind a list that ends at min-p it cuts nothing
                    }
                    __syncthreads();
                    for (int i = threadIdx.x; i < listed; i += kThreads)
                        weight_of[i] = cut.keeps(key_of(list[i]), list_index[i]) ? kept_weight(list[i]) : 0.0;
                    __syncthreads();
                }
            }
            if (!holds) {
                if (threadIdx.x == 0) sh.won = -2;
            } else if (!sure && !draws_all) {
                constexpr int PER = kList / kThreads;
                double total, weight;
                int at;
                if (listed <= kThreads) {
                    const double w[1] = {(int)threadIdx.x < listed ? weight_of[threadIdx.x] : 0.0};
                    at = pick<1>(sh, w, u, 0.0, total, weight);
                } else {
                    double w[PER];
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        const int i = threadIdx.x * PER + e;
                        w[e] = i < listed ? weight_of[i] : 0.0;
                    }
                    at = pick<PER>(sh, w, u, 0.0, total, weight);
                }
                if (threadIdx.x == 0) sh.id = list_index[at], sh.weight = weight, sh.total = total;
            } else {
                // each part's weights: what lies above the list, and its kept tokens of the list
                constexpr int PER = kMaxCluster * kWarps * kSub / kThreads;
                const int parts = segs * kSub;
                double w[PER], total, weight;
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int g = threadIdx.x * PER + e;
                    w[e] = 0.0;
                    if (g < parts) {
                        w[e] = r.of(sh.seg, g / (kWarps * kSub))[g % (kWarps * kSub)];
                        if (!draws_all)
                            for (int i = g ? sh.part_end[g - 1] : 0; i < sh.part_end[g]; ++i) w[e] += weight_of[i];
                    }
                }
                const int won = pick<PER>(sh, w, u, 0.0, total, weight);
                if (threadIdx.x == 0) {
                    // a temperature that takes the weights out of range
                    sh.won = total > 1e-100 && total < 1e250 ? won : -2;
                    sh.won_before = u * total - (sh.won_before - weight);  // the target within the segment
                    sh.total = total;
                }
            }
        }
        r.sync();
        const int won = *r.of(&sh.won, 0);
        const double total = *r.of(&sh.total, 0);
        if (won >= 0 && won / (kWarps * kSub) == rank) {
            const int at = won % (kWarps * kSub), end = min((at / kSub + 1) * seg, n);
            const int from = min((at / kSub) * seg + (at % kSub) * part, end), to = min(from + part, end);
            const double target = *r.of(&sh.won_before, 0);
            const double* all_weights = r.of(weight_of, 0);
            const int* all_index = r.of(list_index, 0);
            const int* ends = r.of(sh.part_end, 0);
            const int l0 = draws_all || won == 0 ? 0 : ends[won - 1], l1 = draws_all ? 0 : ends[won];
            double w;
            const int got = locate(r, from, to, target, w, [&](float v, int i) -> double {
                if (!(v > draw_floor)) return 0.0;
                if (draws_all) return draw(v);
                const int b = bin_of(v);
                if (b > last) return 0.0;
                if (b < first) return draw(v);
                int lo_i = l0, hi_i = l1;  // a token of the list: its weight there
                while (hi_i - lo_i > 1) {
                    const int mid = (lo_i + hi_i) >> 1;
                    if (all_index[mid] <= i) lo_i = mid;
                    else hi_i = mid;
                }
                return all_weights[lo_i];
            });
            if (threadIdx.x == 0) {
                a.ids[row] = got;
                if (a.logprobs) a.logprobs[row] = (float)log(w / total);
            }
        }
        if (won == -1 && rank == 0 && threadIdx.x == 0) {
            a.ids[row] = sh.id;
            if (a.logprobs) a.logprobs[row] = (float)log(sh.weight / sh.total);
        }
        if (ranks > 1) cluster.sync();  // the first block's words have been read
        if (won != -2) return;
    }
    int id;
    float logp;
    r.turn = 0, r.hturn = 0;  // the same in every block
    if (k > 0) {  // against the tokens that can be taken
        Part alive{0.0, 0.0, 0u, 0u, 0};
        r.each([&](float v, int) { alive.n += v > -INFINITY; });
        if (k >= r.reduce(alive).n) k = 0;
    }
    sample_wide(r, logits, top, (uint32_t)k, p, mp, t, u, id, logp);
    if (rank == 0 && threadIdx.x == 0) {
        a.ids[row] = id;
        if (a.logprobs) a.logprobs[row] = logp;
    }
    if (ranks > 1) cluster.sync();
}

}  // namespace
}  // namespace strata

using namespace strata;

// How many clusters of `ranks` blocks the context's device (the current one)
// runs at once with a block a multiprocessor: fewer than its multiprocessors
// divided by `ranks` (15 of 8 on 148), as a cluster stays within a part of them.
static int64_t clusters_at_once(strata_ctx* ctx, int ranks) {
    static std::atomic<int> known[64][4];
    std::atomic<int>* slot = ctx->device < 64 ? &known[ctx->device][ranks == 8 ? 3 : ranks / 2] : nullptr;
    int n = slot ? slot->load(std::memory_order_relaxed) : 0;
    if (n > 0) return n;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ranks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)(kListBytes + kMaxSlice);
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, sample_kernel<true>, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = ctx->sm_count / ranks;
    }
    if (slot) slot->store(n, std::memory_order_relaxed);
    return n;
}

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
    static std::atomic<uint64_t> asked[2];
    cudaError_t e = allow_shared(sample_kernel<true>, kListBytes + kMaxSlice, asked[0], ctx->device);
    if (e == cudaSuccess) e = allow_shared(sample_kernel<false>, kListBytes + kMaxSlice, asked[1], ctx->device);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cudaFuncSetAttribute(sample)");
    // Blocks a row takes: as many as let all rows run at once with a block a
    // multiprocessor (eight are the portable cluster), each with at least 1024
    // logits; one where there are more rows, two a multiprocessor then. Two
    // blocks that share one wait for each other's issue slots in every step: 32
    // rows of 151,936 logits with top-k take 24 us in clusters of 4, 30 in
    // clusters of 8 two a multiprocessor, 17 rows of 32,003 17 us against 22.
    int ranks = kMaxCluster;
    while (ranks > 1 && (vocab <= (int64_t)ranks * 1024 || rows > clusters_at_once(ctx, ranks))) ranks /= 2;
    const int64_t slice = ((vocab + ranks - 1) / ranks + 3) / 4 * 4;
    const bool resident = slice * 4 <= (rows * ranks > ctx->sm_count ? kPairSlice : kMaxSlice);
    const bool packs = stride % 4 == 0 && vocab % 4 == 0 && (uintptr_t)logits_dev % 16 == 0;
    SampleArgs a{logits_dev, stride, temperature_dev, top_k_dev, top_p_dev, min_p_dev, uniform_dev, ids_dev,
                 logprobs_dev, (int)vocab, (int)slice, resident};
    auto kernel = packs ? sample_kernel<true> : sample_kernel<false>;
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
