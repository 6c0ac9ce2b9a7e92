// attention.cu — attention of new tokens over a paged cache: the call, and the
// kernel for few rows a key head (single tokens, short chunks, f32 queries).
//
//   o = sum_j softmax_j(scale q . k_j) v_j,  j over what the row sees
//
// in one pass over the keys, with the running maximum m and sum l of the
// weights: a tile of scores s gives m' = max(m, s), and l and o are scaled by
// exp(m - m') before its weights exp(s - m') are added.
//
// Rows: the r query heads of a key head share its keys, so 16 rows (tokens x r
// heads) are one tile of the tensor cores and every key is read once for them.
// A single token's work is then its keys and values: bound by memory, 16 to 64
// operations a byte. 64 tokens over 100 to 16000 keys of 8 heads of 128: 140 us,
// 6.0 TB/s, 92% of the copy rate; one token over 4100: 15 us, launches and loads that wait on each
// other (lengths, pages, keys, sums to join).
//
// The keys of all blocks of rows together (tiles of 64) are cut evenly over as
// many blocks as run at once, however the sequences' lengths differ: a block
// takes a contiguous range of tiles, of one block of rows or of several, and a
// block of rows that falls to more than one thread block leaves (o, m, l) a
// piece in the workspace, which a second kernel joins. The cut follows from the
// lengths on the device, so that a captured call follows them.
//
// Each group of warps (one or two) goes through keys of its own (16 of a tile's 64) with its own ring
// of asynchronous copies, and no warp waits for another before its block's
// range ends.
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"

namespace strata {
namespace {

constexpr int kGroups = 4;  // of warps: each goes through keys of its own
constexpr int kRows = 16;  // rows of a block
constexpr int kUnit = 16;  // keys a warp takes of a tile
constexpr int kTile = kGroups * kUnit;
// What a block of rows costs besides its tiles, in tiles (64 single tokens over 100 to 16000 keys
// took 155, 142, 140 and 140 us with 1, 3, 4 and 6).
constexpr int kOver = 4;
constexpr int kLeast = 4;  // units of a thread block, or so, where there is little to read: fewer pieces to join

// DP: head_dim rounded up to 64, 128 or 256. Stages and blocks side by side fill
// the shared memory, so that about 128 KB a multiprocessor are under way.
template <int DP, int LIMBS>
struct Cfg {
    static constexpr int kStages = DP == 64 ? 4 : 3;
    static constexpr int kBlocks = DP == 256 ? 1 : DP == 128 ? 2 : 3;
    // Two warps a group share its keys where a row is long: each has half of a row's
    // products, and the scores' halves are added through shared memory (32 single tokens
    // of 2 key heads of 256 in f32, a window of 4096: 74 us with one warp a group, 69 with
    // two; 64 of bf16 131, 128).
    static constexpr int kParts = DP == 256 ? 2 : 1, kWarps = kGroups * kParts, kThreads = kWarps * 32;
    static constexpr int kUnitBytes = kUnit * DP * 2;  // of keys; as much of values
    static constexpr int kQBytes = LIMBS * kRows * DP * 2;
    static constexpr int kRing = kGroups * kStages * 2 * kUnitBytes;
    static constexpr int kJoin = kGroups * kRows * (DP + 2) * 4;
    static constexpr int kHalves = kParts > 1 ? kWarps * kRows * kUnit * 4 : 0;  // scores' halves
    static constexpr int kSmem = kQBytes + (kRing > kJoin ? kRing : kJoin) + kHalves;
    static_assert(kBlocks * (kSmem + 1024) <= 228 * 1024, "blocks do not fit side by side");
};
constexpr int kMaxGrid = 148 * 3;  // blocks of a launch at most; the workspace is for as many

// The workspace: what each block leaves of its first and its last block of rows
// where other blocks have the rest, and which blocks of rows are to be joined.
struct Work {
    Split* split;  // [kMaxGrid]
    float* ml;     // [kMaxGrid][2][2][kRows]
    float* o;      // [kMaxGrid][2][kRows][DP]
};
constexpr int64_t kSplitBytes = kMaxGrid * sizeof(Split), kMlBytes = (int64_t)kMaxGrid * 2 * 2 * kRows * 4;
constexpr int64_t work_bytes_for(int dp) { return kSplitBytes + kMlBytes + (int64_t)kMaxGrid * 2 * kRows * dp * 4; }
inline Work work_of(void* p) {
    char* b = static_cast<char*>(p);
    return {reinterpret_cast<Split*>(b), reinterpret_cast<float*>(b + kSplitBytes), reinterpret_cast<float*>(b + kSplitBytes + kMlBytes)};
}

__device__ __forceinline__ uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two floats as bf16 pairs, the largest limb first: x = limb 0 + limb 1 + ..., each
// rounding leaves 2^-8 of what it rounds at most, so three limbs keep f32's 24 bits.
template <int LIMBS>
__device__ __forceinline__ void limbs(float x, float y, uint32_t (&out)[LIMBS]) {
#pragma unroll
    for (int i = 0; i < LIMBS; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        out[i] = *reinterpret_cast<const uint32_t*>(&h);
        x -= __uint_as_float(out[i] << 16), y -= __uint_as_float(out[i] & 0xFFFF0000u);
    }
}
// Byte offset of 16-byte chunk c of row r in a tile of rows of DP elements: chunks
// are permuted within a row so that 8 rows' same chunk lie in different banks.
template <int DP>
__device__ __forceinline__ int chunk_at(int r, int c) { return r * DP * 2 + ((c ^ (r & 7)) << 4); }

template <int DP, int LIMBS, typename T>
__global__ void __launch_bounds__(Cfg<DP, LIMBS>::kThreads, Cfg<DP, LIMBS>::kBlocks)
    split_kernel(const AttnArgs a, const Work work, int entries, const __grid_constant__ SeqTable tab) {
    using C = Cfg<DP, LIMBS>;
    constexpr int kWarps = C::kWarps, kThreads = C::kThreads, DH = DP / C::kParts;  // a warp's columns of a row
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const qs = smem;
    uint8_t* const ring = smem + C::kQBytes;
    float* const halves = reinterpret_cast<float*>(smem + C::kSmem - C::kHalves);
    __shared__ int64_t scan[kWarps + 2];
    __shared__ int odd_rows[kRows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int group = warp / C::kParts, part = warp % C::kParts;
    const int d = a.c.head_dim;
    // the warps of a group meet
    auto meet = [&] {
        if (C::kParts > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(C::kParts * 32) : "memory");
        else __syncwarp();
    };
    after_previous();
    Cut cut = cut_range<kThreads, kRows, kTile, kOver, kLeast>(a, tab, entries, scan);
    if (threadIdx.x == 0) work.split[blockIdx.x].pieces = 0;
    if (blockIdx.x >= cut.grid) return;
    const int64_t range_begin = cut.pos;

    Piece<kTile> pc;
    while (next_piece<kRows, kTile, kOver>(a, tab, cut, pc)) {
        const RowBlock& b = pc.b;
        const KeyRange<kTile>& kr = pc.kr;
        const int head = pc.head, steps = pc.steps;

        // ---- this warp's keys, kStages - 1 units ahead. A lane copies the same 16 bytes of
        // every kRowsAtOnce-th row.
        constexpr int kChunks = DP / 8, kRowsAtOnce = 32 / kChunks;
        static_assert(kChunks <= 32, "a row is at most 32 lanes");
        const int my_row = lane / kChunks, my_chunk = lane % kChunks;
        const int64_t my_at = (int64_t)head * a.c.head_stride + (int64_t)(part * (kUnit / C::kParts) + my_row) * a.c.token_stride + my_chunk * 8;
        const bool my_column = my_chunk * 8 < d;
        int64_t places = -1;  // of the first key of unit (step & ~31) + lane, its page and row there; -1: none, or not needed
        uint32_t none = 0;    // bit step & 31: the unit has no page, or no key that a row sees
        auto load = [&](int step) {
            if (step < steps) {
                if ((step & 31) == 0) {
                    const int at = step + lane, j = at < steps ? pc.key(at) + group * kUnit : kr.hi;
                    const int page = j < kr.hi && (j + kUnit > kr.lo || j < a.sinks) ? page_of(a.c, b.slot, j) : -1;
                    places = page >= 0 ? place(a.c, page, j, 0) : -1;
                }
                const int64_t at = __shfl_sync(0xFFFFFFFFu, places, step & 31);
                none = (none & ~(1u << (step & 31))) | (at < 0 ? 1u << (step & 31) : 0u);
                if (at >= 0) {
                    const int rows = kr.hi - (pc.key(step) + group * kUnit);  // that any row may see: behind them may be anything
                    const __nv_bfloat16* k = a.c.k + at + my_at;
                    const __nv_bfloat16* v = a.c.v + at + my_at;
                    const uint32_t stage = shared_at(ring) + (group * C::kStages + step % C::kStages) * 2 * C::kUnitBytes;
#pragma unroll
                    for (int i = 0; i < kUnit / kRowsAtOnce / C::kParts; ++i) {
                        const int row = (part * (kUnit / kRowsAtOnce / C::kParts) + i) * kRowsAtOnce + my_row;
                        const int n = my_column && row < rows ? 16 : 0;  // the rest is zeros
                        const uint32_t dst = stage + chunk_at<DP>(row, my_chunk);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(n ? k : a.c.k), "r"(n) : "memory");
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + C::kUnitBytes), "l"(n ? v : a.c.v), "r"(n) : "memory");
                        k += kRowsAtOnce * a.c.token_stride, v += kRowsAtOnce * a.c.token_stride;
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < C::kStages - 1; ++i) load(i);

        // ---- the rows' queries, as limbs
        for (int i = threadIdx.x; i < kRows * (DP / 8); i += kThreads) {
            const int row = i / (DP / 8), c = i % (DP / 8), packed = b.row0 + row;
            float x[8] = {};
            if (row < b.rows && c * 8 < d) {
                const int64_t at = (int64_t)(b.first_row + packed / a.r) * a.q_stride + (int64_t)(head * a.r + packed % a.r) * d + c * 8;
                if (a.wide) {
                    using P = Pack<T, 16 / sizeof(T)>;
#pragma unroll
                    for (int w = 0; w < 8; w += 16 / sizeof(T)) {
                        const P p = *reinterpret_cast<const P*>(static_cast<const T*>(a.q) + at + w);
#pragma unroll
                        for (int u = 0; u < (int)(16 / sizeof(T)); ++u) x[w + u] = to_f32(p.v[u]);
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < 8; ++u) x[u] = load_f32<T>(a.q, at + u);
                }
            }
            uint32_t w[4][LIMBS];
#pragma unroll
            for (int u = 0; u < 4; ++u) limbs<LIMBS>(x[2 * u], x[2 * u + 1], w[u]);
#pragma unroll
            for (int l = 0; l < LIMBS; ++l)
                *reinterpret_cast<uint4*>(qs + l * kRows * DP * 2 + chunk_at<DP>(row, c)) = make_uint4(w[0][l], w[1][l], w[2][l], w[3][l]);
        }
        if (threadIdx.x < kRows) odd_rows[threadIdx.x] = 0;
        __syncthreads();

        float o[DH / 8][4] = {};
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {};
        int p[2];  // positions of this lane's rows; rows that are none are zeros and go nowhere
#pragma unroll
        for (int i = 0; i < 2; ++i) p[i] = g + 8 * i < b.rows ? b.p0 + (b.row0 + g + 8 * i) / a.r : -1;
        const int p_min = b.p0 + b.row0 / a.r, p_max = b.p0 + (b.row0 + b.rows - 1) / a.r;

        for (int step = 0; step < steps; ++step) {
            asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 2) : "memory");
            meet();  // the unit is there, and the last one has been read
            load(step + C::kStages - 1);
            const int j0 = pc.key(step) + group * kUnit;
            const uint32_t ks = shared_at(ring) + (group * C::kStages + step % C::kStages) * 2 * C::kUnitBytes, vs = ks + C::kUnitBytes;
            if (!(none >> (step & 31) & 1)) {
                float s[LIMBS > 1 ? 2 : 1][2][4] = {};  // the small limbs' sums apart
#pragma unroll
                for (int k0 = 0; k0 < DH / 16; ++k0) {
                    const int k = part * (DH / 16) + k0;
                    uint32_t kb[4];
                    ldsm4(kb, ks + chunk_at<DP>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
#pragma unroll
                    for (int u = 0; u < LIMBS; ++u) {
                        uint32_t qa[4];
                        ldsm4(qa, shared_at(qs) + u * kRows * DP * 2 + chunk_at<DP>(lane & 15, 2 * k + (lane >> 4)));
                        mma(s[u > 0][0], qa, kb[0], kb[1]);
                        mma(s[u > 0][1], qa, kb[2], kb[3]);
                    }
                }
                if (LIMBS > 1)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[0][n][i] += s[LIMBS > 1 ? 1 : 0][n][i];
                if (C::kParts > 1) {  // the other half of the row's products
                    float4* const mine = reinterpret_cast<float4*>(halves) + warp * 64 + lane;
                    mine[0] = make_float4(s[0][0][0], s[0][0][1], s[0][0][2], s[0][0][3]);
                    mine[32] = make_float4(s[0][1][0], s[0][1][1], s[0][1][2], s[0][1][3]);
                    meet();  // and again before the next step's are written
                    const float4* const other = reinterpret_cast<const float4*>(halves) + (warp ^ 1) * 64 + lane;
                    const float4 x = other[0], y = other[32];
                    s[0][0][0] += x.x, s[0][0][1] += x.y, s[0][0][2] += x.z, s[0][0][3] += x.w;
                    s[0][1][0] += y.x, s[0][1][1] += y.y, s[0][1][2] += y.z, s[0][1][3] += y.w;
                }
                if (j0 + kUnit - 1 > p_min || (a.window && j0 <= p_max - a.window) || j0 + kUnit > kr.hi) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = j0 + n * 8 + 2 * t4 + (i & 1);
                            if (j >= kr.hi || !sees(a, p[i >> 1], j)) s[0][n][i] = -INFINITY;
                        }
                }
                float w[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float top = fmaxf(fmaxf(s[0][0][2 * i], s[0][0][2 * i + 1]), fmaxf(s[0][1][2 * i], s[0][1][2 * i + 1]));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    const float next = fmaxf(m[i], top * a.scale2), base = next == -INFINITY ? 0.0f : next;
                    if (next != m[i]) {
                        const float alpha = exp2_approx(m[i] - base);
                        l[i] *= alpha;
#pragma unroll
                        for (int n = 0; n < DH / 8; ++n) o[n][2 * i] *= alpha, o[n][2 * i + 1] *= alpha;
                        m[i] = next;
                    }
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const float e = exp2_approx(fmaf(s[0][n][2 * i + u], a.scale2, -base));
                            w[n][2 * i + u] = e;
                            l[i] += e;
                        }
                }
                // weights as the left operand: its 16 keys are the two tiles' columns. One limb
                // rounds them to bf16, as exact as the values they meet (each off by 2^-8 of
                // itself at most; their sum takes them unrounded): three, as for f32, would take
                // three times the products for a result that is rounded to bf16 itself.
                uint32_t wa[LIMBS][4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t x[LIMBS];
                        limbs<LIMBS>(w[n][2 * i], w[n][2 * i + 1], x);
#pragma unroll
                        for (int u = 0; u < LIMBS; ++u) wa[u][2 * n + i] = x[u];
                    }
#pragma unroll
                for (int n = 0; n < DH / 16; ++n) {
                    uint32_t vb[4];
                    ldsm4_t(vb, vs + chunk_at<DP>(lane & 15, part * (DH / 8) + 2 * n + (lane >> 4)));
                    if (LIMBS == 1) {
                        mma(o[2 * n], wa[0], vb[0], vb[1]);
                        mma(o[2 * n + 1], wa[0], vb[2], vb[3]);
                    } else {
                        // the tensor cores round a long running sum towards zero: a unit's
                        // products by themselves, added to it in f32
                        float x[2][4] = {};
#pragma unroll
                        for (int u = LIMBS - 1; u >= 0; --u) {
                            mma(x[0], wa[u], vb[0], vb[1]);
                            mma(x[1], wa[u], vb[2], vb[3]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[2 * n][i] += x[0][i], o[2 * n + 1][i] += x[1][i];
                    }
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");

        // ---- the warps' sums joined, in the ring's memory
        __syncthreads();
        float* const jo = reinterpret_cast<float*>(ring);          // [kGroups][kRows][DP]
        float* const jm = jo + kGroups * kRows * DP;               // [kGroups][2][kRows]
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
            l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
            if (t4 == 0 && part == 0) jm[(group * 2) * kRows + g + 8 * i] = m[i], jm[(group * 2 + 1) * kRows + g + 8 * i] = l[i];
#pragma unroll
            for (int n = 0; n < DH / 8; ++n)
                *reinterpret_cast<float2*>(jo + (group * kRows + g + 8 * i) * DP + part * DH + n * 8 + 2 * t4) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
        __syncthreads();
        const bool whole = pc.whole();
        const int slot = slot_of(pc, range_begin);
        const int64_t wslot = (int64_t)blockIdx.x * 2 + slot;
        for (int i = threadIdx.x; i < b.rows * (DP / 4); i += kThreads) {
            const int row = i / (DP / 4), c = (i % (DP / 4)) * 4;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kGroups; ++w) top = fmaxf(top, jm[(w * 2) * kRows + row]);
            const float base = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, x[4] = {};
#pragma unroll
            for (int w = 0; w < kGroups; ++w) {
                const float f = exp2_approx(jm[(w * 2) * kRows + row] - base);
                const float4 v = *reinterpret_cast<const float4*>(jo + (w * kRows + row) * DP + c);
                sum = fmaf(f, jm[(w * 2 + 1) * kRows + row], sum);
                x[0] = fmaf(f, v.x, x[0]), x[1] = fmaf(f, v.y, x[1]), x[2] = fmaf(f, v.z, x[2]), x[3] = fmaf(f, v.w, x[3]);
            }
            if (!whole) {
                *reinterpret_cast<float4*>(work.o + (wslot * kRows + row) * DP + c) = make_float4(x[0], x[1], x[2], x[3]);
                if (c == 0) work.ml[(wslot * 2) * kRows + row] = top, work.ml[(wslot * 2 + 1) * kRows + row] = sum;
                continue;
            }
            const float inv = 1.0f / sum;  // 0: the row sees nothing, or only scores of -inf
            bool odd = !(sum > 0.0f);
            const int packed = b.row0 + row;
            const int64_t at = (int64_t)(b.first_row + packed / a.r) * a.o_stride + (int64_t)(head * a.r + packed % a.r) * d + c;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                x[u] *= inv;
                if (c + u < d) {
                    odd |= !isfinite(x[u]);
                    from_f32(static_cast<T*>(a.o)[at + u], x[u]);
                }
            }
            if (odd) odd_rows[row] = 1;
        }
        __syncthreads();
        if (whole) {
            for (int row = warp; row < b.rows; row += kWarps)
                if (odd_rows[row]) {
                    const int token = (b.row0 + row) / a.r;
                    careful_row<T>(a, b.slot, b.first_row + token, b.p0 + token, head * a.r + (b.row0 + row) % a.r, head);
                }
        } else if (pc.tile0 == 0 && threadIdx.x == 0) {
            work.split[blockIdx.x] = Split{pc.entry, head, pieces_of(cut, pc), slot};
        }
        __syncthreads();
    }
}

constexpr int kJoiners = 128;  // threads

// Block b joins the block of rows whose first piece thread block b left.
template <int DP, typename T>
__global__ void __launch_bounds__(kJoiners) join_kernel(const AttnArgs a, const Work work, const __grid_constant__ SeqTable tab) {
    __shared__ float weight[kMaxGrid][kRows];  // of a piece's sums
    __shared__ float part[kJoiners / kRows][kRows];
    __shared__ int odd_rows[kRows];
    after_previous(false);
    const Split s = work.split[blockIdx.x];
    if (!s.pieces) return;
    const RowBlock b = row_block(a, sequence_of_tile(tab, s.entry), s.entry, kRows);
    const int head = s.head, d = a.c.head_dim;
    auto slot = [&](int i) { return i == 0 ? (int64_t)blockIdx.x * 2 + s.first_slot : (int64_t)(blockIdx.x + i) * 2; };
    {
        constexpr int kGroups = kJoiners / kRows;
        const int row = threadIdx.x % kRows, group = threadIdx.x / kRows;
        float top = -INFINITY;
#pragma unroll 4
        for (int n = group; n < s.pieces; n += kGroups) {
            const float m = work.ml[(slot(n) * 2) * kRows + row];
            weight[n][row] = m;
            top = fmaxf(top, m);
        }
        part[group][row] = top;
        if (threadIdx.x < kRows) odd_rows[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kGroups; ++i) top = fmaxf(top, part[i][row]);
        __syncthreads();
        const float base = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll 4
        for (int n = group; n < s.pieces; n += kGroups) {
            const float f = exp2_approx(weight[n][row] - base);
            weight[n][row] = f;
            sum = fmaf(f, work.ml[(slot(n) * 2 + 1) * kRows + row], sum);
        }
        part[group][row] = sum;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < b.rows * (DP / 4); i += kJoiners) {
        const int row = i / (DP / 4), c = (i % (DP / 4)) * 4;
        if (c >= d) continue;
        float sum = 0.0f, x[4] = {};
#pragma unroll
        for (int g = 0; g < kJoiners / kRows; ++g) sum += part[g][row];
#pragma unroll 8
        for (int n = 0; n < s.pieces; ++n) {
            const float f = weight[n][row];
            const float4 v = *reinterpret_cast<const float4*>(work.o + (slot(n) * kRows + row) * DP + c);
            x[0] = fmaf(f, v.x, x[0]), x[1] = fmaf(f, v.y, x[1]), x[2] = fmaf(f, v.z, x[2]), x[3] = fmaf(f, v.w, x[3]);
        }
        const float inv = 1.0f / sum;
        bool odd = !(sum > 0.0f);
        const int packed = b.row0 + row;
        const int64_t at = (int64_t)(b.first_row + packed / a.r) * a.o_stride + (int64_t)(head * a.r + packed % a.r) * d + c;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            x[u] *= inv;
            odd |= !isfinite(x[u]);
            from_f32(static_cast<T*>(a.o)[at + u], x[u]);
        }
        if (odd) odd_rows[row] = 1;
    }
    __syncthreads();
    for (int row = threadIdx.x >> 5; row < b.rows; row += kJoiners / 32)
        if (odd_rows[row]) {
            const int token = (b.row0 + row) / a.r;
            careful_row<T>(a, b.slot, b.first_row + token, b.p0 + token, head * a.r + (b.row0 + row) % a.r, head);
        }
}

template <int DP, int LIMBS, typename T>
int launch_split(strata_ctx* ctx, const AttnArgs& a, void* work, const SeqTable& tab, int64_t entries, cudaStream_t s) {
    using C = Cfg<DP, LIMBS>;
    static std::atomic<uint64_t> asked{0};
    cudaError_t e = allow_shared(split_kernel<DP, LIMBS, T>, C::kSmem, asked, ctx->device);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cudaFuncSetAttribute(attention)");
    const int grid = std::min(ctx->sm_count * C::kBlocks, kMaxGrid);
    const Work w = work_of(work);
    e = launch_early(split_kernel<DP, LIMBS, T>, dim3(grid), C::kThreads, C::kSmem, s, a, w, (int)entries, tab);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "attention kernel");
    e = launch_early(join_kernel<DP, T>, dim3(grid), kJoiners, 0, s, a, w, tab);
    return e == cudaSuccess ? STRATA_OK : cuda_fail(ctx, e, "attention join");
}

template <int DP>
int launch_split(strata_ctx* ctx, bool bf16, const AttnArgs& a, void* work, const SeqTable& tab, int64_t entries, cudaStream_t s) {
    if (bf16) return launch_split<DP, 1, __nv_bfloat16>(ctx, a, work, tab, entries, s);
    return launch_split<DP, 3, float>(ctx, a, work, tab, entries, s);
}

// A sequence of kTcRows rows a key head goes to the tiles of 128 rows where the call has
// kTcAll such rows and key heads together. Measured, tiles against 16 rows at a time (us,
// heads of 128; sequences x rows a key head on key heads):
//   keys before   16x16 on 8   16x32 on 8   16x256 on 8   1x64 on 8   1x128 on 8   1x256 on 8
//   0             18, 11       18, 12       21, 47        15, 10      16, 10       18, 11
//   500           29, 22       31, 26       46, 106       26, 18      26, 20       30, 22
//   8000          127, 101     131, 178     155, 1198     64, 36      65, 52       70, 75
//   32000         388, 329     390, 633     518, 4827     121, 91     124, 152     121, 233
//   keys before   1x1024 on 8  16x64 on 1   16x128 on 1   1x512 on 1  1x2048 on 1
//   0             20, 28       15, 10       16, 11        18, 10      20, 19
//   500           35, 40       26, 18       27, 22        29, 18      30, 23
//   8000          65, 221      58, 51       59, 74        61, 34      70, 71
//   32000         143, 781     116, 172     109, 261      171, 72     96, 210
// What the tiles lose below is the join of many pieces (1x512 on 1 behind 8000: 155 us, not
// 61, while a thread block could have a single unit). The keys before are not known on the
// host; the rule is right from some thousands on, and costs up to 8 us in front of them.
constexpr int64_t kTcRows = 32, kTcAll = 2048;

bool tiles(const strata_attention& d, const strata_kv_cache& c) { return d.dtype == STRATA_QUANT_BF16 && c.head_dim <= 128; }
int padded(int64_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

uint64_t needed(const strata_attention& d, const strata_kv_cache& c) {
    const int dp = padded(c.head_dim);
    return (uint64_t)std::max(work_bytes_for(dp), tiles(d, c) ? attention_tc_work_bytes(dp) : 0);
}

}  // namespace
}  // namespace strata

using namespace strata;

extern "C" int strata_cuda_attention_work_bytes(const strata_attention* desc, const strata_kv_cache* cache, uint64_t* bytes) {
    if (!desc || !cache || !bytes) return STRATA_ERR_INVALID;
    strata_attention d = *desc;
    strata_kv_cache c = *cache;
    Why why;
    int64_t tokens = 0, longest = 0;
    const int rc = check_attention(why, d, c, &tokens, &longest);
    if (rc) return rc;
    *bytes = longest ? needed(d, c) : 0;
    return STRATA_OK;
}

extern "C" int strata_cuda_attention_dev(strata_ctx* ctx, const strata_attention* desc, const strata_kv_cache* cache,
                                         const void* q_dev, void* o_dev, void* work_dev, uint64_t work_bytes, void* stream) {
    if (!ctx || !desc || !cache) return STRATA_ERR_INVALID;
    STRATA_CALL_RANGE();
    std::lock_guard<std::mutex> g(ctx->mu);
    strata_attention d = *desc;
    strata_kv_cache c = *cache;
    Why why;
    int64_t tokens = 0, longest = 0;
    int rc = check_attention(why, d, c, &tokens, &longest);
    const int dp = padded(c.head_dim);
    if (!rc && longest) rc = check_attention_buffers(why, d, c, tokens, q_dev, o_dev, work_dev, work_bytes, needed(d, c));
    if (rc) return fail(ctx, rc, "attention: %s", why.text);
    if (!longest) return STRATA_OK;
    const bool bf16 = d.dtype == STRATA_QUANT_BF16;
    const int64_t size = dtype_bytes(d.dtype);
    AttnArgs a = {};
    a.c = cache_args(c);
    a.q = q_dev, a.o = o_dev, a.q_stride = d.q_stride, a.o_stride = d.o_stride;
    a.r = (int)(d.n_head / c.n_kv_head);
    // over all positions (2^31 - 1 at most) it is none; over the table's it is one for tokens behind the table
    a.window = d.window < kMaxTokens ? (int)d.window : 0;
    a.sinks = a.window ? (int)std::min(d.sinks, kMaxTokens) : 0;
    a.scale2 = (float)(d.scale * 1.4426950408889634);
    a.wide = ((uintptr_t)q_dev | (uintptr_t)o_dev) % 16 == 0 && (d.q_stride * size) % 16 == 0 && (d.o_stride * size) % 16 == 0;
    DeviceGuard dev(ctx->device);
    const cudaStream_t s = pick_stream(ctx, stream);
    int64_t many = kMaxTokens + 1;  // tokens from which a sequence is read in tiles
    TcMaps maps;
    const int64_t enough = (kTcRows + a.r - 1) / a.r;
    if (tiles(d, c) && a.wide && longest >= enough) {
        int64_t all = d.seq_offsets ? 0 : d.n_seq * d.seq_len;
        for (int64_t i = 0; d.seq_offsets && i < d.n_seq && all < kTcAll; ++i) {
            const int64_t n = d.seq_offsets[i + 1] - d.seq_offsets[i];
            if (n >= enough) all += n;
        }
        if (all * d.n_head >= kTcAll && attention_tc_maps(a.c, &maps)) {
            many = enough;
            rc = for_row_groups(d, a.r, attention_tc_rows(), many, kMaxTokens + 1, [&](const SeqTable& t, int64_t entries) {
                return launch_attention_tc(ctx, dp, a, work_dev, t, entries, maps, s);
            });
            if (rc) return rc;
        }
    }
    return for_row_groups(d, a.r, kRows, 1, many, [&](const SeqTable& t, int64_t entries) {
        if (dp == 64) return launch_split<64>(ctx, bf16, a, work_dev, t, entries, s);
        if (dp == 128) return launch_split<128>(ctx, bf16, a, work_dev, t, entries, s);
        return launch_split<256>(ctx, bf16, a, work_dev, t, entries, s);
    });
}
