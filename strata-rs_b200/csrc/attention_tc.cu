// attention_tc.cu — attention of a chunk of bf16 queries over a paged cache on
// the 5th-generation tensor cores (the prompt's kernel; attention.cu has the call
// and the kernel for few rows).
//
// A thread block takes 256 rows of one key head (tokens x query heads, token by
// token) as two tiles of 128 and goes through its tiles of 128 keys:
//   S = Q K^T         tcgen05.mma, both operands in shared memory, S in TMEM
//   P = exp2(S - m)   a thread a row, from TMEM through registers and back, rounded to
//                     bf16 (2^-8 of each weight at most, as exact as the values that it
//                     meets; their sum l takes them unrounded): the products take bf16
//   O += P V          tcgen05.mma, P in TMEM (over S), V in shared memory
// While the threads of one tile compute its weights, the tensor cores work for the
// other. Exponentials (16 a clock) and products (8192 flops a clock) of a tile
// take about as long as each other, so both have to run all the time.
//   warps 0-3, 4-7   the rows of tile 0, 1: queries to shared memory, weights,
//                    sums, outputs
//   warp 8           issues the products
//   warps 9, 11      copy keys, values (TMA, 128-byte swizzle; a box is as many
//                    tokens as lie side by side in a page, 16 to 128; a page that is
//                    none is a box outside the pool, which reads as zeros)
//   warp 10          finds the pieces of work
// m moves only when a row's maximum has grown by 2^8 or more (weights are then up to
// 2^8, which costs no precision): O, in TMEM, is rescaled rarely, by the row's own
// thread, between two products that add to it.
//
// Like attention.cu's kernel, thread blocks take equal shares of all tiles of the
// call, and a second kernel joins the blocks of rows that were cut.
//
// A chunk of 1024 tokens behind 20000, 32 heads on 8 of 128: 304 us, 1.13 PFLOP/s (70% of
// the products' measured burst rate); a prompt of 8192: 500 us, 1.10. (A few calls at a
// time: one after another for long, at the power limit, 354 and 563.) The tensor pipe is
// busy for 67% of the cycles. What got it there from 393 and 1046 us: one region of scores
// that the two tiles hand on, so that a tile's next scores wait for the reading of the
// other's and not for its own weights (P has a place of its own); registers shared out by
// warpgroups, so that a row's 128 scores stay in them; few instructions between two batches
// of products; the code kept small (straight-line variants of what is rare cost more in
// instruction fetches than they saved). A cubic for some of the exponentials, to spare the
// special-function unit, made it slower at every share: issue slots are the scarcer.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "attention.cuh"

namespace strata {
namespace {

constexpr int kRowTile = 128, kKeyTile = 128;
constexpr int kRows = 2 * kRowTile;
constexpr int kThreads = 384;  // three warpgroups, which registers are shared out by
constexpr int kRegs = 208, kRegsRest = 88;  // 2 x 208 + 88 = 3 x 168, what the block is launched with
constexpr int kOver = 6;       // what a block of rows costs besides its tiles, in tiles (8 or 4: a prompt of 8192 508, 532 us, not 500)
constexpr int kLeast = 4;      // units of a thread block, or so, where there is little to do: fewer pieces to join
constexpr int kMaxGrid = 148;
constexpr int kMasks = 8;   // tiles whose masks are kept
constexpr int kPieces = 8;  // pieces that are known ahead
constexpr int kReaders = 11; // of a piece: the rows' warps, the products' and the copies'

template <int DP>
struct Cfg {
    static constexpr int kChunks = DP / 64;                      // 128-byte columns of a tile
    static constexpr int kChunkBytes = kKeyTile * 128;
    static constexpr int kTileBytes = kChunks * kChunkBytes;     // of keys or values, and of queries
    static constexpr int kSlots = DP == 64 ? 8 : 5;
    static constexpr int kSmem = (2 + kSlots) * kTileBytes + 1024;
    static_assert(kSmem <= 227 * 1024, "tiles do not fit");
};

// What a thread block leaves of a cut block of rows: [slot][column][row].
struct TcWork {
    Split* split;  // [kMaxGrid]
    float* ml;     // [kMaxGrid][2][2][kRows]
    float* o;      // [kMaxGrid][2][DP][kRows]
};
constexpr int64_t kSplitBytes = kMaxGrid * sizeof(Split), kMlBytes = (int64_t)kMaxGrid * 2 * 2 * kRows * 4;
inline TcWork work_of(void* p) {
    char* b = static_cast<char*>(p);
    return {reinterpret_cast<Split*>(b), reinterpret_cast<float*>(b + kSplitBytes), reinterpret_cast<float*>(b + kSplitBytes + kMlBytes)};
}

__device__ __forceinline__ uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t par) {
    uint32_t ok;
    // up to 20 us asleep, so that warps that wait take no issue slots from those that compute
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(b), "r"(par) : "memory");
    return ok != 0;
}
// Waits for the phase of parity `par`; false, and *err set, after about 20 seconds: warps
// wait while others compute rows again that are not finite, over contexts of any length.
// (In line: a call would keep the compiler from giving warps registers of others.)
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t par, int* err) {
    uint64_t t0 = 0;
#pragma unroll 1
    for (long long i = 0; i < kSpinLimit; ++i) {
        if (bar_try(b, par)) return true;
        if ((i & 15) == 15) {
            const uint64_t t = now_ns();
            if (!t0) t0 = t;
            else if (t - t0 > 20000000000ull) break;
        }
    }
    atomicExch(err, 1);
    return false;
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                 : "memory");
}
// Shared-memory descriptors of 128-byte-swizzled tiles, rows of 128 bytes, 8 rows 1024 bytes apart.
// K-major (rows are M or N, a row holds 64 of K):
__device__ __forceinline__ uint64_t k_major(uint32_t at) {
    return (uint64_t)((at >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// N-major (rows are K, a row holds 64 of N, the next 64 of N a chunk further):
__device__ __forceinline__ uint64_t n_major(uint32_t at) {
    return (uint64_t)((at >> 4) & 0x3FFFu) | ((uint64_t)(kKeyTile * 128 >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: f32 accumulators, bf16 operands, M x N, B N-major where `nb`.
constexpr uint32_t instruction(int M, int N, bool nb) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (nb ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// True for one lane of a converged warp. Products are issued under it, with the rest
// of the warp's control flow the same for all lanes: their operands then are uniform
// registers (issued by `lane == 0` of a diverged warp each product cost 150 clocks and
// the products, not the weights, set the pace).
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 32 columns of the warp's 32 lanes of TMEM, a lane a thread.
__device__ __forceinline__ void tmem_ld(uint32_t at, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A piece as all warps see it, in shared memory (a warp of its own runs ahead and
// finds it: where it lies and how far it goes takes divisions and 64-bit numbers).
struct Known {
    Piece<kKeyTile> piece;
    int last;  // 1: there is none, nor behind it
};

// Columns of TMEM: the tiles' outputs, their weights (two a column), the scores.
constexpr uint32_t kO = 0, kP = 256, kS = 384;

// The lowest n bits (none below 0, all from 32 on).
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

struct Boxes {
    int rows;    // tokens of a box
    int inside;  // heads lie inside tokens: the map's dimensions are (dim, head, token, page), else (dim, token, head, page)
};

// A place in the ring of slots and the parity of the round it is in.
template <int SLOTS>
struct Place {
    uint32_t slot, round;
    __device__ __forceinline__ void operator+=(uint32_t n) {
        slot += n;
        if (slot >= SLOTS) slot -= SLOTS, round ^= 1;
    }
};

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
    tc_kernel(const AttnArgs a, const TcWork work, int entries, int* err, const Boxes box, const __grid_constant__ CUtensorMap kmap,
              const __grid_constant__ CUtensorMap vmap, const __grid_constant__ SeqTable tab) {
    using C = Cfg<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const qs = smem;                     // 2 tiles of queries
    uint8_t* const ring = smem + 2 * C::kTileBytes;  // keys, values, keys, values, ...
    __shared__ __align__(8) uint64_t full[C::kSlots], empty[C::kSlots], landed, q_full[2], s_full[2], s_free[2], p_full[2], o_done[2], drained;
    __shared__ uint32_t masks[kMasks], tmem_at;
    __shared__ int64_t scan[kThreads / 32 + 2];
    __shared__ Known known[kPieces];
    __shared__ __align__(8) uint64_t known_full[kPieces], known_empty[kPieces];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    after_previous();
    Cut cut = cut_range<kThreads, kRows, kKeyTile, kOver, kLeast>(a, tab, entries, scan);
    if (threadIdx.x == 0) work.split[blockIdx.x].pieces = 0;
    if (blockIdx.x >= cut.grid) return;
    const int64_t range_begin = cut.pos;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kSlots; ++i) bar_init(shared_at(&full[i]), 1), bar_init(shared_at(&empty[i]), 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(shared_at(&q_full[i]), 4), bar_init(shared_at(&s_full[i]), 1), bar_init(shared_at(&s_free[i]), 4);
            bar_init(shared_at(&p_full[i]), 4), bar_init(shared_at(&o_done[i]), 1);
        }
        for (int i = 0; i < kPieces; ++i) bar_init(shared_at(&known_full[i]), 1), bar_init(shared_at(&known_empty[i]), kReaders);
        bar_init(shared_at(&landed), 1), bar_init(shared_at(&drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_at(&tmem_at)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        fence_before();
    }
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_at;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
        // ---------------- a row a thread
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + kS, p_at = tmem + lanes + kP + 64 * t, o_at = tmem + lanes + kO + 128 * t;
        uint32_t done = 0, tiles = 0;  // products into O so far, tiles
        bool live = true;
        // A tile's rows of queries and outputs are moved by the warps that own them, DP / 8
        // lanes a row, so that lines are read and written whole; outputs pass through the
        // queries' place in shared memory.
        constexpr int kLanes = DP / 8, kAtOnce = 32 / kLanes;
        const int unit = lane % kLanes, sub = lane / kLanes;
        uint8_t* const mine_at = qs + t * C::kTileBytes + (warp & 3) * 32 * 128;  // this warp's rows of the tile's first column
        auto place_of = [&](int r, int u) { return mine_at + (u / 8) * C::kChunkBytes + r * 128 + ((u ^ r) & 7) * 16; };
        auto has_rows = [&](const Piece<kKeyTile>& pc) { return t * kRowTile < pc.b.rows && pc.steps > 0; };
        auto known_at = [&](uint32_t i) { return live && __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&known_full[i % kPieces]), (i / kPieces) & 1, err)); };
        float m = 0.0f, l = 0.0f;
        for (uint32_t i = 0;; ++i) {
            // ---- piece i - 1's outputs, then piece i's queries
            const Known& kn = known[i % kPieces];
            live = known_at(i);
            if (!live) break;
            const bool last = kn.last, active = !last && has_rows(kn.piece);
            const Piece<kKeyTile>& pc = known[(i + kPieces - 1) % kPieces].piece;
            if (i > 0 && t * kRowTile < pc.b.rows) {
                const RowBlock& b = pc.b;
                const int head = pc.head, d = a.c.head_dim, steps = pc.steps;
                const int in_block = t * kRowTile + row, packed = b.row0 + in_block, token = packed / a.r;
                const bool mine = in_block < b.rows, whole = pc.whole();
                if (steps > 0) {
                    live = __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&o_done[t]), (done - 1) & 1, err));
                    if (!live) break;
                    fence_after();
                } else {
                    l = 0.0f, m = -INFINITY;
                }
                const int64_t slot = (int64_t)blockIdx.x * 2 + slot_of(pc, range_begin);
                const float inv = 1.0f / l;
                float2 all = make_float2(0.0f, 0.0f);  // stays 0 while outputs are finite
#pragma unroll 1
                for (int c0 = 0; c0 < DP; c0 += 32) {
                    float o[32] = {};
                    if (steps > 0) {
                        tmem_ld(o_at + c0, o);
                        tmem_ld_wait();
                    }
                    if (!whole) {
#pragma unroll
                        for (int w = 0; w < 32; ++w) work.o[(slot * DP + c0 + w) * kRows + in_block] = o[w];
                        continue;
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint32_t e[4];
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const float2 y = __fmul2_rn(make_float2(o[8 * u + 2 * w], o[8 * u + 2 * w + 1]), make_float2(inv, inv));
                            all = __ffma2_rn(y, make_float2(0.0f, 0.0f), all);
                            const __nv_bfloat162 two = __floats2bfloat162_rn(y.x, y.y);
                            e[w] = *reinterpret_cast<const uint32_t*>(&two);
                        }
                        *reinterpret_cast<uint4*>(place_of(lane, c0 / 8 + u)) = make_uint4(e[0], e[1], e[2], e[3]);
                    }
                }
                fence_before();
                if (whole) {
                    const int64_t own = mine ? (int64_t)(b.first_row + token) * a.o_stride + (int64_t)(head * a.r + packed % a.r) * d : -1;
                    __syncwarp();
#pragma unroll
                    for (int u = 0; u < kLanes; ++u) {
                        const int64_t at = __shfl_sync(0xFFFFFFFFu, own, u * kAtOnce + sub);
                        const uint4 x = *reinterpret_cast<const uint4*>(place_of(u * kAtOnce + sub, unit));
                        if (at >= 0 && unit * 8 < d) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.o) + at + unit * 8) = x;
                    }
                    const bool odd = !(l > 0.0f) || !(all.x == 0.0f) || !(all.y == 0.0f);
                    for (unsigned rows = __ballot_sync(0xFFFFFFFFu, mine && odd); rows; rows &= rows - 1) {
                        const int at = packed - lane + __ffs(rows) - 1;  // rows of a warp are neighbours
                        __syncwarp();
                        careful_row<__nv_bfloat16>(a, b.slot, b.first_row + at / a.r, b.p0 + at / a.r, head * a.r + at % a.r, head);
                    }
                } else {
                    work.ml[(slot * 2) * kRows + in_block] = m, work.ml[(slot * 2 + 1) * kRows + in_block] = l;
                    if (pc.tile0 == 0 && threadIdx.x == 0) work.split[blockIdx.x] = Split{pc.entry, head, pieces_of(cut, pc), (int)(slot & 1)};
                }
            }
            __syncwarp();
            if (i > 0 && lane == 0) bar_arrive(shared_at(&known_empty[(i - 1) % kPieces]));
            if (last) break;
            if (!active) {
                tiles += kn.piece.steps;
                continue;
            }
            uint4 ahead[kLanes];
            if (active) {
                const RowBlock& b = kn.piece.b;
                const int in_block = t * kRowTile + row, packed = b.row0 + in_block;
                // where this thread's own row lies (divisions: once a row)
                const int64_t own = in_block < b.rows ? (int64_t)(b.first_row + packed / a.r) * a.q_stride + (int64_t)(kn.piece.head * a.r + packed % a.r) * a.c.head_dim : -1;
#pragma unroll
                for (int u = 0; u < kLanes; ++u) {
                    const int64_t at = __shfl_sync(0xFFFFFFFFu, own, u * kAtOnce + sub);
                    ahead[u] = make_uint4(0, 0, 0, 0);
                    if (at >= 0 && unit * 8 < a.c.head_dim) ahead[u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + at + unit * 8);
                }
            }
#pragma unroll
            for (int u = 0; u < kLanes; ++u) *reinterpret_cast<uint4*>(place_of(u * kAtOnce + sub, unit)) = ahead[u];
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(shared_at(&q_full[t]));

            // ---- its tiles
            const int steps = kn.piece.steps;
            const int p = kn.piece.b.p0 + min(kn.piece.b.row0 + t * kRowTile + row, kn.piece.b.row0 + kn.piece.b.rows - 1) / a.r;
            const int p_min = __shfl_sync(0xFFFFFFFFu, p, 0), p_max = __shfl_sync(0xFFFFFFFFu, p, 31);
            const int hidden = a.window && p_max >= a.window ? p_max - a.window : -1;  // the last key that the window takes from some row
            m = -INFINITY, l = 0.0f;
            for (int j = 0; j < steps; ++j, ++tiles, ++done) {
                live = __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&s_full[t]), done & 1, err));
                if (!live) break;
                fence_after();
                float s[kKeyTile];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld(s_at + 32 * i, s + 32 * i);
                tmem_ld_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(shared_at(&s_free[t]));
                const int base = kn.piece.key(j);
                const uint32_t valid = masks[tiles % kMasks];
                const bool masked = valid != 0xFF || base + kKeyTile - 1 > p_min || base <= hidden;
                if (masked) {
                    // bit c of the row: it sees key base + c
                    const int to = p - base, from = a.window && a.window <= to ? to - a.window + 1 : 0, sinks = a.sinks - base;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t bits = below(to + 1 - 32 * w) & (~below(from - 32 * w) | below(sinks - 32 * w)) &
                                              ((valid >> (2 * w) & 1 ? 0xFFFFu : 0u) | (valid >> (2 * w + 1) & 1 ? 0xFFFF0000u : 0u));
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(bits >> c & 1)) s[32 * w + c] = -INFINITY;
                    }
                }
                float top[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) top[c] = fmaxf(s[c], s[c + 8]);
#pragma unroll
                for (int c = 16; c < kKeyTile; c += 16)
#pragma unroll
                    for (int u = 0; u < 8; ++u) top[u] = fmaxf(top[u], fmaxf(s[c + u], s[c + u + 8]));
#pragma unroll
                for (int u = 4; u; u /= 2)
#pragma unroll
                    for (int c = 0; c < u; ++c) top[c] = fmaxf(top[c], top[c + u]);
                const float next = fmaxf(m, top[0] * a.scale2);
                const bool moves = next > m + 8.0f;
                const float f = moves ? exp2_approx(m - next) : 1.0f;
                if (moves) m = next;
                const float down = m == -INFINITY ? 0.0f : -m;
                float2 sum[2] = {};
                uint32_t w[kKeyTile / 2];
#pragma unroll
                for (int c = 0; c < kKeyTile; c += 2) {
                    const float2 x = __ffma2_rn(make_float2(s[c], s[c + 1]), make_float2(a.scale2, a.scale2), make_float2(down, down));
                    const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                    sum[c / 2 & 1] = __fadd2_rn(sum[c / 2 & 1], e);
                    const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
                    w[c / 2] = *reinterpret_cast<const uint32_t*>(&h);
                }
                const float2 both_sums = __fadd2_rn(sum[0], sum[1]);
                l = fmaf(l, f, both_sums.x + both_sums.y);
                if (j > 0) {  // the last product has read P and written O
                    live = __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&o_done[t]), (done - 1) & 1, err));
                    if (!live) break;
                    fence_after();
                    if (__any_sync(0xFFFFFFFFu, moves)) {
#pragma unroll 1
                        for (int c = 0; c < DP; c += 16) {
                            float o[16];
                            tmem_ld16(o_at + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] *= f;
                            tmem_st16(o_at + c, reinterpret_cast<uint32_t*>(o));
                        }
                    }
                }
                tmem_st(p_at, w);
                tmem_st(p_at + 32, w + 32);
                tmem_st_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(shared_at(&p_full[t]));
            }
            if (!live) break;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
        if (warp == 10) {
            // ---------------- pieces, and their queries on the way to L2
            bool live = true, last = false;
            for (uint32_t n = 0; live && !last; ++n) {
                Known& kn = known[n % kPieces];
                if (n >= kPieces) live = __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&known_empty[n % kPieces]), (n / kPieces - 1) & 1, err));
                if (!live) break;
                if (lane == 0) kn.last = !next_piece<kRows, kKeyTile, kOver>(a, tab, cut, kn.piece);
                __syncwarp();
                last = kn.last;
                const RowBlock& b = kn.piece.b;
                for (int row = lane; row < b.rows && !last; row += 32) {
                    const int packed = b.row0 + row;
                    const char* q = static_cast<const char*>(a.q) + ((int64_t)(b.first_row + packed / a.r) * a.q_stride + (int64_t)(kn.piece.head * a.r + packed % a.r) * a.c.head_dim) * 2;
                    for (int at = 0; at < a.c.head_dim * 2; at += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + at));
                }
                if (lane == 0) bar_arrive(shared_at(&known_full[n % kPieces]));
            }
        } else if (warp == 9 || warp == 11) {
            // ---------------- copies: keys by one warp, values by the other
            const bool keys = warp == 9;
            const CUtensorMap* const map = keys ? &kmap : &vmap;
            Place<C::kSlots> to = {keys ? 0u : 1u, 0};
            uint32_t filled = 0, lands = 0, tiles = 0;  // the first `first` of this warp's slots have not been used before
            const uint32_t first = keys ? (C::kSlots + 1) / 2 : C::kSlots / 2;
            bool live = true;
            const int per = kKeyTile / box.rows, i = lane / C::kChunks, c = lane % C::kChunks;  // this lane's box and column
            for (uint32_t n = 0; live; ++n) {
                const Known& kn = known[n % kPieces];
                live = __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&known_full[n % kPieces]), (n / kPieces) & 1, err));
                if (!live || kn.last) break;
                const Piece<kKeyTile> pc = kn.piece;
                __syncwarp();
                if (lane == 0) bar_arrive(shared_at(&known_empty[n % kPieces]));
                const int len = pc.b.p0 + pc.b.n, steps = pc.steps, head = pc.head;
                // lane g: the page of keys 16 g .. 16 g + 15, a tile ahead
                auto page_at = [&](int j) {
                    const int key = j < steps ? pc.key(j) + 16 * (lane & 7) : pc.kr.hi;  // below 2^31: a tile ends at 2^31 at most
                    return lane < 8 && key < pc.kr.hi ? page_of(a.c, pc.b.slot, key) : -1;
                };
                int page = page_at(0);
                for (int j = 0; j < steps && live; ++j, ++tiles, to += 2, ++filled) {
                    const int base = pc.key(j), ahead = page_at(j + 1);
                    const uint32_t valid = __ballot_sync(0xFFFFFFFFu, page >= 0);
                    if (keys && lane == 0) masks[tiles % kMasks] = valid;
                    const int from = __shfl_sync(0xFFFFFFFFu, page, (i * box.rows / 16) & 7);
                    const int token = from >= 0 ? (base + i * box.rows) % a.c.page_size : 0;
                    const int g = from >= 0 ? from : a.c.n_pages;  // outside the pool: zeros
                    if (filled >= first) live = bar_wait(shared_at(&empty[to.slot]), to.round ^ 1, err);
                    live = __all_sync(0xFFFFFFFFu, live);
                    if (!live) break;
                    // the last tokens' page goes on behind them with whatever is there: values of zero instead
                    const bool patch = !keys && len >= base && len - base < kKeyTile && len % box.rows;
                    const uint32_t bar = shared_at(patch ? &landed : &full[to.slot]), dst = shared_at(ring) + to.slot * C::kTileBytes;
                    if (lane == 0) bar_expect(bar, C::kTileBytes);
                    __syncwarp();
                    if (i < per) tma_4d(dst + c * C::kChunkBytes + i * box.rows * 128, map, c * 64, box.inside ? head : token, box.inside ? token : head, g, bar);
                    if (patch) {
                        live = __all_sync(0xFFFFFFFFu, bar_wait(bar, lands++ & 1, err));
                        const int stale = len - base, rows = (stale + box.rows - 1) / box.rows * box.rows - stale;
                        for (int u = lane; u < rows * 8 * C::kChunks; u += 32) {
                            const int row = stale + u % rows, unit = u / rows;  // the swizzle stays within a row
                            *reinterpret_cast<uint4*>(ring + to.slot * C::kTileBytes + (unit / 8) * C::kChunkBytes + row * 128 + (unit % 8) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_async();
                        __syncwarp();
                        if (lane == 0) bar_arrive(shared_at(&full[to.slot]));
                    }
                    page = ahead;
                }
            }
            if (!live) {  // every copy that is under way lands before the block ends
                const uint32_t out = filled < first ? filled : first;
                for (uint32_t n = filled - out; n < filled; ++n) {
                    const uint32_t at = 2 * n + (keys ? 0 : 1);
                    bar_wait(shared_at(&full[at % C::kSlots]), (at / C::kSlots) & 1, err);
                }
            }
        } else if (warp == 8) {
            // ---------------- products
            constexpr uint32_t qk = instruction(kRowTile, kKeyTile, false), pv = instruction(kRowTile, DP, true);
            Place<C::kSlots> k = {0, 0}, v = {1, 0};      // the next keys, the next values
            uint32_t qn[2] = {}, sn = 0, sn1 = 0, pn[2] = {};  // queries, scores that were read, weights
            bool live = true;
            // Between two batches of products only what is queued hides what the issuing warp
            // does: it asks for two barriers at once, and whether a wait ran out once a tile
            // (products on what is not there yet are wrong, not out of bounds).
            auto wait = [&](uint32_t b, uint32_t par) {
                live &= bar_wait(b, par, err);
                fence_after();
            };
            auto wait2 = [&](uint32_t b, uint32_t par, uint32_t b2, uint32_t par2) {
                if (!(bar_try(b, par) & bar_try(b2, par2))) live &= bar_wait(b, par, err) && bar_wait(b2, par2, err);
                fence_after();
            };
            const uint32_t q_at = shared_at(qs), ring_at = shared_at(ring), full_at = shared_at(full), empty_at = shared_at(empty);
            const uint32_t s_full_at = shared_at(s_full), s_free_at = shared_at(s_free), p_full_at = shared_at(p_full), o_done_at = shared_at(o_done);
            // S = Q_t K^T; the keys' slot is free behind it where `last` is set
            auto scores = [&](int t, bool last) {
                const uint64_t q = k_major(q_at + t * C::kTileBytes), at = k_major(ring_at + k.slot * C::kTileBytes);
                __syncwarp();
                if (elected()) {
#pragma unroll
                    for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int step = (c * C::kChunkBytes + 32 * i) >> 4;  // in the descriptors' units of 16 bytes
                            mma_ss(tmem + kS, q + step, at + step, qk, c + i > 0);
                        }
                    commit(s_full_at + 8 * t);
                    if (last) commit(empty_at + 8 * k.slot);
                }
                if (last) k += 2;
            };
            // O_t += P_t V; likewise
            auto values = [&](int t, bool add, bool last) {
                const uint64_t at = n_major(ring_at + v.slot * C::kTileBytes);
                __syncwarp();
                if (elected()) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) mma_ts(tmem + kO + 128 * t, tmem + kP + 64 * t + 8 * i, at + (2048 * i >> 4), pv, add || i > 0);
                    commit(o_done_at + 8 * t);
                    if (last) commit(empty_at + 8 * v.slot);
                }
                if (last) v += 2;
            };
            for (uint32_t i = 0; live; ++i) {
                const Known& kn = known[i % kPieces];
                wait(shared_at(&known_full[i % kPieces]), (i / kPieces) & 1);
                live = __all_sync(0xFFFFFFFFu, live);
                if (!live || kn.last) break;
                const int steps = kn.piece.steps;
                const bool both = kn.piece.b.rows > kRowTile;
                __syncwarp();
                if (lane == 0) bar_arrive(shared_at(&known_empty[i % kPieces]));
                if (steps <= 0) continue;
                // S is one tile's at a time: its reader hands it on at once, and while the
                // rows of one tile compute their weights the other's products run
                wait2(shared_at(&q_full[0]), qn[0]++ & 1, full_at + 8 * k.slot, k.round);
                if (both) wait(shared_at(&q_full[1]), qn[1]++ & 1);
                scores(0, false);
                for (int j = 0; j < steps && live; ++j) {
                    const bool more = j + 1 < steps;
                    wait(s_free_at, sn & 1);
                    if (both) {
                        scores(1, true);
                        if (j > 0) {
                            wait(p_full_at + 8, pn[1]++ & 1);
                            values(1, j > 1, true);
                        }
                        if (more) {
                            wait2(s_free_at + 8, sn1 & 1, full_at + 8 * k.slot, k.round);
                            scores(0, false);
                        } else {
                            wait(s_free_at + 8, sn1 & 1);
                        }
                        ++sn1;
                    } else {
                        // the keys' slot is free once this tile's scores are read
                        if (elected()) commit(empty_at + 8 * k.slot);
                        k += 2;
                        if (more) {
                            wait(full_at + 8 * k.slot, k.round);
                            scores(0, false);
                        }
                    }
                    ++sn;
                    wait2(p_full_at, pn[0]++ & 1, full_at + 8 * v.slot, v.round);
                    values(0, j > 0, !both);
                    live = __all_sync(0xFFFFFFFFu, live);
                }
                if (both && live) {
                    wait(p_full_at + 8, pn[1]++ & 1);
                    values(1, steps > 1, true);
                }
            }
            // nothing is left running when TMEM is given back
            __syncwarp();
            if (elected()) commit(shared_at(&drained));
            bar_wait(shared_at(&drained), 0, err);
            __syncwarp();
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 8) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// Block (b, y) joins 32 rows of the block of rows whose first piece thread block b
// left: a thread a row and every fourth column.
template <int DP>
__global__ void __launch_bounds__(128) tc_join_kernel(const AttnArgs a, const TcWork work, const __grid_constant__ SeqTable tab) {
    __shared__ int odd_rows[32];
    after_previous(false);
    const Split s = work.split[blockIdx.x];
    if (!s.pieces) return;
    const RowBlock b = row_block(a, sequence_of_tile(tab, s.entry), s.entry, kRows);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = a.c.head_dim;
    const int row0 = blockIdx.y * 32, row = row0 + lane;
    if (row0 >= b.rows) return;
    if (threadIdx.x < 32) odd_rows[threadIdx.x] = 0;
    __syncthreads();
    auto slot = [&](int i) { return i == 0 ? (int64_t)blockIdx.x * 2 + s.first_slot : (int64_t)(blockIdx.x + i) * 2; };
    float top = -INFINITY, sum = 0.0f;
    for (int n = 0; n < s.pieces; ++n) top = fmaxf(top, work.ml[(slot(n) * 2) * kRows + row]);
    const float base = top == -INFINITY ? 0.0f : top;
    for (int n = 0; n < s.pieces; ++n)
        sum = fmaf(exp2_approx(work.ml[(slot(n) * 2) * kRows + row] - base), work.ml[(slot(n) * 2 + 1) * kRows + row], sum);
    const float inv = 1.0f / sum;
    bool odd = !(sum > 0.0f);
    const int packed = b.row0 + row;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.o) + (int64_t)(b.first_row + packed / a.r) * a.o_stride + (int64_t)(s.head * a.r + packed % a.r) * d;
    for (int c = warp * 8; c < d; c += 32) {  // d is a multiple of 8
        float o[8] = {};
        for (int n = 0; n < s.pieces; ++n) {
            const float f = exp2_approx(work.ml[(slot(n) * 2) * kRows + row] - base);
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = fmaf(f, work.o[(slot(n) * DP + c + i) * kRows + row], o[i]);
        }
        if (row < b.rows) {
            __nv_bfloat16 e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[i] *= inv;
                odd |= !isfinite(o[i]);
                e[i] = __float2bfloat16_rn(o[i]);
            }
            if (a.wide) *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<const uint4*>(e);
            else
                for (int i = 0; i < 8; ++i) out[c + i] = e[i];
        }
    }
    if (odd && row < b.rows) odd_rows[lane] = 1;
    __syncthreads();
    for (int i = warp; i < 32 && row0 + i < b.rows; i += 4)
        if (odd_rows[i]) {
            const int at = b.row0 + row0 + i;
            careful_row<__nv_bfloat16>(a, b.slot, b.first_row + at / a.r, b.p0 + at / a.r, s.head * a.r + at % a.r, s.head);
        }
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void* p = nullptr;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p) : nullptr;
    }();
    return fn;
}

bool encode(CUtensorMap* map, const void* pool, const CacheArgs& c, const Boxes& box) {
    const cuuint64_t token = c.page_size, head = c.n_kv_head, ts = c.token_stride * 2, hs = c.head_stride * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, box.inside ? head : token, box.inside ? token : head, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[3] = {box.inside ? hs : ts, box.inside ? ts : hs, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t rows = box.rows, size[4] = {64, box.inside ? 1 : rows, box.inside ? rows : 1, 1}, step[4] = {1, 1, 1, 1};
    for (cuuint64_t s : strides)
        if (s >= cuuint64_t(1) << 40) return false;
    return encoder() && encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(pool), dims, strides, size, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP>
int launch(strata_ctx* ctx, const AttnArgs& a, void* work, const SeqTable& tab, int64_t entries, const TcMaps& maps, cudaStream_t s) {
    static std::atomic<uint64_t> asked{0};
    cudaError_t e = allow_shared(tc_kernel<DP>, Cfg<DP>::kSmem, asked, ctx->device);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cudaFuncSetAttribute(attention)");
    const int grid = std::min(ctx->sm_count, kMaxGrid);
    const TcWork w = work_of(work);
    CUtensorMap k, v;
    memcpy(&k, maps.k, sizeof k), memcpy(&v, maps.v, sizeof v);
    e = launch_early(tc_kernel<DP>, dim3(grid), kThreads, Cfg<DP>::kSmem, s, a, w, (int)entries, ctx->err_dev, Boxes{maps.box_rows, maps.inside}, k, v, tab);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "attention kernel");
    e = launch_early(tc_join_kernel<DP>, dim3(grid, kRows / 32), 128, 0, s, a, w, tab);
    return e == cudaSuccess ? STRATA_OK : cuda_fail(ctx, e, "attention join");
}

}  // namespace

int attention_tc_rows() { return kRows; }
int64_t attention_tc_work_bytes(int dp) { return kSplitBytes + kMlBytes + (int64_t)kMaxGrid * 2 * kRows * dp * 4; }
bool attention_tc_maps(const CacheArgs& c, TcMaps* maps) {
    Boxes box = {128, c.token_stride >= (c.n_kv_head - 1) * c.head_stride + c.head_dim};
    while (c.page_size % box.rows) box.rows /= 2;  // 16 at least
    maps->box_rows = box.rows, maps->inside = box.inside;
    static_assert(sizeof(CUtensorMap) <= sizeof maps->k, "a map fits");
    CUtensorMap k, v;
    if (!encode(&k, c.k, c, box) || !encode(&v, c.v, c, box)) return false;
    memcpy(maps->k, &k, sizeof k), memcpy(maps->v, &v, sizeof v);
    return true;
}
int launch_attention_tc(strata_ctx* ctx, int dp, const AttnArgs& a, void* work, const SeqTable& tab, int64_t entries, const TcMaps& maps, cudaStream_t s) {
    return dp == 64 ? launch<64>(ctx, a, work, tab, entries, maps, s) : launch<128>(ctx, a, work, tab, entries, maps, s);
}

}  // namespace strata
