// attention_tc.cu — attention of a chunk of bf16 queries over a paged cache on
// the 5th-generation tensor cores (the prompt's kernel; attention.cu has the call
// and the kernel for few rows).
//
// A thread block takes 256 rows of one key head (tokens x query heads, token by
// token) as two tiles of 128 and goes through its tiles of 128 keys:
//   S = Q K^T         tcgen05.mma, both operands in shared memory, S in TMEM
//   P = exp2(S - m)   a thread a row, from TMEM through registers and back
//   O += P V          tcgen05.mma, P in TMEM (over S), V in shared memory
// While the threads of one tile compute its weights, the tensor cores work for the
// other. Exponentials (16 a clock) and products (8192 flops a clock) of a tile
// take about as long as each other, so both have to run all the time.
//   warps 0-3, 4-7   the rows of tile 0, 1: queries to shared memory, weights,
//                    sums, outputs
//   warp 8           issues the products
//   warp 9           copies keys and values (TMA, 128-byte swizzle; a box is as many
//                    tokens as lie side by side in a page, 16 to 128; a page that is
//                    none is a box outside the pool, which reads as zeros)
// m moves only when a row's maximum has grown by 2^8 or more (weights are then up to
// 2^8, which costs no precision): O, in TMEM, is rescaled rarely, by the row's own
// thread, between two products that add to it.
//
// Like attention.cu's kernel, thread blocks take equal shares of all tiles of the
// call, and a second kernel joins the blocks of rows that were cut.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "attention.cuh"

namespace strata {
namespace {

constexpr int kRowTile = 128, kKeyTile = 128;
constexpr int kRows = 2 * kRowTile;
constexpr int kThreads = 320;
constexpr int kOver = 2;       // what a block of rows costs besides its tiles, in tiles
constexpr int kMaxGrid = 148;
constexpr int kMasks = 8;   // tiles whose masks are kept
constexpr int kPieces = 4;  // pieces that are known ahead
constexpr int kReaders = 9; // of a piece: the rows' warps and the products'

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
// Waits for the phase of parity `par`; false, and *err set, after about a second.
__device__ __noinline__ bool bar_wait_long(uint32_t b, uint32_t par, int* err) {
    const uint64_t t0 = now_ns();
    for (long long i = 0; i < kSpinLimit; ++i) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(b), "r"(par) : "memory");
        if (ok) return true;
        if ((i & 255) == 255 && now_ns() - t0 > 1000000000ull) break;
    }
    atomicExch(err, 1);
    return false;
}
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t par, int* err) {
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(b), "r"(par) : "memory");
        if (ok) return true;
    }
    return bar_wait_long(b, par, err);
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
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A piece as all warps see it, in shared memory (the copies' warp runs ahead and
// finds it; where it lies and how far it goes takes divisions and 64-bit numbers).
struct Known {
    Piece<kKeyTile> piece;
    int last;  // 1: there is none, nor behind it
};

struct Boxes {
    int rows;    // tokens of a box
    int inside;  // heads lie inside tokens: the map's dimensions are (dim, head, token, page), else (dim, token, head, page)
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
    __shared__ __align__(8) uint64_t full[C::kSlots], empty[C::kSlots], landed, q_full[2], s_full[2], p_full[2], o_full[2], drained;
    __shared__ uint32_t masks[kMasks], tmem_at;
    __shared__ int64_t scan[kThreads / 32 + 2];
    __shared__ Known known[kPieces];
    __shared__ __align__(8) uint64_t known_full[kPieces], known_empty[kPieces];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    Cut cut = cut_range<kThreads, kRows, kKeyTile, kOver>(a, tab, entries, scan);
    if (threadIdx.x == 0) work.split[blockIdx.x].pieces = 0;
    if (blockIdx.x >= cut.grid) return;
    const int64_t range_begin = cut.pos;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kSlots; ++i) bar_init(shared_at(&full[i]), 1), bar_init(shared_at(&empty[i]), 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(shared_at(&q_full[i]), 4), bar_init(shared_at(&s_full[i]), 1);
            bar_init(shared_at(&p_full[i]), 4), bar_init(shared_at(&o_full[i]), 1);
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
    const uint32_t tmem = tmem_at;  // S (and P) of tile t at column 128 t, O at 256 + 128 t

    if (warp < 8) {
        // ---------------- a row a thread
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + 128 * t, o_at = tmem + lanes + 256 + 128 * t;
        uint32_t ss = 0, os = 0, tiles = 0;
        bool live = true;
        // This tile's queries of a piece to shared memory (nothing where it has no row of the tile).
        auto load_queries = [&](const Piece<kKeyTile>& pc) {
            if (t * kRowTile >= pc.b.rows || pc.steps <= 0) return;
            const int packed = pc.b.row0 + t * kRowTile + row, d = a.c.head_dim;
            const bool mine = t * kRowTile + row < pc.b.rows;
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + (int64_t)(pc.b.first_row + packed / a.r) * a.q_stride + (int64_t)(pc.head * a.r + packed % a.r) * d;
            uint8_t* const to = qs + t * C::kTileBytes + row * 128;
#pragma unroll
            for (int u0 = 0; u0 < DP / 8; u0 += 8) {
                uint4 x[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    x[u] = make_uint4(0, 0, 0, 0);
                    if (mine && (u0 + u) * 8 < d) {
                        if (a.wide) {
                            x[u] = *reinterpret_cast<const uint4*>(q + (u0 + u) * 8);
                        } else {
                            uint32_t e[4];
                            for (int i = 0; i < 4; ++i) {
                                const __nv_bfloat162 two = __halves2bfloat162(q[(u0 + u) * 8 + 2 * i], q[(u0 + u) * 8 + 2 * i + 1]);
                                e[i] = *reinterpret_cast<const uint32_t*>(&two);
                            }
                            x[u] = make_uint4(e[0], e[1], e[2], e[3]);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) *reinterpret_cast<uint4*>(to + (u0 / 8) * C::kChunkBytes + ((u ^ row) & 7) * 16) = x[u];
            }
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(shared_at(&q_full[t]));
        };
        auto known_at = [&](uint32_t i) { return live && __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&known_full[i % kPieces]), (i / kPieces) & 1, err)); };
        live = known_at(0);
        if (live && !known[0].last) load_queries(known[0].piece);
        for (uint32_t i = 0; live && !known[i % kPieces].last; ++i) {
            const Piece<kKeyTile>& pc = known[i % kPieces].piece;
            const RowBlock& b = pc.b;
            const int head = pc.head, d = a.c.head_dim, steps = pc.steps;
            auto next = [&] {  // the next piece's queries
                live = known_at(i + 1);
                if (live && !known[(i + 1) % kPieces].last) load_queries(known[(i + 1) % kPieces].piece);
            };
            if (t * kRowTile >= b.rows) {  // no row of this tile
                tiles += steps;
                next();
                __syncwarp();
                if (lane == 0) bar_arrive(shared_at(&known_empty[i % kPieces]));
                continue;
            }
            const int in_block = t * kRowTile + row, packed = b.row0 + in_block;
            const bool mine = in_block < b.rows;
            const int token = packed / a.r, p = b.p0 + (mine ? token : (b.row0 + b.rows - 1) / a.r);
            const int p_min = __shfl_sync(0xFFFFFFFFu, p, 0), p_max = __shfl_sync(0xFFFFFFFFu, p, 31);
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < steps; ++j, ++tiles) {
                live = __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&s_full[t]), ss++ & 1, err));
                if (!live) break;
                fence_after();
                float s[kKeyTile];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld(s_at + 32 * i, s + 32 * i);
                tmem_ld_wait();
                const int base = pc.key(j);
                const uint32_t valid = masks[tiles % kMasks];
                if (valid != 0xFF || base + kKeyTile - 1 > p_min || (a.window && base <= p_max - a.window)) {
                    if (a.window) {
#pragma unroll
                        for (int c = 0; c < kKeyTile; ++c)
                            if (!(valid >> (c / 16) & 1) || !sees(a, p, base + c)) s[c] = -INFINITY;
                    } else {
                        const int last = p - base;
#pragma unroll
                        for (int c = 0; c < kKeyTile; ++c)
                            if (!(valid >> (c / 16) & 1) || c > last) s[c] = -INFINITY;
                    }
                }
                float top[2] = {fmaxf(s[0], s[1]), fmaxf(s[2], s[3])};
#pragma unroll
                for (int c = 4; c < kKeyTile; c += 4) top[0] = fmaxf(top[0], fmaxf(s[c], s[c + 1])), top[1] = fmaxf(top[1], fmaxf(s[c + 2], s[c + 3]));
                const float next = fmaxf(m, fmaxf(top[0], top[1]) * a.scale2);
                const bool moves = next > m + 8.0f;
                if (__any_sync(0xFFFFFFFFu, moves)) {
                    const float f = moves ? exp2_approx(m - next) : 1.0f;
                    if (moves) m = next;
                    l *= f;
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < DP; c += 32) {
                            float o[32];
                            tmem_ld(o_at + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= f;
                            tmem_st(o_at + c, reinterpret_cast<uint32_t*>(o));
                        }
                    }
                }
                const float down = m == -INFINITY ? 0.0f : -m;
                float2 sum[2] = {};
#pragma unroll
                for (int c0 = 0; c0 < kKeyTile; c0 += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int c = c0; c < c0 + 32; c += 2) {
                        const float2 x = __ffma2_rn(make_float2(s[c], s[c + 1]), make_float2(a.scale2, a.scale2), make_float2(down, down));
                        const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                        sum[c / 2 & 1] = __fadd2_rn(sum[c / 2 & 1], e);
                        const __nv_bfloat162 h = __floats2bfloat162_rn(e.x, e.y);
                        w[(c - c0) / 2] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    tmem_st16(s_at + c0 / 2, w);
                }
                const float2 both_sums = __fadd2_rn(sum[0], sum[1]);
                l += both_sums.x + both_sums.y;
                tmem_st_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(shared_at(&p_full[t]));
            }
            // the tile's queries have been read: the next piece's, while this one's last product runs
            if (live) next();
            if (steps > 0 && live) {
                live = __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&o_full[t]), os++ & 1, err));
                fence_after();
            }
            if (!live) break;
            const bool whole = pc.whole();
            const int64_t slot = (int64_t)blockIdx.x * 2 + slot_of(pc, range_begin);
            const float inv = 1.0f / l;
            bool odd = !(l > 0.0f);
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.o) + (int64_t)(b.first_row + token) * a.o_stride + (int64_t)(head * a.r + packed % a.r) * d;
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
                float o[32] = {};
                if (steps > 0) {
                    tmem_ld(o_at + c, o);
                    tmem_ld_wait();
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) work.o[(slot * DP + c + i) * kRows + in_block] = o[i];
                } else if (mine) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        o[i] *= inv;
                        if (c + i < d) odd |= !isfinite(o[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        if (c + i < d) {
                            __nv_bfloat16 e[8];
#pragma unroll
                            for (int u = 0; u < 8; ++u) e[u] = __float2bfloat16_rn(o[i + u]);
                            if (a.wide) *reinterpret_cast<uint4*>(out + c + i) = *reinterpret_cast<const uint4*>(e);
                            else
                                for (int u = 0; u < 8; ++u) out[c + i + u] = e[u];
                        }
                }
            }
            fence_before();
            if (whole) {
                for (unsigned rows = __ballot_sync(0xFFFFFFFFu, mine && odd); rows; rows &= rows - 1) {
                    const int at = packed - lane + __ffs(rows) - 1;  // rows of a warp are neighbours
                    careful_row<__nv_bfloat16>(a, b.slot, b.first_row + at / a.r, b.p0 + at / a.r, head * a.r + at % a.r, head);
                }
            } else {
                work.ml[(slot * 2) * kRows + in_block] = m, work.ml[(slot * 2 + 1) * kRows + in_block] = l;
                if (pc.tile0 == 0 && threadIdx.x == 0) work.split[blockIdx.x] = Split{pc.entry, head, pieces_of(cut, pc), (int)(slot & 1)};
            }
            __syncwarp();
            if (lane == 0) bar_arrive(shared_at(&known_empty[i % kPieces]));
        }
    } else if (warp == 9) {
        // ---------------- copies
        uint32_t n = 0, lands = 0, tiles = 0;  // slots filled, boxes waited for, tiles
        bool live = true;
        for (uint32_t i = 0; live; ++i) {
            Known& kn = known[i % kPieces];
            if (i >= kPieces) live = __all_sync(0xFFFFFFFFu, bar_wait(shared_at(&known_empty[i % kPieces]), (i / kPieces - 1) & 1, err));
            if (!live) break;
            if (lane == 0) {
                kn.last = !next_piece<kRows, kKeyTile, kOver>(a, tab, cut, kn.piece);
                bar_arrive(shared_at(&known_full[i % kPieces]));
            }
            __syncwarp();
            const Piece<kKeyTile>& pc = kn.piece;
            if (kn.last) break;
            const int len = pc.b.p0 + pc.b.n, per = kKeyTile / box.rows;
            for (int j = 0; j < pc.steps && live; ++j, ++tiles) {
                const int base = pc.key(j);
                // lane g: the page of keys 16 g .. 16 g + 15
                int page = -1;
                if (lane < 8 && base + 16 * lane < pc.kr.hi) page = page_of(a.c, pc.b.slot, base + 16 * lane);
                const uint32_t valid = __ballot_sync(0xFFFFFFFFu, page >= 0);
                if (lane == 0) masks[tiles % kMasks] = valid;
                // the last tokens' page goes on behind them with whatever is there: zeros instead
                const int stale = len >= base && len < base + kKeyTile && len % box.rows ? len - base : kKeyTile;
                for (int kv = 0; kv < 2 && live; ++kv, ++n) {
                    const uint32_t slot = n % C::kSlots;
                    if (n >= C::kSlots) live = bar_wait(shared_at(&empty[slot]), (n / C::kSlots - 1) & 1, err);
                    live = __all_sync(0xFFFFFFFFu, live);
                    if (!live) break;
                    const bool patch = kv == 1 && stale < kKeyTile;
                    const uint32_t bar = shared_at(patch ? &landed : &full[slot]), dst = shared_at(ring) + slot * C::kTileBytes;
                    if (lane == 0) bar_expect(bar, C::kTileBytes);
                    __syncwarp();
                    const int i = lane / C::kChunks, c = lane % C::kChunks;  // box, column
                    const int from = __shfl_sync(0xFFFFFFFFu, page, (i * box.rows / 16) & 7);
                    if (i < per) {
                        const int token = from >= 0 ? (base + i * box.rows) % a.c.page_size : 0;
                        const int g = from >= 0 ? from : a.c.n_pages;  // outside the pool: zeros
                        tma_4d(dst + c * C::kChunkBytes + i * box.rows * 128, kv ? &vmap : &kmap, c * 64, box.inside ? pc.head : token, box.inside ? token : pc.head, g, bar);
                    }
                    if (patch) {
                        live = __all_sync(0xFFFFFFFFu, bar_wait(bar, lands++ & 1, err));
                        const int rows = (stale + box.rows - 1) / box.rows * box.rows - stale;
                        for (int u = lane; u < rows * 8 * C::kChunks; u += 32) {
                            const int row = stale + u % rows, unit = u / rows;  // the swizzle stays within a row
                            *reinterpret_cast<uint4*>(ring + slot * C::kTileBytes + (unit / 8) * C::kChunkBytes + row * 128 + (unit % 8) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_async();
                        __syncwarp();
                        if (lane == 0) bar_arrive(shared_at(&full[slot]));
                    }
                }
            }
        }
        if (!live)  // every copy that is under way lands before the block ends
            for (uint32_t i = n > C::kSlots ? n - C::kSlots : 0; i < n; ++i) bar_wait(shared_at(&full[i % C::kSlots]), (i / C::kSlots) & 1, err);
    } else if (warp == 8) {
        // ---------------- products
        constexpr uint32_t qk = instruction(kRowTile, kKeyTile, false), pv = instruction(kRowTile, DP, true);
        uint32_t n = 0, ps[2] = {0, 0}, qn[2] = {0, 0};
        bool live = true;
        auto wait = [&](uint64_t* b, uint32_t par) {
            live = live && bar_wait(shared_at(b), par & 1, err);
            fence_after();
        };
        auto scores = [&](int t, uint32_t slot) {
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_ss(tmem + 128 * t, k_major(shared_at(qs) + t * C::kTileBytes + c * C::kChunkBytes + 32 * k),
                           k_major(shared_at(ring) + slot * C::kTileBytes + c * C::kChunkBytes + 32 * k), qk, c + k > 0);
            commit(shared_at(&s_full[t]));
        };
        auto values = [&](int t, uint32_t slot, bool add) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, n_major(shared_at(ring) + slot * C::kTileBytes + 2048 * k), pv, add || k > 0);
        };
        if (lane == 0) {
            for (uint32_t i = 0; live; ++i) {
                const Known& kn = known[i % kPieces];
                wait(&known_full[i % kPieces], i / kPieces);
                const bool none = !live || kn.last;
                const Piece<kKeyTile>& pc = kn.piece;
                if (none) break;
                const int steps = pc.steps;
                const int both = pc.b.rows > kRowTile ? 2 : 1;
                bar_arrive(shared_at(&known_empty[i % kPieces]));
                if (steps > 0) {
                    for (int t = 0; t < both; ++t) wait(&q_full[t], qn[t]++);
                    wait(&full[n % C::kSlots], n / C::kSlots);
                    for (int t = 0; t < both && live; ++t) scores(t, n % C::kSlots);
                    commit(shared_at(&empty[n % C::kSlots]));
                    ++n;
                    for (int j = 0; j < steps && live; ++j) {
                        const uint32_t v = n % C::kSlots, k = (n + 1) % C::kSlots;
                        const bool more = j + 1 < steps;
                        for (int t = 0; t < both && live; ++t) {
                            if (t == 0) wait(&full[v], n / C::kSlots);
                            wait(&p_full[t], ps[t]++);
                            if (live) values(t, v, j > 0);
                            if (t == both - 1) commit(shared_at(&empty[v]));
                            if (more) {
                                if (t == 0) wait(&full[k], (n + 1) / C::kSlots);
                                if (live) scores(t, k);
                                if (t == both - 1) commit(shared_at(&empty[k]));
                            } else {
                                commit(shared_at(&o_full[t]));
                            }
                        }
                        n += more ? 2 : 1;
                    }
                }
            }
            // nothing is left running when TMEM is given back
            commit(shared_at(&drained));
            bar_wait(shared_at(&drained), 0, err);
        }
        __syncwarp();
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
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
    tc_kernel<DP><<<grid, kThreads, Cfg<DP>::kSmem, s>>>(a, w, (int)entries, ctx->err_dev, Boxes{maps.box_rows, maps.inside}, k, v, tab);
    const int rc = check_launch(ctx, "attention kernel");
    if (rc) return rc;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, kRows / 32), cfg.blockDim = dim3(128), cfg.stream = s, cfg.attrs = &at, cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, tc_join_kernel<DP>, a, w, tab);
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
