// attention.cuh — what the attention kernels share: the cache and the call as
// kernel parameters, which keys a block of rows sees, and one row computed
// from the formula alone.
#pragma once
#include "attention_args.h"
#include "attention_groups.h"
#include "attention_keys.h"
#include "sequence.cuh"

namespace strata {

// Launches that overlap the kernel before them in the stream: a block starts while
// that one ends, finds its own bearings and waits for its end (and its writes) with
// after_previous() before it touches memory.
template <typename K, typename... A>
cudaError_t launch_early(K kernel, dim3 grid, int threads, int shared, cudaStream_t s, A... args) {
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = shared, cfg.stream = s, cfg.attrs = &at, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
// Where `next` is set, the kernel behind may then start likewise; a join does not let it:
// its blocks' shared memory would keep blocks of the next attention kernel, which fill
// the multiprocessors exactly, for a second round (64 tokens with heads of 64: 92, 112 us).
__device__ __forceinline__ void after_previous(bool next = true) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (next) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

struct CacheArgs {
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    const int* table;
    const int* len;
    int64_t page_stride, token_stride, head_stride, table_stride;
    int n_pages, page_size, max_pages, n_kv_head, head_dim;
};
inline CacheArgs cache_args(const strata_kv_cache& c) {
    return {static_cast<const __nv_bfloat16*>(c.k_dev), static_cast<const __nv_bfloat16*>(c.v_dev), c.table_dev, c.len_dev,
            c.page_stride, c.token_stride, c.head_stride, c.table_stride, (int)c.n_pages, (int)c.page_size,
            (int)c.max_pages, (int)c.n_kv_head, (int)c.head_dim};
}

struct AttnArgs {
    CacheArgs c;
    const void* q;
    void* o;
    int64_t q_stride, o_stride;
    int r;              // queries' heads a key head
    int window, sinks;  // window 0: none
    float scale2;       // in powers of two: scale * log2(e)
    int wide;           // rows of q and o can be accessed in 16-byte packs
};

// Rows of a key head's queries lie token by token, r heads each: row i of a
// sequence is head i % r of its token i / r. A block of them:
struct RowBlock {
    int slot, first_row, n;  // the sequence: its number, first row of the call, tokens
    int row0, rows;          // the block's rows
    int p0;                  // position of the sequence's first new token (may be negative)
};

__device__ __forceinline__ RowBlock row_block(const AttnArgs& a, const Seq& s, int tile, int per) {
    RowBlock b;
    b.slot = s.slot, b.first_row = s.row, b.n = s.len;
    b.row0 = (tile - s.tile0) * per;
    const int left = s.len * a.r - b.row0;
    b.rows = left < per ? left : per;
    const int len = a.c.len[s.slot];
    b.p0 = (len > 0 ? len : 0) - s.len;
    return b;
}

template <int TILE>
__device__ __forceinline__ KeyRange<TILE> key_range(const AttnArgs& a, int p_min, int p_max) {
    return key_range<TILE>(a.window, a.sinks, a.c.max_pages * a.c.page_size, p_min, p_max);
}
// The keys that some row of a block sees.
template <int TILE>
__device__ __forceinline__ KeyRange<TILE> key_range(const AttnArgs& a, const RowBlock& b) {
    return key_range<TILE>(a, b.p0 + b.row0 / a.r, b.p0 + (b.row0 + b.rows - 1) / a.r);
}
__device__ __forceinline__ bool sees(const AttnArgs& a, int p, int j) {
    return j <= p && (!a.window || j > p - a.window || j < a.sinks);
}

// The page of position j (below the table's reach) of sequence `slot`, or -1.
__device__ __forceinline__ int page_of(const CacheArgs& c, int slot, int j) {
    const int g = c.table[(int64_t)slot * c.table_stride + j / c.page_size];
    return g >= 0 && g < c.n_pages ? g : -1;
}
__device__ __forceinline__ int64_t place(const CacheArgs& c, int page, int j, int head) {
    return (int64_t)page * c.page_stride + (int64_t)(j % c.page_size) * c.token_stride + (int64_t)head * c.head_stride;
}

template <typename T>
__device__ __forceinline__ float load_f32(const void* base, int64_t i) { return to_f32(static_cast<const T*>(base)[i]); }

// The work of all blocks of rows and key heads of a launch, cut evenly over its
// thread blocks: this one's contiguous range of units. A block of rows costs OVER
// units for its queries and outputs, then one a tile (one at least, so that rows
// that see nothing are written).
struct Cut {
    int64_t total, grid;    // units, and thread blocks that get some
    int64_t pos, end;       // this one's
    int entry;              // block of rows that `pos` lies in,
    int64_t entry_at;       // and its first unit
};
template <int ROWS, int TILE, int OVER>
__device__ __forceinline__ int cost_of(const AttnArgs& a, const SeqTable& tab, int entry) {
    const int n = key_range<TILE>(a, row_block(a, sequence_of_tile(tab, entry), entry, ROWS)).tiles;
    return OVER + (n > 0 ? n : 1);
}
// Prefix of v over the block's threads, and its total. `sh`: a number a warp.
template <int THREADS>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* sh, int64_t& total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int64_t x = v;
    for (int w = 1; w < 32; w <<= 1) {
        const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, w);
        if (lane >= w) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int i = 0; i < THREADS / 32; ++i) {
        if (i < warp) before += sh[i];
        total += sh[i];
    }
    return before + x - v;
}
// By all THREADS threads; blocks from c.grid on have none, the others LEAST units or so (half of that at least, or all
// there are). `sh`: THREADS / 32 + 2 numbers.
template <int THREADS, int ROWS, int TILE, int OVER, int LEAST>
__device__ __forceinline__ Cut cut_range(const AttnArgs& a, const SeqTable& tab, int entries, int64_t* sh) {
    Cut c;
    const int heads = a.c.n_kv_head;
    int64_t mine = 0, first = 0;
    for (int e0 = 0; e0 < entries; e0 += THREADS) {
        const int e = e0 + threadIdx.x;
        const int64_t cost = e < entries ? (int64_t)cost_of<ROWS, TILE, OVER>(a, tab, e) * heads : 0;
        if (e0 == 0) first = cost;
        mine += cost;
    }
    const int64_t prefix = block_scan<THREADS>(mine, sh, c.total);
    c.grid = (c.total + LEAST - 1) / LEAST < gridDim.x ? (c.total + LEAST - 1) / LEAST : (int64_t)gridDim.x;
    if (blockIdx.x >= c.grid) return c;
    c.pos = c.total * blockIdx.x / c.grid;
    c.end = c.total * (blockIdx.x + 1) / c.grid;
    int64_t base = 0;
    for (int e0 = 0; e0 < entries; e0 += THREADS) {
        const int e = e0 + threadIdx.x;
        const int64_t cost = e0 == 0 ? first : e < entries ? (int64_t)cost_of<ROWS, TILE, OVER>(a, tab, e) * heads : 0;
        int64_t sum = c.total, before = prefix;  // an entry a thread at most: known already
        if (entries > THREADS) before = base + block_scan<THREADS>(cost, sh, sum);
        if (cost && c.pos >= before && c.pos < before + cost) sh[THREADS / 32] = e, sh[THREADS / 32 + 1] = before;
        base += sum;
        if (base > c.pos) break;
    }
    __syncthreads();
    c.entry = (int)sh[THREADS / 32];
    c.entry_at = sh[THREADS / 32 + 1];
    return c;
}
// The piece of one block of rows and key head that begins at `c.pos`: tiles
// [tile0, tile1) of its `tiles`.
template <int TILE>
struct Piece {
    RowBlock b;
    KeyRange<TILE> kr;
    int head, cost;
    int64_t at;             // the first unit of the block of rows and head
    int64_t begin;          // this piece's
    int entry;
    int tiles, tile0, tile1;
    int steps;              // tiles with keys
    __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == tiles; }
    __device__ __forceinline__ int key(int step) const { return kr.key(tile0 + step); }
};
// The next piece of the thread block's range, from c.pos on; false at its end.
template <int ROWS, int TILE, int OVER>
__device__ __forceinline__ bool next_piece(const AttnArgs& a, const SeqTable& tab, Cut& c, Piece<TILE>& p) {
    while (c.pos < c.end) {
        p.b = row_block(a, sequence_of_tile(tab, c.entry), c.entry, ROWS);
        p.kr = key_range<TILE>(a, p.b);
        p.tiles = p.kr.tiles > 0 ? p.kr.tiles : 1;
        p.cost = OVER + p.tiles;
        p.entry = c.entry;
        p.head = (int)((c.pos - c.entry_at) / p.cost);
        p.at = c.entry_at + (int64_t)p.head * p.cost;
        p.begin = c.pos;
        const int u0 = (int)(c.pos - p.at), u1 = (int)(c.end - p.at < p.cost ? c.end - p.at : p.cost);
        p.tile0 = u0 > OVER ? u0 - OVER : 0;
        p.tile1 = u1 > OVER ? u1 - OVER : 0;
        p.steps = (p.kr.tiles < p.tile1 ? p.kr.tiles : p.tile1) - p.tile0;
        c.pos = p.at + u1;
        const int64_t all = (int64_t)p.cost * a.c.n_kv_head;
        if (c.pos >= c.entry_at + all) c.entry_at += all, ++c.entry;
        if (p.tile1 > p.tile0) return true;  // else the range ends within the block's first OVER units
    }
    return false;
}
// Which of a thread block's two places a piece's sums go to, where others have the rest.
template <int TILE>
__device__ __forceinline__ int slot_of(const Piece<TILE>& p, int64_t range_begin) { return p.begin == range_begin ? 0 : 1; }
// Thread blocks that have pieces of `p`, of which this one has the first: the
// last of them is the last that begins at or before its last unit.
template <int TILE>
__device__ __forceinline__ int pieces_of(const Cut& c, const Piece<TILE>& p) {
    return (int)(((p.at + p.cost) * c.grid - 1) / c.total - blockIdx.x) + 1;
}

// What a thread block leaves for the join: which block of rows it has the first piece of.
struct Split {
    int entry, head;
    int pieces;      // 0: none
    int first_slot;  // of the first piece; the others are their thread blocks' slot 0
};

// One row, by a warp, key by key and leaving out what it does not see: for rows
// whose result is not finite, since in a product of tiles a NaN or an infinity
// that a row does not see meets its weight of zero (and gives a NaN).
// A lane scores a key at a time and holds every 32nd element of the output.
template <typename T>
__device__ __noinline__ void careful_row(const AttnArgs& a, int slot, int token, int p, int head, int kv_head) {
    const int lane = threadIdx.x & 31, d = a.c.head_dim;
    const int64_t q = (int64_t)token * a.q_stride + (int64_t)head * d;
    float m = -INFINITY, l = 0.0f, o[8] = {};
    bool seen = false;
    const KeyRange<64> kr = key_range<64>(a, p, p);
    for (int tile = 0; tile < kr.tiles; ++tile)
        for (int half = 0; half < 64; half += 32) {
            const int j0 = kr.key(tile) + half, j = j0 + lane;
            float s = -INFINITY;
            bool live = j < kr.hi && sees(a, p, j);
            int64_t at = 0;
            if (live) {
                const int page = page_of(a.c, slot, j);
                live = page >= 0;
                if (live) at = place(a.c, page, j, kv_head);
            }
            if (live) {
                float sum = 0.0f;
                for (int i = 0; i < d; ++i) sum = fmaf(load_f32<T>(a.q, q + i), __bfloat162float(a.c.k[at + i]), sum);
                s = sum * a.scale2;
            }
            if (l != l) break;  // a NaN stays one
            const unsigned any = __ballot_sync(0xFFFFFFFFu, live);
            if (!any) continue;
            float top = s;
            bool nan = live && s != s;
            for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, w));
            const float next = fmaxf(m, top);
            const float alpha = m == next ? 1.0f : exp2f(m - next);
            // a score of -inf has no weight (where all are, the formula gives NaN: below)
            const float e = !live || s == -INFINITY ? 0.0f : nan ? s : exp2f(s - next);
            seen = true;
            m = next;
            l *= alpha;
            for (int i = 0; i < 8; ++i) o[i] *= alpha;
#pragma unroll 8
            for (int from = 0; from < 32; ++from) {
                const float w = __shfl_sync(0xFFFFFFFFu, e, from);
                const int64_t row = __shfl_sync(0xFFFFFFFFu, at, from);
                if (!(any >> from & 1)) continue;
                l += w;
                for (int i = 0; i < 8; ++i)
                    if (lane + 32 * i < d) o[i] = fmaf(w, __bfloat162float(a.c.v[row + lane + 32 * i]), o[i]);
            }
        }
    T* out = static_cast<T*>(a.o) + (int64_t)token * a.o_stride + (int64_t)head * d;
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < d) from_f32(out[lane + 32 * i], seen ? o[i] / l : 0.0f);
}

// attention_tc.cu: bf16 chunks with heads of up to 128 on the tensor cores, in
// blocks of attention_tc_rows() rows. The maps describe the pools to the copies;
// they fail where a stride is outside what a map can hold.
struct TcMaps {
    alignas(64) unsigned char k[128], v[128];
    int box_rows, inside;
};
int attention_tc_rows();
int64_t attention_tc_work_bytes(int dp);
bool attention_tc_maps(const CacheArgs& c, TcMaps* maps);
int launch_attention_tc(strata_ctx* ctx, int dp, const AttnArgs& a, void* work, const SeqTable& tab, int64_t entries, const TcMaps& maps,
                        cudaStream_t s);

}  // namespace strata
