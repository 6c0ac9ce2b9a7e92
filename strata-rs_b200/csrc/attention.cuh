// attention.cuh — what the attention kernels share: the cache and the call as
// kernel parameters, which keys a block of rows sees, and one row computed
// from the formula alone.
#pragma once
#include "attention_args.h"
#include "sequence.cuh"

namespace strata {

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
    float scale, scale2;  // the second in powers of two: scale * log2(e)
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

// The keys that some row of a block sees: [0, sink) and [lo, hi); in tiles of
// kTile keys, first those of the sinks, then those from lo on.
constexpr int kTile = 64;
struct KeyRange {
    int lo, hi, sink_tiles, tiles;
    __device__ __forceinline__ int key(int tile) const {
        return (tile < sink_tiles ? tile : lo / kTile + (tile - sink_tiles)) * kTile;
    }
};
__device__ __forceinline__ KeyRange key_range(const AttnArgs& a, int p_min, int p_max) {
    KeyRange k;
    const int cap = a.c.max_pages * a.c.page_size;  // below 2^31
    k.hi = p_max < cap ? p_max + 1 : cap;
    if (k.hi < 0) k.hi = 0;
    k.lo = a.window && p_min >= a.window ? p_min - a.window + 1 : 0;
    if (k.lo > k.hi) k.lo = k.hi;
    const int sink = a.sinks < k.lo ? a.sinks : k.lo, first = k.lo / kTile;
    k.sink_tiles = (sink + kTile - 1) / kTile;
    if (k.sink_tiles > first) k.sink_tiles = first;  // the rest lies in lo's own tile
    k.tiles = k.sink_tiles + (k.hi + kTile - 1) / kTile - first;
    return k;
}
__device__ __forceinline__ KeyRange key_range(const AttnArgs& a, const RowBlock& b) {
    return key_range(a, b.p0 + b.row0 / a.r, b.p0 + (b.row0 + b.rows - 1) / a.r);
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
    const KeyRange kr = key_range(a, p, p);
    for (int tile = 0; tile < kr.tiles; ++tile)
        for (int half = 0; half < kTile; half += 32) {
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
            for (unsigned left = any; left; left &= left - 1) {
                const int from = __ffs(left) - 1;
                const float w = __shfl_sync(0xFFFFFFFFu, e, from);
                const int64_t row = __shfl_sync(0xFFFFFFFFu, at, from);
                l += w;
                for (int i = 0; i < 8; ++i)
                    if (lane + 32 * i < d) o[i] = fmaf(w, __bfloat162float(a.c.v[row + lane + 32 * i]), o[i]);
            }
        }
    T* out = static_cast<T*>(a.o) + (int64_t)token * a.o_stride + (int64_t)head * d;
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < d) from_f32(out[lane + 32 * i], seen ? o[i] / l : 0.0f);
}

}  // namespace strata
