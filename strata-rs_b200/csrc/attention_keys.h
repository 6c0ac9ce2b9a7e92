// attention_keys.h — which keys a block of rows of the attention kernels sees, in
// tiles. Free of CUDA, so that it is tested on the host as well
// (tests/attention_keys_check.cpp).
#pragma once

#ifdef __CUDACC__
#define STRATA_BOTH __host__ __device__ __forceinline__
#else
#define STRATA_BOTH inline
#endif

namespace strata {

// The keys that some row of a block sees: [0, sink) and [lo, hi); in tiles of
// TILE keys, first those of the sinks, then those from lo on.
template <int TILE>
struct KeyRange {
    int lo, hi, sink_tiles, tiles;
    STRATA_BOTH int key(int tile) const { return (tile < sink_tiles ? tile : lo / TILE + (tile - sink_tiles)) * TILE; }
};
// Tiles of n keys, 0 <= n < 2^31 (n + TILE - 1 may be above what an int holds).
template <int TILE>
STRATA_BOTH int tiles_of(int n) { return n / TILE + (n % TILE > 0); }

// Of rows at positions p_min to p_max (from below 0 to 2^31 - 2), over a table that
// reaches `cap` positions (below 2^31).
template <int TILE>
STRATA_BOTH KeyRange<TILE> key_range(int window, int sinks, int cap, int p_min, int p_max) {
    KeyRange<TILE> k;
    k.hi = p_max < cap ? p_max + 1 : cap;
    if (k.hi < 0) k.hi = 0;
    k.lo = window && p_min >= window ? p_min - window + 1 : 0;
    if (k.lo > k.hi) k.lo = k.hi;
    const int sink = sinks < k.lo ? sinks : k.lo, first = k.lo / TILE;
    k.sink_tiles = tiles_of<TILE>(sink);
    if (k.sink_tiles > first) k.sink_tiles = first;  // the rest lies in lo's own tile
    k.tiles = k.sink_tiles + tiles_of<TILE>(k.hi) - first;
    return k;
}

}  // namespace strata
