// The tiles of keys that a block of rows goes through (csrc/attention_keys.h): every
// key that a row sees lies in exactly one of them, for small tables by trying all
// positions, and next to 2^31 positions by the same numbers in 64 bits.
#include <cstdint>
#include <cstdio>
#include <vector>

#include "attention_keys.h"

using namespace strata;

static int failures = 0;
#define EXPECT(cond, ...)                                                              \
    do {                                                                               \
        if (!(cond)) {                                                                 \
            if (++failures < 10) std::printf("line %d: %s: ", __LINE__, #cond), std::printf(__VA_ARGS__), std::puts(""); \
        }                                                                              \
    } while (0)

template <int TILE>
static void small() {
    for (int cap : {16, 32})
        for (int window : {0, 1, 2, 5, 15, 16, 17, 31, 32, 33, 60})
            for (int sinks : {0, 1, 3, 16, 40})
                for (int p_min = -3; p_min < 50; ++p_min)
                    for (int p_max = p_min; p_max < p_min + 9; ++p_max) {
                        const auto k = key_range<TILE>(window, window ? sinks : 0, cap, p_min, p_max);
                        std::vector<int> times(128, 0);
                        EXPECT(k.tiles >= 0 && k.sink_tiles >= 0, "%d %d %d", k.tiles, p_min, p_max);
                        for (int t = 0; t < k.tiles; ++t)
                            for (int j = k.key(t); j < k.key(t) + TILE; ++j) ++times[j];
                        for (int j = 0; j < cap; ++j) {
                            bool seen = false;
                            for (int p = p_min; p <= p_max; ++p) seen |= j <= p && (!window || j > p - window || j < sinks);
                            EXPECT(times[j] <= 1 && (!seen || times[j] == 1), "window %d sinks %d cap %d rows %d to %d key %d: %d", window, sinks, cap, p_min, p_max, j, times[j]);
                        }
                    }
}

template <int TILE>
static void large() {
    const int64_t end = (int64_t(1) << 31) - 1;
    for (int64_t cap : {end - 15, end - 31, end - 63, end - 127, end - 255})
        for (int64_t p_max : {end - 1, cap, cap - 1, cap - 40, cap - 1000})
            for (int64_t rows : {1, 300})
                for (int64_t window : {int64_t(0), int64_t(1), int64_t(100), int64_t(5000), end - 2, end - 1})
                    for (int64_t sinks : {int64_t(0), int64_t(7), end - 200, end}) {
                        const int64_t p_min = p_max - rows + 1;
                        const int64_t hi = p_max + 1 < cap ? p_max + 1 : cap;
                        int64_t lo = window && p_min >= window ? p_min - window + 1 : 0;
                        if (lo > hi) lo = hi;
                        const int64_t first = lo / TILE;
                        int64_t sink = ((window ? sinks < lo ? sinks : lo : 0) + TILE - 1) / TILE;
                        if (sink > first) sink = first;
                        const auto k = key_range<TILE>((int)window, window ? (int)sinks : 0, (int)cap, (int)p_min, (int)p_max);
                        EXPECT(k.lo == lo && k.hi == hi && k.sink_tiles == sink && k.tiles == sink + (hi + TILE - 1) / TILE - first,
                               "window %lld sinks %lld cap %lld rows %lld to %lld: %d tiles", (long long)window, (long long)sinks, (long long)cap, (long long)p_min, (long long)p_max, k.tiles);
                        if (k.tiles > 0) EXPECT(k.key(k.tiles - 1) >= 0 && k.key(k.tiles - 1) <= hi, "the last tile's keys begin at %d", k.key(k.tiles - 1));
                    }
}

int main() {
    small<4>(), small<16>(), large<64>(), large<128>();
    if (!failures) std::puts("ok");
    return failures ? 1 : 0;
}
