// The launches of an attention call (csrc/attention_groups.h): each sequence of the
// lengths asked for is in one of them, in its place, and a launch's blocks of rows can
// be numbered in ints by steps of a thread block's threads.
#include <climits>
#include <cstdio>
#include <random>
#include <vector>

#include "attention_groups.h"

using namespace strata;

static int failures = 0;
#define EXPECT(cond)                                                                      \
    do {                                                                                  \
        if (!(cond) && ++failures < 10) std::printf("line %d: %s\n", __LINE__, #cond);    \
    } while (0)

constexpr int64_t kStep = 1024;  // threads of a block at most

static void uniform(int64_t n_seq, int64_t seq_len, int r, int per) {
    strata_attention d = {};
    d.n_seq = n_seq, d.seq_len = seq_len;
    const int64_t blocks = (seq_len * r + per - 1) / per;
    int64_t next = 0;
    const int rc = for_row_groups(d, r, per, 1, kMaxTokens + 1, [&](const SeqTable& t, int64_t entries) {
        EXPECT(t.uniform && t.slot0 == next && t.first == next * seq_len && t.pitch == seq_len && t.len_all == seq_len && t.tiles_all == blocks);
        EXPECT(t.n > 0 && entries == t.n * blocks && entries + kStep <= INT_MAX);
        next += t.n;
        return STRATA_OK;
    });
    EXPECT(rc == STRATA_OK && next == n_seq);
}

static void ragged(const std::vector<int64_t>& lens, int64_t start, int r, int per, int64_t from, int64_t below) {
    std::vector<int64_t> off = {start};
    for (int64_t n : lens) off.push_back(off.back() + n);
    strata_attention d = {};
    d.n_seq = (int64_t)lens.size(), d.seq_offsets = off.data();
    size_t at = 0;
    auto skip = [&] {
        while (at < lens.size() && (lens[at] <= 0 || lens[at] < from || lens[at] >= below)) ++at;
    };
    const int rc = for_row_groups(d, r, per, from, below, [&](const SeqTable& t, int64_t entries) {
        EXPECT(!t.uniform && t.n > 0 && t.n <= kSeqGroup && t.tile[0] == 0 && t.tile[t.n] == entries && entries + kStep <= INT_MAX);
        for (int i = 0; i < t.n; ++i, ++at) {
            skip();
            EXPECT(at < lens.size() && t.slot[i] == (int64_t)at && t.row[i] == off[at] && t.len[i] == lens[at]);
            EXPECT(t.tile[i + 1] - t.tile[i] == (lens[at] * r + per - 1) / per);
        }
        return STRATA_OK;
    });
    skip();
    EXPECT(rc == STRATA_OK && at == lens.size());
}

int main() {
    for (int per : {16, 256}) {
        for (int64_t n : {1, 7, 225}) uniform(n, 1, 4, per), uniform(n, 50, 1, per), uniform(n, 1000, 16, per);
        uniform(kMaxTokens, 1, 1, per), uniform(kMaxTokens - 300, 1, 65536, per), uniform(1 << 20, 2047, 16, per);
        uniform(1, kMaxTokens, 1, per), uniform(3, kMaxTokens / 4, 4, per);
        std::mt19937 rng(1);
        for (int64_t from : {1, 8})
            for (int64_t below : {int64_t(8), kMaxTokens + 1})
                for (int n : {1, 5, 224, 225, 700}) {
                    std::vector<int64_t> lens(n);
                    for (auto& v : lens) v = rng() % 4 ? rng() % 20 : rng() % 3000;
                    ragged(lens, rng() % 5, 1 + rng() % 9, per, from, below);
                }
        ragged(std::vector<int64_t>(40, 1 << 15), 0, 65536, per, 1, kMaxTokens + 1);  // 2^31 rows each, nearly
    }
    int calls = 0;
    strata_attention d = {};
    d.n_seq = kMaxTokens, d.seq_len = 1;
    EXPECT(for_row_groups(d, 1, 16, 1, kMaxTokens + 1, [&](const SeqTable&, int64_t) { return ++calls, STRATA_ERR_CUDA; }) == STRATA_ERR_CUDA && calls == 1);
    d.seq_len = 0;
    EXPECT(for_row_groups(d, 1, 16, 1, kMaxTokens + 1, [&](const SeqTable&, int64_t) { return ++calls, STRATA_ERR_CUDA; }) == STRATA_OK && calls == 1);
    if (!failures) std::puts("ok");
    return failures ? 1 : 0;
}
