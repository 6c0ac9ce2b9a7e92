// attention_groups.h — the sequences of an attention call as launches. Host only and
// free of CUDA, as sequence_args.h; tested without a device (tests/attention_groups_check.cpp).
#pragma once
#include <algorithm>

#include "../../include/strata_attention.h"
#include "sequence_table.h"

namespace strata {

// Blocks of rows of a launch at most. Thread blocks go through their numbers in steps of
// their threads, in ints, so the last step has to end below 2^31; one sequence has 2^27 at
// most (kMaxTokens rows a key head, 16 a block).
constexpr int64_t kMaxEntries = int64_t(1) << 30;

// Calls launch(table, entries) for each group of the sequences of `from` tokens or
// more but below `below`, cut into blocks of `per` rows.
template <typename F>
int for_row_groups(const strata_attention& d, int r, int per, int64_t from, int64_t below, F launch) {
    auto blocks = [&](int64_t n) { return (n * r + per - 1) / per; };
    if (!d.seq_offsets) {
        if (d.seq_len < from || d.seq_len >= below) return STRATA_OK;
        const int64_t most = kMaxEntries / blocks(d.seq_len);  // sequences of a launch
        for (int64_t first = 0; first < d.n_seq; first += most) {
            const int64_t n = std::min(most, d.n_seq - first);
            SeqTable t = uniform_table(n, first * d.seq_len, d.seq_len, first, d.seq_len, 1);
            t.tiles_all = (int)blocks(d.seq_len);
            const int rc = launch(t, n * t.tiles_all);
            if (rc) return rc;
        }
        return STRATA_OK;
    }
    SeqTable t = ragged_table();
    int64_t entries = 0;
    for (int64_t i = 0; i < d.n_seq; ++i) {
        const int64_t n = d.seq_offsets[i + 1] - d.seq_offsets[i];
        if (n > 0 && n >= from && n < below) {
            if (t.n == kSeqGroup || entries + blocks(n) > kMaxEntries) {
                const int rc = launch(t, entries);
                if (rc) return rc;
                t = ragged_table();
                entries = 0;
            }
            add_sequence(t, i, d.seq_offsets[i], n, 1);
            entries += blocks(n);
            t.tile[t.n] = (int)entries;
        }
    }
    return t.n ? launch(t, entries) : STRATA_OK;
}

}  // namespace strata
