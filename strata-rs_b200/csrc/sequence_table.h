// sequence_table.h — the sequences of a call in the launches' parameters. Host only
// and free of CUDA, as sequence_args.h.
#pragma once
#include "sequence_args.h"

namespace strata {

// The sequences of one launch, by value in the kernel's parameters: no copy
// to wait for, nothing to allocate, and a captured graph holds its own. Empty
// sequences are left out; calls with more ragged sequences than kSeqGroup
// launch once per group.
constexpr int kSeqGroup = 224;  // with its four numbers a sequence, the table stays within 4 KB
struct SeqTable {
    int n;                   // sequences in this launch
    int uniform;             // 1: sequence i is state `slot0 + i`, rows from first + i * pitch, all len long
    int first, pitch, slot0, len_all, tiles_all;
    int row[kSeqGroup];      // ragged: first row,
    int len[kSeqGroup];      // rows,
    int slot[kSeqGroup];     // number in the call (its state's),
    int tile[kSeqGroup + 1]; // and tiles before each sequence
};

inline SeqTable uniform_table(int64_t n, int64_t first, int64_t pitch, int64_t slot0, int64_t len, int64_t rows) {
    SeqTable t;
    t.n = (int)n;
    t.uniform = 1;
    t.first = (int)first;
    t.pitch = (int)pitch;
    t.slot0 = (int)slot0;
    t.len_all = (int)len;
    t.tiles_all = (int)((len + rows - 1) / rows);
    return t;
}
inline SeqTable ragged_table() {
    SeqTable t;
    t.n = t.uniform = 0;
    t.first = t.pitch = t.slot0 = t.len_all = t.tiles_all = 0;
    t.tile[0] = 0;
    return t;
}
inline void add_sequence(SeqTable& t, int64_t slot, int64_t row, int64_t len, int64_t rows) {
    t.slot[t.n] = (int)slot;
    t.row[t.n] = (int)row;
    t.len[t.n] = (int)len;
    t.tile[t.n + 1] = t.tile[t.n] + (int)((len + rows - 1) / rows);
    ++t.n;
}

// Calls launch(table, tiles) for each group of sequences, cut into tiles of
// `rows` rows. Of ragged ones those below `below` rows only.
template <typename F>
int for_sequence_groups(int64_t n_seq, int64_t seq_len, const int64_t* off, int64_t rows, int64_t below, F launch) {
    if (!off) {
        if (seq_len == 0) return STRATA_OK;
        const SeqTable t = uniform_table(n_seq, 0, seq_len, 0, seq_len, rows);
        return launch(t, n_seq * t.tiles_all);
    }
    SeqTable t = ragged_table();
    for (int64_t i = 0; i < n_seq; ++i) {
        const int64_t len = off[i + 1] - off[i];
        if (len > 0 && len < below) add_sequence(t, i, off[i], len, rows);
        if (t.n == kSeqGroup || (i + 1 == n_seq && t.n)) {
            const int rc = launch(t, (int64_t)t.tile[t.n]);
            if (rc) return rc;
            t = ragged_table();
        }
    }
    return STRATA_OK;
}

}  // namespace strata
