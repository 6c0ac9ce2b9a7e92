// sequence.cuh — what the sequence operators share: the sequences of a call
// as a kernel parameter, typed vector access, and the call's device.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "runtime.cuh"
#include "sequence_args.h"

namespace strata {

// Makes the context's device current for the call and puts back the caller's.
struct DeviceGuard {
    int before = -1;
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        if (before != device) cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// The sequences of one launch, by value in the kernel's parameters: no copy
// to wait for, nothing to allocate, and a captured graph holds its own. Calls
// with more ragged sequences than kSeqGroup launch once per group.
constexpr int kSeqGroup = 256;
struct SeqTable {
    int n;                     // sequences in this launch
    int uniform;               // 1: sequence i holds rows [first + i * len, first + (i + 1) * len)
    int first, len, tiles;     // uniform: rows and tiles of each sequence
    int row[kSeqGroup + 1];    // ragged: first row of each sequence, and the row behind the last
    int tile[kSeqGroup + 1];   // ragged: tiles before each sequence
};

// Tile `b` of the launch: its sequence, that sequence's first row and number
// of rows, and the tile's number in it.
__device__ __forceinline__ void find_tile(const SeqTable& t, int b, int& seq, int& row, int& len, int& tile) {
    if (t.uniform) {
        seq = b / t.tiles;
        tile = b - seq * t.tiles;
        row = t.first + seq * t.len;
        len = t.len;
        return;
    }
    int lo = 0, hi = t.n;  // tile[lo] <= b < tile[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.tile[mid] <= b) lo = mid;
        else hi = mid;
    }
    seq = lo;
    row = t.row[lo];
    len = t.row[lo + 1] - row;
    tile = b - t.tile[lo];
}

// Calls launch(table, tiles, first sequence) for each group of sequences that has tiles of `rows` rows.
template <typename F>
int for_sequence_groups(int64_t n_seq, int64_t seq_len, const int64_t* off, int64_t rows, F launch) {
    if (!off) {
        if (seq_len == 0) return STRATA_OK;
        SeqTable t;
        t.n = (int)n_seq;
        t.uniform = 1;
        t.first = 0;
        t.len = (int)seq_len;
        t.tiles = (int)((seq_len + rows - 1) / rows);
        return launch(t, n_seq * t.tiles, int64_t(0));
    }
    for (int64_t s0 = 0; s0 < n_seq; s0 += kSeqGroup) {
        SeqTable t;
        t.n = (int)(n_seq - s0 < kSeqGroup ? n_seq - s0 : kSeqGroup);
        t.uniform = 0;
        t.first = t.len = t.tiles = 0;
        int64_t tiles = 0;
        for (int i = 0; i < t.n; ++i) {
            t.row[i] = (int)off[s0 + i];
            t.tile[i] = (int)tiles;
            tiles += (off[s0 + i + 1] - off[s0 + i] + rows - 1) / rows;
        }
        t.row[t.n] = (int)off[s0 + t.n];
        t.tile[t.n] = (int)tiles;
        if (!tiles) continue;
        const int rc = launch(t, tiles, s0);
        if (rc) return rc;
    }
    return STRATA_OK;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// VEC elements as they lie in memory: 16-byte accesses where VEC * sizeof(T)
// is 16, plain ones otherwise.
template <typename T, int VEC>
struct alignas(VEC * sizeof(T) >= 16 ? 16 : VEC * sizeof(T)) Pack {
    T v[VEC];
};

}  // namespace strata
