// sequence.cuh — what the sequence operators share: the sequences of a call
// as a kernel parameter, typed vector access, and the call's device.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
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

// Lets `kernel` have `bytes` of dynamic shared memory on the current device:
// asked for once per device.
template <typename K>
cudaError_t allow_shared(K kernel, int bytes, std::atomic<uint64_t>& asked, int device) {
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device < 64 && (asked.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

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

// A sequence of a launch as a kernel sees it.
struct Seq {
    int slot, row, len;
    int tile0;  // tiles of the sequences before it
};

__device__ __forceinline__ Seq sequence_at(const SeqTable& t, int i) {
    if (t.uniform) return Seq{t.slot0 + i, t.first + i * t.pitch, t.len_all, i * t.tiles_all};
    return Seq{t.slot[i], t.row[i], t.len[i], t.tile[i]};
}

// The sequence that tile `b` of the launch belongs to.
__device__ __forceinline__ Seq sequence_of_tile(const SeqTable& t, int b) {
    if (t.uniform) return sequence_at(t, b / t.tiles_all);
    int lo = 0, hi = t.n;  // tile[lo] <= b < tile[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.tile[mid] <= b) lo = mid;
        else hi = mid;
    }
    return sequence_at(t, lo);
}

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

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// VEC elements as they lie in memory: one access where VEC is a power of two
// (16 bytes at most), plain ones otherwise.
template <typename T, int VEC>
struct alignas(VEC & (VEC - 1) ? sizeof(T) : VEC * sizeof(T) >= 16 ? 16 : VEC * sizeof(T)) Pack {
    T v[VEC];
};

}  // namespace strata
