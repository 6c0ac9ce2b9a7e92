// sequence.cuh — what the sequence operators share: the sequences of a call
// as a kernel parameter, typed vector access, and the call's device.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "runtime.cuh"
#include "sequence_table.h"

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
