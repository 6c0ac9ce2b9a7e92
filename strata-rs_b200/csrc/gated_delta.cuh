// gated_delta.cuh — what the two forms of the gated delta rule share: the
// call's buffers, the gates, and the entry of the chunked form.
#pragma once
#include "sequence.cuh"

namespace strata {

struct DeltaArgs {
    const void *q, *k, *v;
    const float *gate, *beta, *coef, *shift;
    float* state;
    void* o;
    int64_t q_stride, k_stride, v_stride, o_stride, gate_stride, beta_stride;
    int k_heads, v_heads, k_dim, v_dim;
    int col_blocks;
    int tiled, raw_gates, norm;
    float scale, eps;
};

__device__ __forceinline__ int key_head(const DeltaArgs& a, int h) {
    return a.tiled ? h % a.k_heads : h / (a.v_heads / a.k_heads);
}

// The log of the decay and the step of value head h from what the call gives.
__device__ __forceinline__ void gates(const DeltaArgs& a, int h, float& g, float& beta) {
    if (!a.raw_gates) return;
    const float z = g + (a.shift ? a.shift[h] : 0.0f);
    g = a.coef[h] * (fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z))));  // softplus without overflow
    beta = 1.0f / (1.0f + expf(-beta));
}

// gated_delta_chunk.cu: the call's sequences of `from` tokens (1 at least) and more.
uint64_t delta_chunk_work(const strata_gated_delta& d, int64_t from);
int delta_chunk_enqueue(strata_ctx* ctx, const strata_gated_delta& d, const DeltaArgs& a, void* work, int64_t from,
                        cudaStream_t s);

}  // namespace strata
