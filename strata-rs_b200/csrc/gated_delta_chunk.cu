// gated_delta_chunk.cu — the gated delta rule over prompts, kChunk tokens at a
// time, on the tensor cores.
//
// With G_i the sum of the log decays of a chunk's tokens up to i, the updates
// u_i = beta_i (v_i - e^{g_i} S_{i-1}^T k_i) of a chunk that starts at state S
// solve (I + A) U = X with
//   A_ij = beta_i e^{G_i - G_j} k_i . k_j  (i > j),
//   X_i  = beta_i (v_i - e^{G_i} S^T k_i),
// and then
//   o_i = scale (e^{G_i} S^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) u_j),
//   S  <- e^{G_C} S + sum_j e^{G_C - G_j} k_j u_j^T.
// T = (I + A)^-1 and P_ij = e^{G_i - G_j} (q_i . k_j) do not depend on S:
// delta_prepare_kernel computes them for all chunks at once (and U = T X needs
// no second product with the keys). delta_scan_kernel then goes through the
// chunks of a sequence in order with S in registers.
//
// Precision. Products over k_dim run on the tensor cores as f16 limbs: x 2^e =
// hi + lo with the exponent e taken per vector (a key, a query, a column of S)
// from its largest magnitude. A limb pair carries 22 bits of what is within 2^-18
// of that, 2^-40 of it below, and lo hi + hi lo + hi hi is summed in f32, the two
// small products first. That keeps f32-like results at f16 rate; plain tf32 would
// carry 11 bits. Keys and queries given as bf16 are exact in one limb.
// The two triangular products over a chunk's tokens, T X and P U, take tf32 limbs
// instead, which have f32's exponents: tokens of one column may differ by any
// factor (outliers, states that grow), and a scale shared by a chunk would let
// later ones take bits from earlier ones. hi is rounded, so that lo lacks the last
// of f32's bits at most. (In plain f32 on the CUDA cores these two cost 0.38 us a
// chunk: reading the operands for a dot product a lane fills shared memory's
// bandwidth.) Only what is added to S at the chunk's end, a sum over its tokens
// anyway, shares a scale per column and 16 tokens. The scan adds to S outside the
// tensor core, where the addition rounds to nearest.
//
// Layout of the scan. The columns of S are independent, and products are
// written transposed: a group of warps has 16 columns of S as the 16 rows of
// m16n8k16 (k8 in tf32) products, S^T K^T, X^T T^T, U^T P^T, U^T K. An accumulator
// tile is then, split into limbs, the left operand of the next product as it lies,
// and the right operands (keys, queries, T, P) are the same for all columns: they
// are staged in shared memory by bulk copies one chunk ahead.
// Two warps of a group hold half of S's rows each and follow the chain from
// chunk to chunk; the sums over k_dim, X and U go between them through shared
// memory, half of the tokens each. Two more take S's limbs and U from there and
// compute half of the chunk's outputs each, off the chain, up to a chunk behind.
// One sequence is bound by that chain (about 3000 cycles a chunk of 32 tokens at
// k_dim 128 and f32: a conversion, a product, an exchange, three times over); a
// batch by how many groups share a multiprocessor, four where shared memory
// allows.
//
// Measured at 32 value and 16 key heads of 128 x 128: one sequence of 8192 f32
// tokens 623 us, 86 of it prepare (366 MB, 4.3 TB/s; warps wait for loads and
// for their row sums) and 535 the scan (2.1 us a chunk, 128 blocks). The tensor
// pipe is busy for 36% of the scan's cycles: chunks of 64 would halve the steps
// of the chain, but their images do not fit shared memory three deep. Eight bf16
// sequences of 1 to 2049 tokens, 7036 in all, 416 us (84 and 327).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "gated_delta.cuh"

namespace strata {
namespace {

constexpr int kChunk = 32;
constexpr int kThreads = 128;                  // of a prepare block
constexpr int kPitchT = kChunk + 8;            // floats of a row of T or P: 32-byte steps that no two of 4 rows share
constexpr int kMatT = kChunk * kPitchT * 4;
constexpr int kGates = 2 * kMatT;              // T, P, then the gate rows; the last one starts with e^{G_C}
enum { kBeta, kXk, kOq, kDown, kTotal, kGateRows };
constexpr int kImageT = kGates + kGateRows * kChunk * 4;
constexpr uint64_t kMaxWork = uint64_t(256) << 20;

// The image of a chunk's keys and queries: K limbs, then Q limbs, rows of
// DK halves padded to 16-byte steps that no two of 8 rows share.
template <int DK, int LIMBS>
struct Image {
    static constexpr int kPitch = DK * 2 + 16;
    static constexpr int kLimb = kChunk * kPitch;
    static constexpr int kBytes = 2 * LIMBS * kLimb;
};

// The power of two that brings a number of this (biased) exponent to [2^14, 2^15),
// and its inverse. Both stay normal numbers.
__device__ __forceinline__ void power_of(uint32_t exponent, float& up, float& down) {
    int f = 268 - (int)exponent;
    f = f < 2 ? 2 : f > 252 ? 252 : f;
    up = __uint_as_float((uint32_t)f << 23);
    down = __uint_as_float((uint32_t)(254 - f) << 23);
}
__device__ __forceinline__ void power_for(float m, float& up, float& down) {
    power_of((__float_as_uint(m) >> 23) & 255u, up, down);
}

// (x, y) as two f16 limbs, packed with x in the low half.
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(  // no state but its registers: free to be scheduled
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same of 8 products, tf32: what a register holds beyond 11 bits is not read.
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// x as two tf32 limbs. A NaN whose bits carry into the sign is still one in lo.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ uint32_t shared_addr(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

// Copies `bytes` (a multiple of 16) into shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// Waits for a phase of `bar`, a second at most: false if it has not completed by then.
__device__ __forceinline__ bool bulk_wait(uint32_t bar, uint32_t parity) {
    uint64_t begun = 0;
    for (long long i = 0; i < kSpinLimit; ++i) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if ((i & 255) == 255) {
            uint64_t now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (begun == 0) begun = now;
            else if (now - begun > 1000000000ull) break;
        }
    }
    return false;
}

// ---------------------------------------------------------------- prepare

constexpr int kPitchA = kChunk + 4;  // floats of a row of A: 16-byte steps that no two of 8 rows share

// The image, then the two products and the row factors; the warps' scratch
// takes the image's place once that has been used.
template <int DK, int LIMBS>
constexpr int prepare_smem() {
    constexpr int scratch = 4 * kChunk * kPitchA * 4, image = Image<DK, LIMBS>::kBytes;
    return (image > scratch ? image : scratch) + (2 * kChunk * (kChunk + 1) + 2 * kChunk) * 4;
}

// 2^(i + f) for |f| <= 1, good to 2^-22 of itself: a decay between two tokens as
// the exact difference of the whole parts of their sums and the rounded one of
// the rest, so that its precision does not depend on its size. From 2^-127 down it
// is zero, from i = 128 up infinite (a second factor would reach further, for 25%
// of the prepare kernel's time).
__device__ __forceinline__ float power(int i, float f) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(f));
    i = min(max(i, -127), 128);
    return y * __int_as_float((i + 127) << 23);
}

// Reduces 16 values of a lane across the warp: v[0] becomes value lane / 2's.
template <typename F>
__device__ __forceinline__ void reduce_rows(float (&v)[16], F op) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 8, o = 16; n > 0; n >>= 1, o >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float keep = lane & o ? v[i + n] : v[i], send = lane & o ? v[i] : v[i + n];
            v[i] = op(keep, __shfl_xor_sync(0xFFFFFFFFu, send, o));
        }
    v[0] = op(v[0], __shfl_xor_sync(0xFFFFFFFFu, v[0], 1));
}

// One block per chunk and key head: limbs of K and Q, K K^T and Q K^T; then,
// for each value head of that key head, one warp for T and one for P.
template <typename T, int DK, int LIMBS>
__global__ void __launch_bounds__(kThreads) delta_prepare_kernel(const DeltaArgs a, const __grid_constant__ SeqTable tab,
                                                                 uint8_t* __restrict__ images,
                                                                 uint8_t* __restrict__ images_t) {
    using I = Image<DK, LIMBS>;
    constexpr int PER = DK / 32;  // elements of a row a lane holds
    extern __shared__ __align__(16) uint8_t smem[];
    float(*kk)[kChunk + 1] =
        reinterpret_cast<float(*)[kChunk + 1]>(smem + prepare_smem<DK, LIMBS>() - (2 * kChunk * (kChunk + 1) + 2 * kChunk) * 4);
    float(*qk)[kChunk + 1] = kk + kChunk;
    float* fk = &qk[kChunk][0];  // what a row of limbs is to be multiplied with
    float* fq = fk + kChunk;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float(*A)[kPitchA] = reinterpret_cast<float(*)[kPitchA]>(smem) + warp * kChunk;
    const int tile = blockIdx.x / a.k_heads, hk = blockIdx.x - tile * a.k_heads;
    const Seq seq = sequence_of_tile(tab, tile);
    const int t0 = (tile - seq.tile0) * kChunk, n = min(kChunk, seq.len - t0);
    const int64_t row = (int64_t)seq.row + t0;

    const int per = a.v_heads / a.k_heads;
    auto value_head = [&](int task) { return a.tiled ? hk + (task >> 1) * a.k_heads : hk * per + (task >> 1); };
    auto gate_of = [&](int h, float& g, float& beta) {
        g = lane < n ? a.gate[(row + lane) * a.gate_stride + h] : 0.0f;
        beta = lane < n ? a.beta[(row + lane) * a.beta_stride + h] : 0.0f;
    };
    float g_first = 0.0f, b_first = 0.0f;  // the warp's first task's, there by the time they are needed
    if (warp < 2 * per) gate_of(value_head(warp), g_first, b_first);

    const T* K = static_cast<const T*>(a.k) + row * a.k_stride + (int64_t)hk * a.k_dim + lane * PER;
    const T* Q = static_cast<const T*>(a.q) + row * a.q_stride + (int64_t)hk * a.k_dim + lane * PER;
    const bool whole = a.k_dim == DK && PER * sizeof(T) >= 4 && a.k_stride % PER == 0 && a.q_stride % PER == 0 &&
                       ((uintptr_t)a.k | (uintptr_t)a.q) % (PER * sizeof(T)) == 0;
    float x[16][PER];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int i = warp * 8 + (r & 7);
        const T* p = r < 8 ? K + i * a.k_stride : Q + i * a.q_stride;
        if (i < n && whole) {
            const Pack<T, PER> in = *reinterpret_cast<const Pack<T, PER>*>(p);
#pragma unroll
            for (int e = 0; e < PER; ++e) x[r][e] = to_f32(in.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e) x[r][e] = i < n && lane * PER + e < a.k_dim ? to_f32(p[e]) : 0.0f;
        }
    }
    {
        float most[16], squares[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            most[r] = squares[r] = 0.0f;
#pragma unroll
            for (int e = 0; e < PER; ++e)
                most[r] = fmaxf(most[r], fabsf(x[r][e])), squares[r] = fmaf(x[r][e], x[r][e], squares[r]);
        }
        // lane 2 r (and the next) ends up with row r's
        reduce_rows(most, [](float a, float b) { return fmaxf(a, b); });
        reduce_rows(squares, [](float a, float b) { return a + b; });
        float up, down;
        power_for(most[0], up, down);
        if (!(lane & 1)) {
            const int r = lane >> 1, i = warp * 8 + (r & 7);
            const float f = a.norm ? 1.0f / sqrtf(squares[0] + a.eps) : 1.0f;
            (r < 8 ? fk : fq)[i] = i < n ? (r < 8 ? down * f : down * f * a.scale) : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = warp * 8 + (r & 7);
            const float scale = __shfl_sync(0xFFFFFFFFu, up, r * 2);
            uint8_t* at = smem + (r < 8 ? 0 : LIMBS * I::kLimb) + i * I::kPitch + lane * PER * 2;
            Pack<__half, PER> hi, lo;
#pragma unroll
            for (int e = 0; e + 1 < PER; e += 2) {
                uint32_t h, l;
                split(x[r][e] * scale, x[r][e + 1] * scale, h, l);
                const __half2 h2 = *reinterpret_cast<const __half2*>(&h), l2 = *reinterpret_cast<const __half2*>(&l);
                hi.v[e] = __low2half(h2), hi.v[e + 1] = __high2half(h2);
                lo.v[e] = __low2half(l2), lo.v[e + 1] = __high2half(l2);
            }
            if (PER & 1) {
                hi.v[PER - 1] = __float2half_rn(x[r][PER - 1] * scale);
                lo.v[PER - 1] = __float2half_rn(x[r][PER - 1] * scale - __half2float(hi.v[PER - 1]));
            }
            *reinterpret_cast<Pack<__half, PER>*>(at) = hi;
            if (LIMBS == 2) *reinterpret_cast<Pack<__half, PER>*>(at + I::kLimb) = lo;
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the copy below reads what was just written
    __syncthreads();
    if (threadIdx.x == 0) {  // the image, as the scan will stage it, on its way out
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                         images + (int64_t)blockIdx.x * I::kBytes),
                     "r"(shared_addr(smem)), "r"(I::kBytes)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    {  // warps 0, 1: K K^T; 2, 3: Q K^T; 16 rows each, up to the diagonal
        const int m0 = (warp & 1) * 16;
        const uint32_t left = shared_addr(smem) + (warp < 2 ? 0 : LIMBS * I::kLimb) + (m0 + (lane & 15)) * I::kPitch +
                              (lane >> 4) * 16;
        const uint32_t right = shared_addr(smem) + ((lane & 7) + ((lane >> 4) << 3)) * I::kPitch + ((lane >> 3) & 1) * 16;
        float c[4][4] = {}, s[4][4] = {};
#pragma unroll
        for (int ks = 0; ks < DK / 16; ++ks) {
            uint32_t ah[4], al[4];
            ldmatrix(ah, left + ks * 32);
            if (LIMBS == 2) ldmatrix(al, left + I::kLimb + ks * 32);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                if (p * 16 > m0) break;
                uint32_t bh[4], bl[4];
                ldmatrix(bh, right + p * 16 * I::kPitch + ks * 32);
                mma(c[2 * p], ah, bh[0], bh[1]);
                mma(c[2 * p + 1], ah, bh[2], bh[3]);
                if (LIMBS == 2) {
                    ldmatrix(bl, right + I::kLimb + p * 16 * I::kPitch + ks * 32);
                    mma(s[2 * p], ah, bl[0], bl[1]);
                    mma(s[2 * p + 1], ah, bl[2], bl[3]);
                    mma(s[2 * p], al, bh[0], bh[1]);
                    mma(s[2 * p + 1], al, bh[2], bh[3]);
                }
            }
        }
        float(*out)[kChunk + 1] = warp < 2 ? kk : qk;
        const float* f = warp < 2 ? fk : fq;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = m0 + (lane >> 2) + (r >> 1) * 8, j = t * 8 + (lane & 3) * 2 + (r & 1);
                out[i][j] = (c[t][r] + s[t][r]) * f[i] * fk[j];
            }
    }
    // the image is out of shared memory before the scratch takes its place
    if (threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncthreads();
    for (int task = warp; task < 2 * per; task += kThreads / 32) {
        const int h = value_head(task);
        float g = g_first, beta = b_first;
        if (task != warp) gate_of(h, g, beta);
        if (lane < n) {
            gates(a, h, g, beta);
            // e^-10000 is zero and e^10000 infinite; a sum of these stays a number, so that differences do
            if (g < -1e4f) g = -1e4f;
            if (g > 1e4f) g = 1e4f;
        }
        double G = (double)g * 1.4426950408889634;  // in powers of two
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xFFFFFFFFu, G, o);
            if (lane >= o) G += up;
        }
        uint8_t* image = images_t + ((int64_t)tile * a.v_heads + h) * kImageT;
        float* out = reinterpret_cast<float*>(image + kGates) + lane;
        float v[kChunk];  // a row a lane: beta_i e^{G_i - G_j} k_i . k_j, or e^{G_i - G_j} q_i . k_j
        const float(*products)[kChunk + 1] = task & 1 ? qk : kk;
        const int diagonal = task & 1 ? lane : lane - 1;  // the row's last column
        const int Gi = __double2int_rn(G);  // whole (at most 32 * 1e4 log2 e; a NaN is the rest's) and rest
        const float Gf = (float)(G - (double)Gi);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            const int i = __shfl_sync(0xFFFFFFFFu, Gi, j);
            const float f = __shfl_sync(0xFFFFFFFFu, Gf, j);
            v[j] = j <= diagonal ? power(Gi - i, Gf - f) * products[lane][j] : 0.0f;
        }
        if (task & 1) {
            float4* row = reinterpret_cast<float4*>(image + kMatT) + lane * (kPitchT / 4);
#pragma unroll
            for (int j = 0; j < kChunk; j += 4) row[j / 4] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            const int end_i = __shfl_sync(0xFFFFFFFFu, Gi, 31);
            const float end_f = __shfl_sync(0xFFFFFFFFu, Gf, 31);
            const float before = power(Gi, Gf), after = power(end_i - Gi, end_f - Gf);
            if (lane == 0) out[kTotal * kChunk] = power(end_i, end_f);
            out[kBeta * kChunk] = beta;
            out[kXk * kChunk] = beta * before * fk[lane];
            out[kOq * kChunk] = before * fq[lane];
            out[kDown * kChunk] = after * fk[lane];
            continue;
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kChunk; j += 4)
            *reinterpret_cast<float4*>(&A[lane][j]) =
                make_float4(-beta * v[j], -beta * v[j + 1], -beta * v[j + 2], -beta * v[j + 3]);
        __syncwarp();
        // T = (I + A)^-1, a column a lane, row by row (A holds its negative)
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            float acc[2] = {lane == i ? 1.0f : 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j + 4 <= i; j += 4) {
                const float4 w = *reinterpret_cast<const float4*>(&A[i][j]);
                acc[0] = fmaf(w.x, v[j], acc[0]), acc[1] = fmaf(w.y, v[j + 1], acc[1]);
                acc[0] = fmaf(w.z, v[j + 2], acc[0]), acc[1] = fmaf(w.w, v[j + 3], acc[1]);
            }
#pragma unroll
            for (int j = i & ~3; j < i; ++j) acc[j & 1] = fmaf(A[i][j], v[j], acc[j & 1]);
            v[i] = acc[0] + acc[1];
        }
#pragma unroll
        for (int i = 0; i < kChunk; ++i) reinterpret_cast<float*>(image)[i * kPitchT + lane] = v[i];
    }
}

// ------------------------------------------------------------------- scan

// A scan block: GROUPS groups of 16 columns of S, each with kParts warps for S
// and two for the outputs.
constexpr int kStages = 3;  // the chunk being read, the next, and the one whose outputs are still to come
constexpr int kMaxShared = 227 * 1024;
template <int DK, int GROUPS>
struct Split {
    static constexpr int kParts = 2, kCols = GROUPS * 16;
    static constexpr int kHolders = GROUPS * kParts * 32, kThreads = kHolders + GROUPS * 64;
    static constexpr int kRows = DK / kParts;    // rows of S a warp holds
};

// What a group's warps hand on to its outputs' (two, for even and odd chunks):
// S's limbs and their row factors, and U. Limbs lie as left operands take them:
// two rows of hi, two of lo. Tiles of U, X and S^T K^T lie as accumulators do.
template <int DK>
struct Handoff {
    uint4 hi[DK / 16][32], lo[DK / 16][32];
    float2 down[2][32];
    float4 u[4][32];
};
// And among each other, within a chunk: parts of S^T K^T, X, and the limbs of U
// scaled to the chunk's end with what undoes their scale.
struct Shared {
    float4 y[2][4][32], x[4][32];
    uint4 e[4][32];
    float2 e_down[2][32];
};

// Of the four tiles of 8 tokens of a chunk, those (k = 0, 1) that the warp `part`
// of a pair takes: together as long as the other's in a triangular product.
__device__ __forceinline__ int tile_of(int part, int k) { return k ? 3 - part : part; }

template <int DK, int LIMBS, int GROUPS>
constexpr int scan_smem() {
    return kStages * (Image<DK, LIMBS>::kBytes + kImageT) + 2 * GROUPS * (int)sizeof(Handoff<DK>) +
           GROUPS * (int)sizeof(Shared);
}

// Named barriers of a group: `threads` of them arrive in all.
__device__ __forceinline__ void group_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void group_arrive(int id, int threads) {
    asm volatile("bar.arrive %0, %1;\n" ::"r"(id), "r"(threads) : "memory");
}

// Powers for two rows of the warp's tile from a lane's largest magnitudes of each:
// rows lie across 4 lanes. The exponents of both go through one exchange.
__device__ __forceinline__ void row_powers(float m0, float m1, float (&up)[2], float (&down)[2]) {
    uint32_t e = __byte_perm(__float_as_uint(m0) << 1, __float_as_uint(m1) << 1, 0x7733) & 0x00FF00FFu;
    e = __vmaxu2(e, __shfl_xor_sync(0xFFFFFFFFu, e, 1));
    e = __vmaxu2(e, __shfl_xor_sync(0xFFFFFFFFu, e, 2));
    power_of(e & 255u, up[0], down[0]);
    power_of(e >> 16, up[1], down[1]);
}

// Tiles x (16 rows by 8 N columns) as limbs of a left operand, scaled by row;
// down: what undoes the scale, for the two rows of a lane.
template <int N>
__device__ __forceinline__ void limbs(const float (&x)[N][4], uint32_t (&hi)[N / 2][4], uint32_t (&lo)[N / 2][4],
                                      float (&down)[2]) {
    float m0 = 0.0f, m1 = 0.0f, up[2];
#pragma unroll
    for (int t = 0; t < N; ++t) {
        m0 = fmaxf(m0, fmaxf(fabsf(x[t][0]), fabsf(x[t][1])));
        m1 = fmaxf(m1, fmaxf(fabsf(x[t][2]), fabsf(x[t][3])));
    }
    row_powers(m0, m1, up, down);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
        split(x[2 * k][0] * up[0], x[2 * k][1] * up[0], hi[k][0], lo[k][0]);
        split(x[2 * k][2] * up[1], x[2 * k][3] * up[1], hi[k][1], lo[k][1]);
        split(x[2 * k + 1][0] * up[0], x[2 * k + 1][1] * up[0], hi[k][2], lo[k][2]);
        split(x[2 * k + 1][2] * up[1], x[2 * k + 1][3] * up[1], hi[k][3], lo[k][3]);
    }
}

// A tile's four values of a lane (two of a row, two of the row 8 on) as limbs.
__device__ __forceinline__ uint4 tile_limbs(float a, float b, float c, float d, float up0, float up1) {
    uint4 w;
    split(a * up0, b * up0, w.x, w.z);
    split(c * up1, d * up1, w.y, w.w);
    return w;
}
// Two tiles' limbs as a left operand.
__device__ __forceinline__ void operand(const uint4& a, const uint4& b, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    hi[0] = a.x, hi[1] = a.y, hi[2] = b.x, hi[3] = b.y;
    lo[0] = a.z, lo[1] = a.w, lo[2] = b.z, lo[3] = b.w;
}

// The tiles of X^T M^T of the warp PART of a pair, M lower triangular. A lane holds
// tokens 2 c and 2 c + 1 of a tile of X where a product's left operand has its
// terms c and c + 4: the right one is read in the same order.
template <int PART>
__device__ __forceinline__ void triangular(const float* M, const float4 (&X)[4][32], float (&acc)[2][4]) {
    const int lane = threadIdx.x & 31;
    const float* m = M + (lane >> 2) * kPitchT + (lane & 3) * 2;
    float hl[2][4] = {}, lh[2][4] = {};  // apart: a product waits for the last one into its sum
#pragma unroll
    for (int t = 0; t <= 3 - PART; ++t) {
        const float4 x = X[t][lane];
        uint32_t ah[4], al[4];
        split_tf32(x.x, ah[0], al[0]), split_tf32(x.z, ah[1], al[1]);
        split_tf32(x.y, ah[2], al[2]), split_tf32(x.w, ah[3], al[3]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int out = k ? 3 - PART : PART;
            if (t > out) continue;  // later tokens' columns of M are zero
            const float2 w = *reinterpret_cast<const float2*>(m + out * 8 * kPitchT + t * 8);
            uint32_t bh[2], bl[2];
            split_tf32(w.x, bh[0], bl[0]), split_tf32(w.y, bh[1], bl[1]);
            mma_tf32(hl[k], ah, bl);
            mma_tf32(lh[k], al, bh);
            mma_tf32(acc[k], ah, bh);
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[k][r] += hl[k][r] + lh[k][r];
}
__device__ __forceinline__ void triangular(int part, const float* M, const float4 (&X)[4][32], float (&acc)[2][4]) {
    if (part == 0) triangular<0>(M, X, acc);
    else triangular<1>(M, X, acc);
}

template <typename T, int DK, int LIMBS, int GROUPS>
__global__ void __launch_bounds__((Split<DK, GROUPS>::kThreads), 1)
    delta_scan_kernel(const DeltaArgs a, const __grid_constant__ SeqTable tab, const uint8_t* __restrict__ images,
                      const uint8_t* __restrict__ images_t, int* err) {
    using I = Image<DK, LIMBS>;
    using L = Split<DK, GROUPS>;
    constexpr int PARTS = L::kParts, ROWS = L::kRows, NT = ROWS / 8, KS = ROWS / 16;
    constexpr int kStage = I::kBytes + kImageT;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(8) uint64_t arrived[kStages], ready[GROUPS][2][2];  // ready: S's limbs, U; even and odd chunks
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the warps of S first, then those of the outputs, spread evenly over the schedulers
    const bool holds = threadIdx.x < L::kHolders;
    const int group = holds ? warp / PARTS : (warp - GROUPS * PARTS) / 2;
    const int part = holds ? warp % PARTS : (warp - GROUPS * PARTS) % 2;
    Handoff<DK>* const hands = reinterpret_cast<Handoff<DK>*>(smem + kStages * kStage) + group * 2;
    Shared& sh = reinterpret_cast<Shared*>(smem + kStages * kStage + 2 * GROUPS * sizeof(Handoff<DK>))[group];
    // Named barriers: chunk written out (even, odd), and among a group's warps of
    // S. Those only arrive at `ready` and may be a chunk ahead of the outputs
    // there, so that even and odd chunks have their own: one is used again two
    // chunks on, behind the outputs' arrival at bar_done for its last chunk.
    const int bar_done = 1, bar_g = 3 + group;
    int b = blockIdx.x;
    const int cb = b % a.col_blocks;
    b /= a.col_blocks;
    const int h = b % a.v_heads;
    const Seq seq = sequence_at(tab, b / a.v_heads);
    const int hk = key_head(a, h);
    const int chunks = (seq.len + kChunk - 1) / kChunk;
    const int j0 = cb * L::kCols + group * 16 + (lane >> 2), j1 = j0 + 8;  // the lane's two columns of S
    const bool in0 = j0 < a.v_dim, in1 = j1 < a.v_dim;
    const int tc = (lane & 3) * 2;
    const int d0 = part * ROWS + tc;  // its first row of S (warps of S)

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_addr(&arrived[i])) : "memory");
        for (int i = 0; i < GROUPS * 4; ++i)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_addr(&ready[i / 4][i / 2 % 2][i % 2])),
                         "n"(PARTS)
                         : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    auto stage = [&](int c) {  // by one thread
        const int64_t tile = seq.tile0 + c;
        const uint32_t dst = shared_addr(smem + (c % kStages) * kStage), bar = shared_addr(&arrived[c % kStages]);
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(kStage) : "memory");
        bulk_copy(dst, images + (tile * a.k_heads + hk) * I::kBytes, I::kBytes, bar);
        bulk_copy(dst + I::kBytes, images_t + (tile * a.v_heads + h) * kImageT, kImageT, bar);
    };
    if (threadIdx.x == 0) stage(0);
    // Waits for a phase. Where it does not come (a second is long past), the
    // thread goes on without waiting, so that no other is left behind at a
    // barrier, and the call is reported as timed out.
    bool there = true;
    auto wait = [&](const uint64_t* bar, int parity) {
        if (!there) return;
        there = bulk_wait(shared_addr(bar), parity);
        if (!there) {
            bulk_wait(shared_addr(bar), parity);  // no copy in flight when the block ends
            atomicExch(err, 1);
        }
    };
    auto wait_chunk = [&](int c) { wait(&arrived[c % kStages], (c / kStages) & 1); };
    auto wait_ready = [&](int what, int c) { wait(&ready[group][what][c & 1], (c >> 1) & 1); };
    auto set_ready = [&](int what, int c) {  // by every warp of S
        __syncwarp();
        if (lane == 0)
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_addr(&ready[group][what][c & 1])) : "memory");
    };
    const uint32_t lane_b = ((lane & 7) + ((lane >> 4) << 3));  // row of a right operand's pair of tiles
    const uint32_t half_b = ((lane >> 3) & 1) * 16;             // and its half of a row

    if (!holds) {  // ---- outputs of the tokens of two tiles
        T* O = static_cast<T*>(a.o) + (int64_t)seq.row * a.o_stride + (int64_t)h * a.v_dim;
        for (int c = 0; c < chunks; ++c) {
            wait_chunk(c);
            const uint8_t* image = smem + (c % kStages) * kStage;
            const Handoff<DK>& hand = hands[c & 1];
            const float* gate = reinterpret_cast<const float*>(image + I::kBytes + kGates);
            const uint32_t q_at = shared_addr(image) + LIMBS * I::kLimb +
                                  (tile_of(part, lane >> 4) * 8 + (lane & 7)) * I::kPitch + half_b;
            float out[2][4] = {};
            wait_ready(0, c);
#pragma unroll
            for (int k = 0; k < PARTS; ++k) {  // the parts of k_dim, each with its own row factors
                float o1[2][4] = {};
                uint32_t hi[KS][4];
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint4 h4 = hand.hi[k * KS + ks][lane], l4 = hand.lo[k * KS + ks][lane];
                    const uint32_t lo[4] = {l4.x, l4.y, l4.z, l4.w};
                    hi[ks][0] = h4.x, hi[ks][1] = h4.y, hi[ks][2] = h4.z, hi[ks][3] = h4.w;
                    uint32_t bq[4];
                    if (LIMBS == 2) {
                        ldmatrix(bq, q_at + I::kLimb + (k * KS + ks) * 32);
                        mma(o1[0], hi[ks], bq[0], bq[1]);
                        mma(o1[1], hi[ks], bq[2], bq[3]);
                    }
                    ldmatrix(bq, q_at + (k * KS + ks) * 32);
                    mma(o1[0], lo, bq[0], bq[1]);
                    mma(o1[1], lo, bq[2], bq[3]);
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t bq[4];
                    ldmatrix(bq, q_at + (k * KS + ks) * 32);
                    mma(o1[0], hi[ks], bq[0], bq[1]);
                    mma(o1[1], hi[ks], bq[2], bq[3]);
                }
                const float2 down = hand.down[k][lane];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) out[t][r] = fmaf(o1[t][r], r < 2 ? down.x : down.y, out[t][r]);
            }
            wait_ready(1, c);
            float y[2][4] = {};
            triangular(part, reinterpret_cast<const float*>(image + I::kBytes + kMatT), hand.u, y);
            T* row = O + (int64_t)(c * kChunk + tc) * a.o_stride;
            const int left = seq.len - (c * kChunk + tc);  // tokens from the lane's first
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int t = tile_of(part, k) * 8;
                const float2 oq = *reinterpret_cast<const float2*>(gate + kOq * kChunk + t + tc);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float res = fmaf(r & 1 ? oq.y : oq.x, out[k][r], y[k][r]);
                    if (t + (r & 1) < left && (r < 2 ? in0 : in1))
                        from_f32(row[(t + (r & 1)) * a.o_stride + (r < 2 ? j0 : j1)], res);
                }
            }
            // the stage and the handoff may be written again (two chunks on)
            if (c + 2 < chunks) group_arrive(bar_done + (c & 1), L::kThreads);
        }
        return;
    }

    // ---- the state
    float* S = a.state + ((int64_t)seq.slot * a.v_heads + h) * a.k_dim * a.v_dim;
    float s[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = d0 + t * 8 + (r & 1), j = r < 2 ? j0 : j1;
            s[t][r] = d < a.k_dim && j < a.v_dim ? S[(int64_t)d * a.v_dim + j] : 0.0f;
        }
    const T* V = static_cast<const T*>(a.v) + (int64_t)seq.row * a.v_stride + (int64_t)h * a.v_dim;
    V += (int64_t)tc * a.v_stride;
    T coming[2][4];  // the next chunk's values, not touched before it begins
    auto fetch = [&](int c) {
        const T* row = V + (int64_t)c * kChunk * a.v_stride;
        const int left = seq.len - c * kChunk - tc;  // tokens from the lane's first
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = tile_of(part, k) * 8 + (r & 1);
                const bool in = t < left && (r < 2 ? in0 : in1);
                from_f32(coming[k][r], 0.0f);
                if (in) coming[k][r] = row[t * a.v_stride + (r < 2 ? j0 : j1)];
            }
    };
    fetch(0);
    for (int c = 0; c < chunks; ++c) {
        // chunk c - 2 is written out, so its stage can take chunk c + 1 and its handoff this chunk's
        if (c >= 2) group_sync(bar_done + (c & 1), L::kThreads);
        if (threadIdx.x == 0 && c + 1 < chunks && there) stage(c + 1);
        wait_chunk(c);
        Handoff<DK>& hand = hands[c & 1];
        const uint8_t* image = smem + (c % kStages) * kStage;
        const uint32_t base = shared_addr(image);
        const float* gate = reinterpret_cast<const float*>(image + I::kBytes + kGates);
        float v[2][4];
        {  // this warp's part of S^T K^T
            uint32_t hi[KS][4], lo[KS][4];
            float down[2], y[4][4] = {};
            limbs<NT>(s, hi, lo, down);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) v[k][r] = to_f32(coming[k][r]);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                hand.hi[part * KS + ks][lane] = make_uint4(hi[ks][0], hi[ks][1], hi[ks][2], hi[ks][3]);
                hand.lo[part * KS + ks][lane] = make_uint4(lo[ks][0], lo[ks][1], lo[ks][2], lo[ks][3]);
            }
            hand.down[part][lane] = make_float2(down[0], down[1]);
            const uint32_t at = base + lane_b * I::kPitch + part * ROWS * 2 + half_b;
            uint32_t bk[KS][2][4];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint32_t k_at = at + p * 16 * I::kPitch + ks * 32;
                    ldmatrix(bk[ks][p], k_at);
                    mma(y[2 * p], lo[ks], bk[ks][p][0], bk[ks][p][1]);
                    mma(y[2 * p + 1], lo[ks], bk[ks][p][2], bk[ks][p][3]);
                    if (LIMBS == 2) {
                        uint32_t bl[4];
                        ldmatrix(bl, k_at + I::kLimb);
                        mma(y[2 * p], hi[ks], bl[0], bl[1]);
                        mma(y[2 * p + 1], hi[ks], bl[2], bl[3]);
                    }
                }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    mma(y[2 * p], hi[ks], bk[ks][p][0], bk[ks][p][1]);
                    mma(y[2 * p + 1], hi[ks], bk[ks][p][2], bk[ks][p][3]);
                }
#pragma unroll
            for (int t = 0; t < 4; ++t)
                sh.y[part][t][lane] =
                    make_float4(y[t][0] * down[0], y[t][1] * down[0], y[t][2] * down[1], y[t][3] * down[1]);
        }
        // S's limbs are handed on only now: the outputs' products take the tensor
        // cores while this chain exchanges and scales, not before
        set_ready(0, c);
        group_sync(bar_g, PARTS * 32);
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // X of this warp's tokens
            const int t = tile_of(part, k);
            const float2 beta = *reinterpret_cast<const float2*>(gate + kBeta * kChunk + t * 8 + tc);
            const float2 xk = *reinterpret_cast<const float2*>(gate + kXk * kChunk + t * 8 + tc);
            float4 y = sh.y[0][t][lane];
#pragma unroll
            for (int q = 1; q < PARTS; ++q) {
                const float4 w = sh.y[q][t][lane];
                y.x += w.x, y.y += w.y, y.z += w.z, y.w += w.w;
            }
            sh.x[t][lane] = make_float4(beta.x * v[k][0] - xk.x * y.x, beta.y * v[k][1] - xk.y * y.y,
                                        beta.x * v[k][2] - xk.x * y.z, beta.y * v[k][3] - xk.y * y.w);
        }
        group_sync(bar_g, PARTS * 32);
        if (c + 1 < chunks) fetch(c + 1);

        {  // U = T X, this warp's tokens, and its limbs scaled to the chunk's end
            float u[2][4] = {}, m0 = 0.0f, m1 = 0.0f, up[2], down[2];
            triangular(part, reinterpret_cast<const float*>(image + I::kBytes), sh.x, u);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int t = tile_of(part, k);
                hand.u[t][lane] = make_float4(u[k][0], u[k][1], u[k][2], u[k][3]);
                const float2 e = *reinterpret_cast<const float2*>(gate + kDown * kChunk + t * 8 + tc);
                u[k][0] *= e.x, u[k][1] *= e.y, u[k][2] *= e.x, u[k][3] *= e.y;
                m0 = fmaxf(m0, fmaxf(fabsf(u[k][0]), fabsf(u[k][1])));
                m1 = fmaxf(m1, fmaxf(fabsf(u[k][2]), fabsf(u[k][3])));
            }
            row_powers(m0, m1, up, down);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                sh.e[tile_of(part, k)][lane] = tile_limbs(u[k][0], u[k][1], u[k][2], u[k][3], up[0], up[1]);
            sh.e_down[part][lane] = make_float2(down[0], down[1]);
        }
        set_ready(1, c);
        group_sync(bar_g, PARTS * 32);
        // S <- e^{G_C} S + U^T K, with U scaled to the chunk's end; each warp's tokens have their own scale
        {
            uint32_t hi[2][4], lo[2][4], at[2];
            float2 down[2];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                operand(sh.e[tile_of(ks, 0)][lane], sh.e[tile_of(ks, 1)][lane], hi[ks], lo[ks]);
                down[ks] = sh.e_down[ks][lane];
                at[ks] = base + (tile_of(ks, lane >> 3 & 1) * 8 + (lane & 7)) * I::kPitch + part * ROWS * 2 + (lane >> 4) * 16;
            }
            const float total = gate[kTotal * kChunk];
#pragma unroll
            for (int p = 0; p < NT / 2; ++p) {
                float c1[2][2][4] = {};
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    uint32_t bh[4], bl[4];
                    ldmatrix_trans(bh, at[ks] + p * 32);
                    mma(c1[ks][0], lo[ks], bh[0], bh[1]);
                    mma(c1[ks][1], lo[ks], bh[2], bh[3]);
                    if (LIMBS == 2) {
                        ldmatrix_trans(bl, at[ks] + I::kLimb + p * 32);
                        mma(c1[ks][0], hi[ks], bl[0], bl[1]);
                        mma(c1[ks][1], hi[ks], bl[2], bl[3]);
                    }
                    mma(c1[ks][0], hi[ks], bh[0], bh[1]);
                    mma(c1[ks][1], hi[ks], bh[2], bh[3]);
                }
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float first = fmaf(total, s[2 * p + t][r], c1[0][t][r] * (r < 2 ? down[0].x : down[0].y));
                        s[2 * p + t][r] = fmaf(c1[1][t][r], r < 2 ? down[1].x : down[1].y, first);
                    }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = d0 + t * 8 + (r & 1), j = r < 2 ? j0 : j1;
            if (d < a.k_dim && j < a.v_dim) S[(int64_t)d * a.v_dim + j] = s[t][r];
        }
}

// ------------------------------------------------------------------- host

int padded_dim(int64_t k_dim) { return k_dim <= 32 ? 32 : k_dim <= 64 ? 64 : k_dim <= 96 ? 96 : 128; }

// Bytes of the images of one chunk over all heads.
struct ChunkBytes {
    uint64_t keys, rest;
    uint64_t all() const { return keys + rest; }
};
ChunkBytes chunk_bytes(const strata_gated_delta& d) {
    const uint64_t limbs = d.dtype == STRATA_QUANT_BF16 ? 1 : 2;
    return ChunkBytes{2 * limbs * kChunk * (uint64_t)(padded_dim(d.k_dim) * 2 + 16) * (uint64_t)d.n_k_head,
                      (uint64_t)kImageT * (uint64_t)d.n_v_head};
}

// The launches of a call: groups of sequences, each read in pieces of as many
// chunks as the workspace bound allows (one per sequence at least). Calls
// launch(table, tiles) in order. Sequences below `from` tokens are left out.
template <typename F>
int plan_chunks(const strata_gated_delta& d, int64_t from, F launch) {
    const uint64_t fit = kMaxWork / chunk_bytes(d).all();
    const int64_t cap = fit < 1 ? 1 : (int64_t)fit;
    auto per_sequence = [&](int64_t n) { return cap / n > 1 ? cap / n : int64_t(1); };
    if (!d.seq_offsets) {
        const int64_t group = d.n_seq < cap ? d.n_seq : cap;
        for (int64_t i = 0; i < d.n_seq; i += group) {
            const int64_t n = d.n_seq - i < group ? d.n_seq - i : group, step = per_sequence(n) * kChunk;
            for (int64_t t = 0; t < d.seq_len; t += step) {
                const int64_t len = d.seq_len - t < step ? d.seq_len - t : step;
                const SeqTable tab = uniform_table(n, i * d.seq_len + t, d.seq_len, i, len, kChunk);
                const int rc = launch(tab, n * tab.tiles_all);
                if (rc) return rc;
            }
        }
        return STRATA_OK;
    }
    const int64_t group = cap < kSeqGroup ? cap : kSeqGroup;
    auto length = [&](int64_t i) {
        const int64_t len = d.seq_offsets[i + 1] - d.seq_offsets[i];
        return len < from ? int64_t(0) : len;
    };
    for (int64_t i = 0; i < d.n_seq;) {
        int64_t end = i, live = 0;  // sequences [i, end), `live` of them with tokens
        while (end < d.n_seq && live < group) live += length(end) > 0, ++end;
        for (int64_t t = 0; live > 0;) {
            // the longest piece (in chunks, of every sequence that still has tokens) that fits
            int64_t fits = 1, over = cap + 1;
            while (over - fits > 1) {
                const int64_t mid = (fits + over) / 2;
                int64_t sum = 0;
                for (int64_t k = i; k < end; ++k) {
                    const int64_t left = (length(k) - t + kChunk - 1) / kChunk;
                    sum += left <= 0 ? 0 : left < mid ? left : mid;
                }
                if (sum <= cap) fits = mid;
                else over = mid;
            }
            const int64_t step = fits * kChunk;
            // the longest first, so that no long one is left to start last
            int64_t order[kSeqGroup], count = 0, left = 0;
            for (int64_t k = i; k < end; ++k)
                if (length(k) > t) order[count++] = k;
            std::stable_sort(order, order + count, [&](int64_t x, int64_t y) { return length(x) > length(y); });
            SeqTable tab = ragged_table();
            for (int64_t n = 0; n < count; ++n) {
                const int64_t k = order[n], len = length(k) - t;
                add_sequence(tab, k, d.seq_offsets[k] + t, len < step ? len : step, kChunk);
                left += len > step;
            }
            const int rc = launch(tab, (int64_t)tab.tile[tab.n]);
            if (rc) return rc;
            t += step;
            live = left;
        }
        i = end;
    }
    return STRATA_OK;
}

template <typename T, int DK, int LIMBS, int GROUPS>
int enqueue_scan(strata_ctx* ctx, DeltaArgs a, const SeqTable& t, const uint8_t* images, const uint8_t* images_t,
                 cudaStream_t s) {
    using L = Split<DK, GROUPS>;
    auto scan = delta_scan_kernel<T, DK, LIMBS, GROUPS>;
    constexpr int smem = scan_smem<DK, LIMBS, GROUPS>();
    static_assert(smem <= kMaxShared - 1024, "a block's shared memory");
    static std::atomic<uint64_t> asked;
    const cudaError_t e = allow_shared(scan, smem, asked, ctx->device);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cudaFuncSetAttribute(gated_delta)");
    a.col_blocks = (a.v_dim + L::kCols - 1) / L::kCols;
    const int64_t grid = (int64_t)t.n * a.v_heads * a.col_blocks;
    if (grid > kMaxTokens) return fail(ctx, STRATA_ERR_INVALID, "gated_delta: %d sequences of %d heads", t.n, a.v_heads);
    scan<<<(unsigned)grid, L::kThreads, smem, s>>>(a, t, images, images_t, ctx->err_dev);
    return check_launch(ctx, "gated_delta scan kernel");
}

template <typename T, int DK, int LIMBS>
int enqueue(strata_ctx* ctx, const strata_gated_delta& d, const DeltaArgs& a, uint8_t* work, int64_t from,
            cudaStream_t s) {
    auto prepare = delta_prepare_kernel<T, DK, LIMBS>;
    constexpr int smem = prepare_smem<DK, LIMBS>();
    static std::atomic<uint64_t> asked;
    const cudaError_t e = allow_shared(prepare, smem, asked, ctx->device);
    if (e != cudaSuccess) return cuda_fail(ctx, e, "cudaFuncSetAttribute(gated_delta)");
    const uint64_t keys = chunk_bytes(d).keys;
    return plan_chunks(d, from, [&](const SeqTable& t, int64_t tiles) {
        const int64_t grid = tiles * a.k_heads;
        if (grid > kMaxTokens)
            return fail(ctx, STRATA_ERR_INVALID, "gated_delta: %lld chunks of %d heads", (long long)tiles, a.k_heads);
        uint8_t* images_t = work + keys * (uint64_t)tiles;
        prepare<<<(unsigned)grid, kThreads, smem, s>>>(a, t, work, images_t);
        const int rc = check_launch(ctx, "gated_delta prepare kernel");
        if (rc) return rc;
        // blocks of two groups while they all run side by side (the shortest
        // chain), of four where there are more and four fit
        if constexpr (scan_smem<DK, LIMBS, 4>() <= kMaxShared - 1024) {
            if ((int64_t)t.n * a.v_heads * ((a.v_dim + 31) / 32) > ctx->sm_count && a.v_dim > 32)
                return enqueue_scan<T, DK, LIMBS, 4>(ctx, a, t, work, images_t, s);
        }
        return enqueue_scan<T, DK, LIMBS, 2>(ctx, a, t, work, images_t, s);
    });
}

template <typename T, int LIMBS>
int enqueue_dim(strata_ctx* ctx, const strata_gated_delta& d, const DeltaArgs& a, uint8_t* work, int64_t from,
                cudaStream_t s) {
    switch (padded_dim(d.k_dim)) {
        case 32: return enqueue<T, 32, LIMBS>(ctx, d, a, work, from, s);
        case 64: return enqueue<T, 64, LIMBS>(ctx, d, a, work, from, s);
        case 96: return enqueue<T, 96, LIMBS>(ctx, d, a, work, from, s);
        default: return enqueue<T, 128, LIMBS>(ctx, d, a, work, from, s);
    }
}

}  // namespace

uint64_t delta_chunk_work(const strata_gated_delta& d, int64_t from) {
    int64_t most = 0;
    plan_chunks(d, from, [&](const SeqTable&, int64_t tiles) {
        if (tiles > most) most = tiles;
        return (int)STRATA_OK;
    });
    return (uint64_t)most * chunk_bytes(d).all();
}

int delta_chunk_enqueue(strata_ctx* ctx, const strata_gated_delta& d, const DeltaArgs& a, void* work, int64_t from,
                        cudaStream_t s) {
    uint8_t* w = static_cast<uint8_t*>(work);
    if (d.dtype == STRATA_QUANT_BF16) return enqueue_dim<__nv_bfloat16, 1>(ctx, d, a, w, from, s);
    return enqueue_dim<float, 2>(ctx, d, a, w, from, s);
}

}  // namespace strata
