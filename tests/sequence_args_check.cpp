// The argument checks of the sequence operators (csrc/sequence_args.h) run on
// the host: what is refused, with which status, and that packed strides are
// filled in. Buffers are addresses only; nothing is dereferenced.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <limits>

#include "sequence_args.h"

using namespace strata;

static int failures = 0;
#define EXPECT(cond)                                          \
    do {                                                      \
        if (!(cond)) {                                        \
            std::printf("line %d: %s\n", __LINE__, #cond);    \
            ++failures;                                       \
        }                                                     \
    } while (0)

template <typename T = void>
static T* at(uintptr_t a) {
    return reinterpret_cast<T*>(a);
}

static strata_short_conv conv() {
    strata_short_conv d = {};
    d.n_seq = 2, d.seq_len = 5, d.channels = 64, d.taps = 4;
    return d;
}
static strata_gated_delta delta() {
    strata_gated_delta d = {};
    d.n_seq = 2, d.seq_len = 3, d.n_k_head = 2, d.n_v_head = 4, d.k_dim = 16, d.v_dim = 8, d.scale = 0.25, d.l2_eps = -1;
    return d;
}

template <typename F>
static int conv_with(F change) {
    strata_short_conv d = conv();
    change(d);
    Why why;
    int64_t tokens, longest;
    return check_short_conv(why, d, &tokens, &longest);
}
template <typename F>
static int delta_with(F change) {
    strata_gated_delta d = delta();
    change(d);
    Why why;
    int64_t tokens, longest;
    return check_gated_delta(why, d, &tokens, &longest);
}

static void sequences() {
    Why why;
    int64_t tokens = -1, longest = -1;
    const int64_t good[] = {3, 3, 10, 12}, falling[] = {0, 5, 4, 9}, negative[] = {-1, 5, 6, 9},
                  big[] = {0, 1, 2, int64_t(1) << 31}, empty[] = {7, 7, 7, 7};
    EXPECT(check_sequences(why, 3, 0, good, &tokens, &longest) == STRATA_OK && tokens == 12 && longest == 7);
    EXPECT(check_sequences(why, 3, 0, empty, &tokens, &longest) == STRATA_OK && tokens == 7 && longest == 0);
    EXPECT(check_sequences(why, 3, 0, falling, &tokens, &longest) == STRATA_ERR_INVALID);
    EXPECT(check_sequences(why, 3, 0, negative, &tokens, &longest) == STRATA_ERR_INVALID);
    EXPECT(check_sequences(why, 3, 0, big, &tokens, &longest) == STRATA_ERR_INVALID);
    EXPECT(check_sequences(why, 4, 9, nullptr, &tokens, &longest) == STRATA_OK && tokens == 36 && longest == 9);
    EXPECT(check_sequences(why, 4, 0, nullptr, &tokens, &longest) == STRATA_OK && tokens == 0);
    EXPECT(check_sequences(why, 0, 9, nullptr, &tokens, &longest) == STRATA_ERR_INVALID);
    EXPECT(check_sequences(why, -1, 9, nullptr, &tokens, &longest) == STRATA_ERR_INVALID);
    EXPECT(check_sequences(why, 4, -1, nullptr, &tokens, &longest) == STRATA_ERR_INVALID);
    EXPECT(check_sequences(why, 1 << 16, 1 << 15, nullptr, &tokens, &longest) == STRATA_ERR_INVALID);
    EXPECT(check_sequences(why, INT64_MAX, INT64_MAX, nullptr, &tokens, &longest) == STRATA_ERR_INVALID);
}

static void overlaps() {
    const Rows a{"a", at(1000), 64, 64, 10};  // 1000 .. 1640
    EXPECT(overlap(a, Rows{"b", at(1639), 4, 4, 1}));
    EXPECT(!overlap(a, Rows{"b", at(1640), 4, 4, 1}));
    EXPECT(!overlap(a, Rows{"b", at(996), 4, 4, 1}));
    EXPECT(overlap(a, Rows{"b", at(996), 5, 5, 1}));
    EXPECT(!overlap(a, Rows{"b", nullptr, 64, 64, 10}));
    EXPECT(!overlap(a, Rows{"b", at(1000), 64, 64, 0}));
    const Rows left{"l", at(1000), 32, 96, 10};  // columns of rows of 96
    EXPECT(!overlap(left, Rows{"r", at(1032), 64, 96, 10}));
    EXPECT(!overlap(Rows{"r", at(1032), 64, 96, 10}, left));
    EXPECT(overlap(left, Rows{"r", at(1028), 64, 96, 10}));
    EXPECT(overlap(left, Rows{"r", at(1032), 68, 96, 10}));
    EXPECT(overlap(left, Rows{"r", at(1000), 32, 96, 10}));
    EXPECT(!overlap(left, Rows{"r", at(1000 + 96 + 32), 64, 96, 10}));
    EXPECT(!overlap(Rows{"r", at(1000 + 96 + 32), 64, 96, 10}, left));
    EXPECT(overlap(left, Rows{"r", at(1032), 64, 100, 10}));  // other pitch: taken as overlapping
}

static void short_conv() {
    auto same = [](strata_short_conv&) {};
    EXPECT(conv_with(same) == STRATA_OK);
    EXPECT(conv_with([](auto& d) { d.channels = 0; }) == STRATA_ERR_INVALID);
    EXPECT(conv_with([](auto& d) { d.taps = 0; }) == STRATA_ERR_INVALID);
    EXPECT(conv_with([](auto& d) { d.taps = 9; }) == STRATA_ERR_INVALID);
    EXPECT(conv_with([](auto& d) { d.taps = 8; }) == STRATA_OK);
    EXPECT(conv_with([](auto& d) { d.x_stride = 63; }) == STRATA_ERR_INVALID);
    EXPECT(conv_with([](auto& d) { d.y_stride = -64; }) == STRATA_ERR_INVALID);
    EXPECT(conv_with([](auto& d) { d.x_stride = INT64_MAX; }) == STRATA_ERR_INVALID);
    // rows and states whose byte offsets would pass 64 bits
    EXPECT(conv_with([](auto& d) { d.seq_len = 1 << 26, d.x_stride = int64_t(1) << 30; }) == STRATA_ERR_INVALID);
    EXPECT(conv_with([](auto& d) { d.seq_len = 1 << 24, d.x_stride = int64_t(1) << 30; }) == STRATA_OK);
    EXPECT(conv_with([](auto& d) { d.n_seq = 1 << 28, d.seq_len = 0, d.channels = 1 << 27; }) == STRATA_ERR_INVALID);
    EXPECT(conv_with([](auto& d) { d.dtype = STRATA_QUANT_F16; }) == STRATA_ERR_UNSUPPORTED_QUANT);
    EXPECT(conv_with([](auto& d) { d.dtype = STRATA_QUANT_Q8_0; }) == STRATA_ERR_UNSUPPORTED_QUANT);
    EXPECT(conv_with([](auto& d) { d.dtype = STRATA_QUANT_BF16; }) == STRATA_OK);

    strata_short_conv d = conv();
    Why why;
    int64_t tokens, longest;
    EXPECT(check_short_conv(why, d, &tokens, &longest) == STRATA_OK && d.x_stride == 64 && d.y_stride == 64);
    auto buffers = [&](const void* x, const float* w, const float* b, const float* s, const void* y) {
        return check_short_conv_buffers(why, d, tokens, x, w, b, s, y);
    };
    const uintptr_t X = 0x10000, W = 0x20000, B = 0x30000, S = 0x40000, Y = 0x50000;
    EXPECT(buffers(at(X), at<float>(W), at<float>(B), at<float>(S), at(Y)) == STRATA_OK);
    EXPECT(buffers(at(X), at<float>(W), nullptr, at<float>(S), at(Y)) == STRATA_OK);
    EXPECT(buffers(nullptr, at<float>(W), nullptr, at<float>(S), at(Y)) == STRATA_ERR_INVALID);
    EXPECT(buffers(at(X), nullptr, nullptr, at<float>(S), at(Y)) == STRATA_ERR_INVALID);
    EXPECT(buffers(at(X), at<float>(W), nullptr, nullptr, at(Y)) == STRATA_ERR_INVALID);
    EXPECT(buffers(at(X), at<float>(W), nullptr, at<float>(S), nullptr) == STRATA_ERR_INVALID);
    EXPECT(buffers(at(X + 2), at<float>(W), nullptr, at<float>(S), at(Y)) == STRATA_ERR_INVALID);
    EXPECT(buffers(at(X), at<float>(W), nullptr, at<float>(S), at(X)) == STRATA_ERR_INVALID);
    EXPECT(buffers(at(X), at<float>(W), nullptr, at<float>(S), at(S + 16)) == STRATA_ERR_INVALID);
    EXPECT(buffers(at(X), at<float>(X + 64), nullptr, at<float>(X + 256), at(Y)) == STRATA_ERR_INVALID);
    d.taps = 1;
    EXPECT(buffers(at(X), at<float>(W), nullptr, nullptr, at(Y)) == STRATA_OK);
}

static void gated_delta() {
    EXPECT(delta_with([](auto&) {}) == STRATA_OK);
    EXPECT(delta_with([](auto& d) { d.n_k_head = 3; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.n_k_head = 0; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.n_v_head = 0; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.k_dim = 0; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.k_dim = 257; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.k_dim = 256; }) == STRATA_OK);
    EXPECT(delta_with([](auto& d) { d.v_dim = 0; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.scale = NAN; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.scale = INFINITY; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.l2_eps = NAN; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.l2_eps = INFINITY; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.l2_eps = 0.0; }) == STRATA_OK);
    EXPECT(delta_with([](auto& d) { d.q_stride = 31; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.v_stride = 31; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.gate_stride = 3; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.o_stride = -1; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.seq_len = 1 << 28, d.v_stride = int64_t(1) << 28; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) {
               d.n_seq = 1 << 24, d.seq_len = 1, d.n_k_head = 1, d.n_v_head = 65536, d.k_dim = 256, d.v_dim = 8192;
           }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.scale = 1e39; }) == STRATA_ERR_INVALID);
    EXPECT(delta_with([](auto& d) { d.dtype = STRATA_QUANT_F16; }) == STRATA_ERR_UNSUPPORTED_QUANT);

    strata_gated_delta d = delta();
    d.q_stride = d.k_stride = d.v_stride = 96;  // q | k | v side by side: 32 + 32 + 32
    Why why;
    int64_t tokens, longest;
    EXPECT(check_gated_delta(why, d, &tokens, &longest) == STRATA_OK && d.o_stride == 32 && d.gate_stride == 4);
    const uintptr_t Q = 0x10000, G = 0x20000, E = 0x21000, S = 0x40000, O = 0x50000, C = 0x60000, W = 0x70000;
    auto buffers = [&](uintptr_t o, uintptr_t s, const float* coef, uintptr_t work, uint64_t have, uint64_t need) {
        return check_gated_delta_buffers(why, d, tokens, at(Q), at(Q + 128), at(Q + 256), at<float>(G), at<float>(E),
                                         coef, nullptr, at<float>(s), at(o), at(work), have, need);
    };
    EXPECT(buffers(O, S, nullptr, 0, 0, 0) == STRATA_OK);
    EXPECT(buffers(O, S, nullptr, 0, 0, 64) == STRATA_ERR_SCRATCH_LIMIT);
    EXPECT(buffers(O, S, nullptr, W, 63, 64) == STRATA_ERR_SCRATCH_LIMIT);
    EXPECT(buffers(O, S, nullptr, W, 64, 64) == STRATA_OK);
    EXPECT(buffers(O, S, nullptr, W + 8, 64, 64) == STRATA_ERR_INVALID);
    EXPECT(buffers(O, S, nullptr, S + 16, 64, 64) == STRATA_ERR_INVALID);
    EXPECT(buffers(O, S, nullptr, O + 16, 64, 64) == STRATA_ERR_INVALID);
    EXPECT(buffers(O, S, nullptr, Q + 16, 64, 64) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q + 256, S, nullptr, 0, 0, 0) == STRATA_ERR_INVALID);
    EXPECT(buffers(S, S, nullptr, 0, 0, 0) == STRATA_ERR_INVALID);
    EXPECT(buffers(O, Q, nullptr, 0, 0, 0) == STRATA_ERR_INVALID);
    EXPECT(buffers(0, S, nullptr, 0, 0, 0) == STRATA_ERR_INVALID);
    EXPECT(buffers(O, S + 2, nullptr, 0, 0, 0) == STRATA_ERR_INVALID);
    d.raw_gates = 1;
    EXPECT(buffers(O, S, nullptr, 0, 0, 0) == STRATA_ERR_INVALID);
    EXPECT(buffers(O, S, at<float>(C), 0, 0, 0) == STRATA_OK);
}

static void sample() {
    Why why;
    auto with = [&](int64_t rows, int64_t vocab, int64_t stride, uintptr_t logits, uintptr_t u, uintptr_t ids,
                    uintptr_t lp) {
        return check_sample(why, at<float>(logits), rows, vocab, stride, nullptr, nullptr, nullptr, nullptr,
                            at<double>(u), at<int32_t>(ids), at<float>(lp));
    };
    const uintptr_t L = 0x100000, U = 0x1000, I = 0x2000, P = 0x3000;
    EXPECT(with(3, 100, 0, L, U, I, P) == STRATA_OK);
    EXPECT(with(3, 100, 0, L, U, I, 0) == STRATA_OK);
    EXPECT(with(3, 100, 99, L, U, I, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 100, L, U, I, P) == STRATA_OK);
    EXPECT(with(0, 100, 0, L, U, I, P) == STRATA_ERR_INVALID);
    EXPECT(with((1 << 24) + 1, 100, 0, L, U, I, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 0, 0, L, U, I, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, (1 << 22) + 1, 0, L, U, I, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, 0, U, I, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, 0, I, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, U, 0, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L + 2, U, I, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, U + 4, I, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, U, L + 8, P) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, U, I, I + 8) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, U, I, U) == STRATA_ERR_INVALID);
}

int main() {
    sequences();
    overlaps();
    short_conv();
    gated_delta();
    sample();
    if (!failures) std::puts("ok");
    return failures ? 1 : 0;
}
