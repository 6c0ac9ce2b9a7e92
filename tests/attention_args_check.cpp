// The argument checks of the attention operators (csrc/attention_args.h) run on
// the host: what is refused, with which status, and that packed strides are
// filled in. Buffers are addresses only; nothing is dereferenced.
#include <cmath>
#include <cstdio>
#include <limits>

#include "attention_args.h"

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

static strata_kv_cache pool() {
    strata_kv_cache c = {};
    c.k_dev = at(0x1000000), c.v_dev = at(0x2000000), c.table_dev = at<int32_t>(0x10000), c.len_dev = at<int32_t>(0x20000);
    c.n_pages = 10, c.page_size = 32, c.n_kv_head = 2, c.head_dim = 64, c.max_pages = 4;
    return c;
}
template <typename F>
static int cache_with(F change, int64_t n_seq = 3) {
    strata_kv_cache c = pool();
    change(c);
    Why why;
    return check_kv_cache(why, c, n_seq);
}
static strata_kv_append append() {
    strata_kv_append d = {};
    d.n_seq = 3, d.seq_len = 5, d.n_head = 4, d.n_rot = 64, d.freq_base = 1e4;
    return d;
}
static strata_attention attention() {
    strata_attention d = {};
    d.n_seq = 3, d.seq_len = 5, d.n_head = 4, d.scale = 0.125;
    return d;
}
template <typename F>
static int append_with(F change) {
    strata_kv_append d = append();
    strata_kv_cache c = pool();
    change(d);
    Why why;
    int64_t tokens, longest;
    return check_kv_append(why, d, c, &tokens, &longest);
}
template <typename F>
static int attention_with(F change) {
    strata_attention d = attention();
    strata_kv_cache c = pool();
    change(d);
    Why why;
    int64_t tokens, longest;
    return check_attention(why, d, c, &tokens, &longest);
}

static void caches() {
    strata_kv_cache c = pool();
    Why why;
    EXPECT(check_kv_cache(why, c, 3) == STRATA_OK && c.head_stride == 64 && c.token_stride == 128 && c.page_stride == 32 * 128 && c.table_stride == 4);
    c = pool(), c.token_stride = 64, c.head_stride = 32 * 64;  // heads outside tokens
    EXPECT(check_kv_cache(why, c, 3) == STRATA_OK && c.page_stride == 2 * 32 * 64);
    c = pool(), c.page_stride = 2 * 32 * 128;  // both pools in one
    EXPECT(check_kv_cache(why, c, 3) == STRATA_OK);
    c = pool(), c.token_stride = 256, c.head_stride = 128;  // keys and values head by head
    EXPECT(check_kv_cache(why, c, 3) == STRATA_OK && c.page_stride == 32 * 256);
    const int64_t big = int64_t(1) << 62;
    EXPECT(cache_with([](auto& c) { c.head_dim = 256; }) == STRATA_OK);
    EXPECT(cache_with([](auto& c) { c.head_dim = 264; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.head_dim = 0; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.head_dim = 60; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.page_size = 8; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.page_size = 40; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.page_size = 48; }) == STRATA_OK);
    EXPECT(cache_with([](auto& c) { c.page_size = -16; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([=](auto& c) { c.page_size = big; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.n_pages = 0; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([=](auto& c) { c.n_pages = big; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.n_kv_head = 0; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.n_kv_head = 1025; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.max_pages = 0; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.max_pages = (1 << 26); }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.max_pages = (1 << 26) - 1; }) == STRATA_OK);
    EXPECT(cache_with([](auto& c) { c.table_stride = 3; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.table_stride = 5; }) == STRATA_OK);
    EXPECT(cache_with([=](auto& c) { c.table_stride = big; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.table_stride = int64_t(1) << 31; }, kMaxTokens) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.head_stride = 56; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.head_stride = 68; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([=](auto& c) { c.head_stride = big; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.head_stride = -64; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.token_stride = 120; }) == STRATA_ERR_INVALID);  // neither layout
    EXPECT(cache_with([](auto& c) { c.token_stride = 132; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([=](auto& c) { c.token_stride = big; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.page_stride = 32 * 128 - 8; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([](auto& c) { c.page_stride = 32 * 128 + 4; }) == STRATA_ERR_INVALID);
    EXPECT(cache_with([=](auto& c) { c.page_stride = big; }) == STRATA_ERR_INVALID);
}

static void appends() {
    EXPECT(append_with([](auto&) {}) == STRATA_OK);
    EXPECT(append_with([](auto& d) { d.n_head = 0; }) == STRATA_OK);
    EXPECT(append_with([](auto& d) { d.n_head = 3; }) == STRATA_OK);  // no multiple is asked for
    EXPECT(append_with([](auto& d) { d.n_head = -1; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.n_rot = 0, d.freq_base = 0; }) == STRATA_OK);
    EXPECT(append_with([](auto& d) { d.n_rot = 33; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.n_rot = 66; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.n_rot = -2; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.freq_base = 0; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.freq_base = INFINITY; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.freq_base = NAN; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.q_stride = 255; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.k_stride = 127; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.v_stride = -1; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.q_out_stride = INT64_MAX; }) == STRATA_ERR_INVALID);
    EXPECT(append_with([](auto& d) { d.dtype = STRATA_QUANT_F16; }) == STRATA_ERR_UNSUPPORTED_QUANT);
    EXPECT(append_with([](auto& d) { d.q_dtype = STRATA_QUANT_Q8_0; }) == STRATA_ERR_UNSUPPORTED_QUANT);
    EXPECT(append_with([](auto& d) { d.n_seq = 0; }) == STRATA_ERR_INVALID);

    strata_kv_append d = append();
    strata_kv_cache c = pool();
    Why why;
    int64_t tokens, longest;
    EXPECT(check_kv_append(why, d, c, &tokens, &longest) == STRATA_OK && d.q_stride == 256 && d.k_stride == 128 && d.q_out_stride == 256 && tokens == 15);
    auto buffers = [&](uintptr_t q, uintptr_t k, uintptr_t v, uintptr_t o) { return check_kv_append_buffers(why, d, c, tokens, at(q), at(k), at(v), at(o)); };
    const uintptr_t Q = 0x100000, K = 0x200000, V = 0x300000, O = 0x400000;
    EXPECT(buffers(Q, K, V, O) == STRATA_OK);
    EXPECT(buffers(Q, K, V, Q) == STRATA_OK);  // in place
    d.q_dtype = STRATA_QUANT_BF16;
    EXPECT(buffers(Q, K, V, Q) == STRATA_ERR_INVALID);
    d.q_dtype = STRATA_QUANT_F32;
    EXPECT(buffers(Q, K, V, Q + 4) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, K, V, K) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, K, V, 0x1000000) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, K, 0x2000000 + 64, O) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, K, V, 0x10000) == STRATA_ERR_INVALID);
    EXPECT(buffers(0, K, V, O) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, 0, V, O) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, K, 0, O) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, K, V, 0) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q + 2, K, V, O) == STRATA_ERR_INVALID);
    d.n_head = 0;
    EXPECT(buffers(0, K, V, 0) == STRATA_OK);
    d.n_head = 4;
    c.v_dev = c.k_dev;
    EXPECT(buffers(Q, K, V, O) == STRATA_ERR_INVALID);
    c.v_dev = at(0x2000008);
    EXPECT(buffers(Q, K, V, O) == STRATA_ERR_INVALID);
    c.v_dev = at(0x2000000), c.len_dev = nullptr;
    EXPECT(buffers(Q, K, V, O) == STRATA_ERR_INVALID);
}

static void attentions() {
    EXPECT(attention_with([](auto&) {}) == STRATA_OK);
    EXPECT(attention_with([](auto& d) { d.n_head = 3; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.n_head = 0; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.window = -1; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.sinks = -1; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.window = INT64_MAX, d.sinks = INT64_MAX; }) == STRATA_OK);
    EXPECT(attention_with([](auto& d) { d.scale = 0; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.scale = -1; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.scale = NAN; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.scale = 1e39; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.scale = 3e38; }) == STRATA_ERR_INVALID);  // times log2(e) it is infinite
    EXPECT(attention_with([](auto& d) { d.scale = 2e38; }) == STRATA_OK);
    EXPECT(attention_with([](auto& d) { d.q_stride = 100; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.o_stride = 100; }) == STRATA_ERR_INVALID);
    EXPECT(attention_with([](auto& d) { d.dtype = STRATA_QUANT_F16; }) == STRATA_ERR_UNSUPPORTED_QUANT);
    EXPECT(attention_with([](auto& d) { d.n_seq = 1, d.seq_len = 1 << 20, d.n_head = 65536; }) == STRATA_ERR_INVALID);

    strata_attention d = attention();
    strata_kv_cache c = pool();
    Why why;
    int64_t tokens, longest;
    EXPECT(check_attention(why, d, c, &tokens, &longest) == STRATA_OK && d.q_stride == 256 && d.o_stride == 256 && tokens == 15);
    auto buffers = [&](uintptr_t q, uintptr_t o, uintptr_t w, uint64_t have, uint64_t need) {
        return check_attention_buffers(why, d, c, tokens, at(q), at(o), at(w), have, need);
    };
    const uintptr_t Q = 0x100000, O = 0x400000, W = 0x500000;
    EXPECT(buffers(Q, O, W, 4096, 4096) == STRATA_OK);
    EXPECT(buffers(Q, O, W, 4095, 4096) == STRATA_ERR_SCRATCH_LIMIT);
    EXPECT(buffers(Q, O, 0, 4096, 4096) == STRATA_ERR_SCRATCH_LIMIT);
    EXPECT(buffers(Q, O, W + 8, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(0, O, W, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, 0, W, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, Q, W, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, O, O, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, O, Q + 16, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, 0x1000010, W, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, O, 0x2000010, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q, O, 0x10000, 4096, 4096) == STRATA_ERR_INVALID);
    EXPECT(buffers(Q + 1, O, W, 4096, 4096) == STRATA_ERR_INVALID);
}

static void logprobs() {
    Why why;
    const uintptr_t L = 0x100000, T = 0x1000, P = 0x2000, E = 0x3000, I = 0x4000, A = 0x5000;
    auto with = [&](int64_t rows, int64_t vocab, int64_t stride, uintptr_t l, uintptr_t t, uintptr_t p, uintptr_t e, int64_t top, uintptr_t i, uintptr_t a) {
        return check_logprobs(why, at<float>(l), rows, vocab, stride, at<int32_t>(t), at<float>(p), at<float>(e), top, at<int32_t>(i), at<float>(a));
    };
    EXPECT(with(3, 100, 0, L, T, P, E, 5, I, A) == STRATA_OK);
    EXPECT(with(3, 100, 0, L, T, P, 0, 0, 0, 0) == STRATA_OK);
    EXPECT(with(3, 100, 0, L, 0, 0, E, 0, 0, 0) == STRATA_OK);
    EXPECT(with(0, 100, 0, 0, 0, 0, 0, 5, 0, 0) == STRATA_OK);
    EXPECT(with(3, 100, 0, L, 0, P, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, 0, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, P, E, 5, 0, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, P, E, 5, I, 0) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, 0, T, P, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(-1, 100, 0, L, T, P, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with((1 << 24) + 1, 100, 0, L, T, P, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 0, 0, L, T, P, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, (1 << 22) + 1, 0, L, T, P, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 99, L, T, P, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, P, E, 33, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, P, E, -1, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L + 2, T, P, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, L + 40, E, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, P, P + 8, 5, I, A) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, P, E, 5, I, I + 56) == STRATA_ERR_INVALID);
    EXPECT(with(3, 100, 0, L, T, P, E, 5, I, I + 60) == STRATA_OK);
    EXPECT(with(3, 100, 0, L, T, T + 8, E, 5, I, A) == STRATA_ERR_INVALID);
}

int main() {
    caches();
    appends();
    attentions();
    logprobs();
    if (!failures) std::puts("ok");
    return failures ? 1 : 0;
}
