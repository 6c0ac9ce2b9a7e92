// An append's two pools (csrc/attention_args.h): interleaved ones are taken, those of
// which a key's and a value's row share elements are refused. Compared with the
// elements of both, one by one, for small caches of every layout.
#include <cstdio>
#include <vector>

#include "attention_args.h"

using namespace strata;

static int failures = 0, shared = 0, apart = 0;

static void compare(strata_kv_cache c, int64_t shift) {
    strata_kv_append d = {};
    d.n_seq = 1, d.seq_len = 1, d.n_rot = 0;
    const int64_t base = int64_t(1) << 40;
    c.k_dev = reinterpret_cast<void*>(base), c.v_dev = reinterpret_cast<void*>(base + 2 * shift);
    c.table_dev = reinterpret_cast<const int32_t*>(0x10000), c.len_dev = reinterpret_cast<const int32_t*>(0x20000), c.max_pages = 4;
    Why why;
    int64_t tokens, longest;
    int rc = check_kv_append(why, d, c, &tokens, &longest);
    if (rc) {
        std::printf("shape: %s\n", why.text), ++failures;
        return;
    }
    rc = check_kv_append_buffers(why, d, c, tokens, nullptr, reinterpret_cast<void*>(0x100000), reinterpret_cast<void*>(0x200000), nullptr);
    std::vector<char> key(c.n_pages * c.page_stride + c.page_size * c.token_stride + c.n_kv_head * c.head_stride, 0);
    bool share = false;
    for (int pass = 0; pass < 2; ++pass)
        for (int64_t g = 0; g < c.n_pages; ++g)
            for (int64_t i = 0; i < c.page_size; ++i)
                for (int64_t h = 0; h < c.n_kv_head; ++h)
                    for (int64_t e = 0; e < c.head_dim; ++e) {
                        const int64_t at = g * c.page_stride + i * c.token_stride + h * c.head_stride + e;
                        if (pass == 0) key[at] = 1;
                        else if (at + shift >= 0 && at + shift < (int64_t)key.size()) share |= key[at + shift];
                    }
    (share ? shared : apart) += 1;
    if (rc != (share ? STRATA_ERR_INVALID : STRATA_OK) && ++failures < 10)
        std::printf("strides %lld %lld %lld, %lld elements apart: %d (%s), %s\n", (long long)c.page_stride, (long long)c.token_stride, (long long)c.head_stride,
                    (long long)shift, rc, why.text, share ? "they share some" : "they share none");
}

int main() {
    struct Shape {
        int64_t pages, heads, dim, page, token, head;
    };
    for (const Shape& s : {Shape{3, 2, 8, 0, 0, 0}, Shape{1, 1, 8, 0, 0, 0}, Shape{3, 2, 16, 2 * 16 * 32, 0, 0},          // packed, pages of both
                           Shape{2, 2, 16, 0, 64, 32}, Shape{2, 3, 8, 0, 64, 8}, Shape{2, 3, 8, 0, 64, 16},              // heads of both, tokens of both
                           Shape{2, 2, 8, 0, 8, 16 * 8}, Shape{2, 2, 8, 0, 16, 16 * 16}, Shape{2, 3, 8, 1024, 16, 16 * 24},  // heads outside tokens
                           Shape{2, 2, 16, 16 * 72 + 40, 72, 24}, Shape{4, 1, 8, 16 * 24, 24, 8}}) {
        strata_kv_cache c = {};
        c.n_pages = s.pages, c.page_size = 16, c.n_kv_head = s.heads, c.head_dim = s.dim;
        c.page_stride = s.page, c.token_stride = s.token, c.head_stride = s.head;
        for (int64_t shift = -5000; shift <= 5000; shift += 8) compare(c, shift);
        for (int64_t shift : {int64_t(1) << 36, -(int64_t(1) << 36)}) compare(c, shift);
    }
    if (shared < 1000 || apart < 1000) std::printf("%d that share, %d that do not\n", shared, apart), ++failures;
    if (!failures) std::puts("ok");
    return failures ? 1 : 0;
}
