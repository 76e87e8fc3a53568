// What the paged-cache entry points refuse on the host, without a GPU: a
// context made by hand (no device memory) and addresses that are never read.
// Every call here is refused before any HIP call.
#include <stdio.h>

#include "internal.hpp"

static int failures = 0;
#define EXPECT(status, call)                                                     \
    do {                                                                         \
        const int got = (call);                                                  \
        if (got != (status)) {                                                   \
            printf("line %d: %d, expected %d: %s\n", __LINE__, got, status, #call); \
            ++failures;                                                          \
        }                                                                        \
    } while (0)

int main() {
    qff_ctx ctx;
    ctx.cfg = qff_ctx_cfg{4, 1000, 64};
    alignas(16) static char mem[64];
    void *a = mem, *odd = mem + 4;
    const float* w = reinterpret_cast<const float*>(mem);
    const int32_t* ints = reinterpret_cast<const int32_t*>(mem);
    const qff_gqa_params p{w, w, 1e7f, 64, 1.0f / 16, 1e-6f, 0};
    const qff_kv_pages kv{a, a, ints, 10, 64, 16};   // 1024 positions: max_ctx in whole pages
    const int I = QFF_ERR_INVALID_ARG, U = QFF_ERR_UNSUPPORTED, W = QFF_ERR_WORKSPACE;

    auto decode = [&](const qff_kv_pages* k, const qff_gqa_params* prm = nullptr, void* q = nullptr, int batch = 5,
                      qff_dtype in = QFF_F32, qff_dtype out = QFF_F32) {
        return qff_gqa_decode_paged(&ctx, nullptr, prm ? prm : &p, q ? q : a, a, a, in, k, ints, a, out, batch);
    };
    EXPECT(W, decode(&kv));   // batch past the context's: the last check, so all the others passed
    EXPECT(I, decode(nullptr));
    EXPECT(I, decode(&kv, nullptr, nullptr, 0));
    EXPECT(I, decode(&kv, nullptr, nullptr, -1));
    EXPECT(I, decode(&kv, nullptr, odd));
    EXPECT(I, decode(&kv, nullptr, nullptr, 5, QFF_F16));
    EXPECT(I, decode(&kv, nullptr, nullptr, 5, QFF_F32, static_cast<qff_dtype>(7)));
    for (int i = 0; i < 11; ++i) {
        qff_kv_pages k = kv;
        int want = I;
        switch (i) {
            case 0: k.k = nullptr; break;
            case 1: k.v = nullptr; break;
            case 2: k.table = nullptr; break;
            case 3: k.k = odd; break;
            case 4: k.v = odd; break;
            case 5: k.num_pages = 0; break;
            case 6: k.page_size = 0; break;
            case 7: k.table_cols = 0; break;
            case 8: k.page_size = 48; k.table_cols = 1; want = U; break;
            case 9: k.page_size = 8; want = U; break;
            case 10: k.table_cols = 17; want = W; break;
        }
        EXPECT(want, decode(&k));
        EXPECT(want, qff_gqa_prefill_paged(&ctx, nullptr, &p, a, a, a, QFF_F32, &k, 0, a, QFF_F32, 65));
        EXPECT(want, qff_gqa_decode_shared(&ctx, nullptr, &p, a, a, a, QFF_F32, &k, ints, ints, ints, a, QFF_F32, 5));
    }
    EXPECT(I, qff_gqa_prefill_paged(&ctx, nullptr, &p, a, odd, a, QFF_F32, &kv, 0, a, QFF_F32, 65));
    EXPECT(I, qff_gqa_prefill_paged(&ctx, nullptr, &p, a, a, odd, QFF_F32, &kv, 0, a, QFF_F32, 65));
    qff_kv_pages big = kv;
    big.page_size = 8192;
    big.table_cols = 1;
    EXPECT(U, decode(&big));
    big.page_size = 4096;
    big.table_cols = 1 << 30;   // (the product is taken in 64 bits)
    EXPECT(W, decode(&big));
    qff_gqa_params q = p;
    q.q_norm_w = reinterpret_cast<const float*>(odd);
    EXPECT(I, decode(&kv, &q));
    q = p;
    q.kv_f16 = 2;
    EXPECT(I, decode(&kv, &q));
    q = p;
    q.rotary_dim = 128;
    EXPECT(U, decode(&kv, &q));
    EXPECT(I, qff_gqa_decode_paged(nullptr, nullptr, &p, a, a, a, QFF_F32, &kv, ints, a, QFF_F32, 1));
    EXPECT(I, qff_gqa_decode_paged(&ctx, nullptr, nullptr, a, a, a, QFF_F32, &kv, ints, a, QFF_F32, 1));
    EXPECT(I, qff_gqa_decode_paged(&ctx, nullptr, &p, a, a, a, QFF_F32, &kv, nullptr, a, QFF_F32, 1));
    EXPECT(I, qff_gqa_decode_paged(&ctx, nullptr, &p, a, a, a, QFF_F32, &kv, ints, nullptr, QFF_F32, 1));
    EXPECT(W, qff_gqa_decode_shared(&ctx, nullptr, &p, a, a, a, QFF_F32, &kv, ints, ints, ints, a, QFF_F32, 5));
    EXPECT(I, qff_gqa_decode_shared(&ctx, nullptr, &p, a, a, a, QFF_F32, &kv, ints, nullptr, ints, a, QFF_F32, 5));
    EXPECT(I, qff_gqa_decode_shared(&ctx, nullptr, &p, a, a, a, QFF_F32, &kv, ints, ints, nullptr, a, QFF_F32, 5));

    auto prefill = [&](int start, int T, void* out = nullptr, const qff_kv_pages* k = nullptr) {
        return qff_gqa_prefill_paged(&ctx, nullptr, &p, a, a, a, QFF_F32, k ? k : &kv, start, out ? out : a, QFF_F32, T);
    };
    EXPECT(W, prefill(0, 65));       // more tokens than the context's
    EXPECT(W, prefill(990, 20));     // past its max_ctx, inside the table
    EXPECT(I, prefill(0, 0));
    EXPECT(I, prefill(-1, 4));
    EXPECT(I, prefill(1020, 5));     // past the table
    EXPECT(I, prefill(0x7fffffff, 5));
    EXPECT(I, prefill(0, 65, odd));

    // copies: two pools of 100 pages
    void* pools[2] = {a, a};
    auto copy = [&](std::vector<int32_t> s, std::vector<int32_t> d, size_t bytes = 16, int pages = 100, int npools = 2) {
        return qff_pages_copy(&ctx, nullptr, pools, npools, bytes, pages, s.data(), d.data(), static_cast<int>(s.size()));
    };
    EXPECT(QFF_OK, copy({}, {}));
    EXPECT(QFF_OK, qff_pages_copy(&ctx, nullptr, pools, 2, 16, 100, nullptr, nullptr, 0));
    for (int round = 0; round < 2; ++round) {   // (a refused call leaves no mark on the next)
        EXPECT(I, copy({1, 2}, {3, 3}));
        EXPECT(I, copy({1, 2}, {2, 3}));
        EXPECT(I, copy({1, 2}, {3, 1}));
        EXPECT(I, copy({7}, {7}));
        EXPECT(I, copy({100}, {1}));
        EXPECT(I, copy({1}, {100}));
        EXPECT(I, copy({-1}, {1}));
        EXPECT(I, copy({1}, {-1}));
        EXPECT(I, copy({99, 98}, {64, 99}));
    }
    for (uint64_t word : ctx.page_bits)
        if (word) ++failures, printf("a mark was left\n");
    EXPECT(U, copy({1}, {2}, 8));
    EXPECT(U, copy({1}, {2}, 24));
    EXPECT(U, copy({1}, {2}, (size_t{1} << 31) + 16));
    EXPECT(I, copy({1}, {2}, 0));
    EXPECT(I, copy({1}, {2}, 16, 0));
    EXPECT(I, copy({1}, {2}, 16, 100, 0));
    EXPECT(I, qff_pages_copy(&ctx, nullptr, nullptr, 2, 16, 100, ints, ints, 1));
    EXPECT(I, qff_pages_copy(&ctx, nullptr, pools, 2, 16, 100, nullptr, ints, 1));
    EXPECT(I, qff_pages_copy(&ctx, nullptr, pools, 2, 16, 100, ints, nullptr, 1));
    EXPECT(I, qff_pages_copy(&ctx, nullptr, pools, 2, 16, 100, ints, ints, -1));
    EXPECT(I, qff_pages_copy(nullptr, nullptr, pools, 2, 16, 100, ints, ints, 1));
    pools[1] = odd;
    EXPECT(I, copy({1}, {2}));
    pools[1] = nullptr;
    EXPECT(I, copy({1}, {2}));
    printf("%d failures\n", failures);
    return failures != 0;
}
