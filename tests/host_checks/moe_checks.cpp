// What the expert block's and the sampling entry points refuse on the host,
// without a GPU: a context made by hand (no device memory) and addresses that are
// never read. Every call here is refused, or has nothing to do, before any HIP call.
#include <math.h>
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
    float* f = reinterpret_cast<float*>(mem);
    int32_t* ints = reinterpret_cast<int32_t*>(mem);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(mem);
    const int I = QFF_ERR_INVALID_ARG, U = QFF_ERR_UNSUPPORTED, W = QFF_ERR_WORKSPACE;
    const qff_dtype bad = static_cast<qff_dtype>(7);
    const qff_q4_matrices m{w, a, a}, none{};

    // the norm: nothing of it is refused for its tokens' number, so 0 stands for a call that passes
    auto norm = [&](int tokens, int cols = 128, const void* x = nullptr, void* y = nullptr, const void* nw = nullptr, float eps = 1e-6f,
                    const qff_q4_matrices* g = nullptr, float* coef = nullptr, qff_dtype xd = QFF_F32, qff_dtype yd = QFF_F32,
                    qff_dtype wd = QFF_F32, qff_dtype sb = QFF_BF16) {
        return qff_rms_norm(&ctx, nullptr, x ? x : a, xd, nw ? nw : a, wd, eps, g, sb, y ? y : a, yd, coef, cols, tokens);
    };
    EXPECT(QFF_OK, norm(0));
    EXPECT(QFF_OK, norm(0, 8192, nullptr, nullptr, nullptr, 0.0f, &m));
    EXPECT(QFF_OK, qff_rms_norm(&ctx, nullptr, nullptr, QFF_BF16, a, QFF_F32, 1e-6f, nullptr, bad, nullptr, QFF_BF16, nullptr, 64, 0));
    EXPECT(I, norm(-1));
    EXPECT(U, norm(1, 8256));
    EXPECT(U, norm(1, 100));
    EXPECT(I, norm(1, 0));
    EXPECT(I, norm(1, 128, odd));
    EXPECT(I, norm(1, 128, nullptr, odd));
    EXPECT(I, norm(1, 128, nullptr, nullptr, odd));
    EXPECT(I, norm(1, 128, nullptr, nullptr, nullptr, -1.0f));
    EXPECT(I, norm(1, 128, nullptr, nullptr, nullptr, NAN));
    EXPECT(I, norm(1, 128, nullptr, nullptr, nullptr, 1e-6f, &m));   // a gate and nowhere to put its coefficient
    EXPECT(I, norm(1, 128, nullptr, nullptr, nullptr, 1e-6f, &none, f));
    EXPECT(I, norm(1, 128, nullptr, nullptr, nullptr, 1e-6f, &m, f, QFF_F32, QFF_F32, QFF_F32, QFF_F32));
    EXPECT(I, norm(1, 128, nullptr, nullptr, nullptr, 1e-6f, nullptr, f, QFF_F16));
    EXPECT(I, norm(1, 128, nullptr, nullptr, nullptr, 1e-6f, nullptr, f, QFF_F32, QFF_F16));
    EXPECT(I, norm(1, 128, nullptr, nullptr, nullptr, 1e-6f, nullptr, f, QFF_F32, QFF_F32, QFF_F16));
    EXPECT(I, qff_rms_norm(&ctx, nullptr, nullptr, QFF_F32, a, QFF_F32, 1e-6f, nullptr, QFF_BF16, a, QFF_F32, f, 128, 1));
    EXPECT(I, qff_rms_norm(nullptr, nullptr, a, QFF_F32, a, QFF_F32, 1e-6f, nullptr, QFF_BF16, a, QFF_F32, f, 128, 1));

    const qff_moe_weights p{m, m, m, m, m, m, QFF_BF16, 8, 128, 64};
    auto up = [&](const qff_moe_weights* q, int tokens = 65, int top = 2, const void* x = nullptr, const int32_t* idx = nullptr,
                  void* h = nullptr, qff_dtype xd = QFF_F32, qff_dtype hd = QFF_F16) {
        return qff_moe_gate_up(&ctx, nullptr, q, x ? x : a, xd, idx ? idx : ints, top, h ? h : a, hd, tokens);
    };
    auto down = [&](const qff_moe_weights* q, int tokens = 65, int top = 2, const void* h = nullptr, const void* res = nullptr,
                    void* y = nullptr, qff_dtype hd = QFF_F16, qff_dtype yd = QFF_F32) {
        return qff_moe_down(&ctx, nullptr, q, h ? h : a, hd, ints, f, top, f, res, y ? y : a, yd, tokens);
    };
    EXPECT(W, up(&p));   // tokens past the context's: the last check but the addresses'
    EXPECT(W, down(&p));
    EXPECT(QFF_OK, up(&p, 0));
    EXPECT(QFF_OK, down(&p, 0));
    EXPECT(I, up(nullptr));
    EXPECT(I, down(nullptr));
    EXPECT(I, up(&p, -1));
    EXPECT(I, down(&p, -1));
    EXPECT(I, up(&p, 65, 0));
    EXPECT(I, down(&p, 65, 0));
    EXPECT(U, up(&p, 65, 17));
    EXPECT(U, down(&p, 65, 17));
    EXPECT(I, up(&p, 4, 2, odd));
    EXPECT(I, up(&p, 4, 2, nullptr, nullptr, odd));
    EXPECT(I, up(&p, 65, 2, nullptr, nullptr, nullptr, QFF_F16));
    EXPECT(I, up(&p, 65, 2, nullptr, nullptr, nullptr, QFF_F32, bad));
    EXPECT(I, down(&p, 4, 2, odd));
    EXPECT(I, down(&p, 4, 2, nullptr, odd));
    EXPECT(I, down(&p, 4, 2, nullptr, nullptr, odd));
    EXPECT(I, down(&p, 65, 2, nullptr, nullptr, nullptr, bad));
    EXPECT(I, down(&p, 65, 2, nullptr, nullptr, nullptr, QFF_F32, QFF_F16));
    EXPECT(I, qff_moe_gate_up(nullptr, nullptr, &p, a, QFF_F32, ints, 2, a, QFF_F32, 1));
    EXPECT(I, qff_moe_gate_up(&ctx, nullptr, &p, a, QFF_F32, nullptr, 2, a, QFF_F32, 1));
    EXPECT(I, qff_moe_gate_up(&ctx, nullptr, &p, nullptr, QFF_F32, ints, 2, a, QFF_F32, 1));
    EXPECT(I, qff_moe_gate_up(&ctx, nullptr, &p, a, QFF_F32, ints, 2, nullptr, QFF_F32, 1));
    EXPECT(I, qff_moe_down(nullptr, nullptr, &p, a, QFF_F32, ints, f, 2, f, nullptr, a, QFF_F32, 1));
    EXPECT(I, qff_moe_down(&ctx, nullptr, &p, a, QFF_F32, nullptr, f, 2, f, nullptr, a, QFF_F32, 1));
    EXPECT(I, qff_moe_down(&ctx, nullptr, &p, a, QFF_F32, ints, nullptr, 2, f, nullptr, a, QFF_F32, 1));
    for (int i = 0; i < 20; ++i) {
        qff_moe_weights q = p;
        int wu = I, wd = I;   // what each half says
        switch (i) {
            case 0: q.sb_dtype = QFF_F32; break;
            case 1: q.experts = 0; break;
            case 2: q.experts = 513; wu = wd = U; break;
            case 3: q.hidden = 0; break;
            case 4: q.hidden = 96; wu = wd = U; break;
            case 5: q.hidden = 4160; wu = wd = U; break;
            case 6: q.inter = -64; break;
            case 7: q.inter = 32; wu = wd = U; break;
            case 8: q.inter = 8192; wu = wd = U; break;
            case 9: q.gate = none; wd = W; break;      // (the down products do not read it)
            case 10: q.up.scales = nullptr; wd = W; break;
            case 11: q.up.w = reinterpret_cast<const uint32_t*>(odd); wd = W; break;
            case 12: q.down = none; wu = W; break;
            case 13: q.down.biases = nullptr; wu = W; break;
            case 14: q.shared_gate = none; wd = W; break;   // half a shared expert
            case 15: q.shared_up = none; wd = W; break;
            case 16: q.shared_up.biases = nullptr; wd = W; break;
            case 17: q.shared_down.scales = nullptr; wu = W; break;
            case 18: q.shared_down = none; wu = W; wd = W; break;
            case 19: q.shared_gate = q.shared_up = none; wu = W; wd = W; break;
        }
        EXPECT(wu, up(&q));
        EXPECT(wd, down(&q));
    }

    auto sample = [&](int batch, int vocab = 100, qff_dtype dt = QFF_F32) {
        return qff_sample(&ctx, nullptr, a, dt, f, f, ints, f, f, ints, f, vocab, batch);
    };
    EXPECT(W, sample(5));
    EXPECT(W, sample(5, 262144));
    EXPECT(U, sample(5, 262145));
    EXPECT(I, sample(5, 0));
    EXPECT(I, sample(5, 100, QFF_F16));
    EXPECT(I, sample(-1));
    EXPECT(QFF_OK, sample(0));
    EXPECT(QFF_OK, qff_sample(&ctx, nullptr, nullptr, QFF_F32, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1, 0));
    EXPECT(I, qff_sample(nullptr, nullptr, a, QFF_F32, f, f, ints, f, f, ints, f, 100, 1));
    EXPECT(I, qff_sample(&ctx, nullptr, nullptr, QFF_F32, f, f, ints, f, f, ints, f, 100, 1));
    EXPECT(I, qff_sample(&ctx, nullptr, a, QFF_F32, nullptr, f, ints, f, f, ints, f, 100, 1));
    EXPECT(I, qff_sample(&ctx, nullptr, a, QFF_F32, f, f, ints, f, f, nullptr, f, 100, 1));
    EXPECT(W, qff_sample(&ctx, nullptr, a, QFF_BF16, f, nullptr, nullptr, nullptr, nullptr, ints, nullptr, 100, 5));
    printf("%d failures\n", failures);
    return failures != 0;
}
