// Batches that qff_sample refuses on the host: a context made by hand, addresses that are never read.
#include <stdio.h>

#include "internal.hpp"

int main() {
    qff_ctx ctx;
    ctx.cfg = qff_ctx_cfg{100000, 64, 1};
    alignas(16) static char mem[64];
    float* f = reinterpret_cast<float*>(mem);
    int32_t* ints = reinterpret_cast<int32_t*>(mem);
    auto sample = [&](int vocab, int batch) {
        return qff_sample(&ctx, nullptr, f, QFF_F32, f, nullptr, nullptr, nullptr, nullptr, ints, nullptr, vocab, batch);
    };
    // (more than a grid's second dimension; more than max_batch; a vocabulary too large; nothing to do)
    const int got[] = {sample(1000, 65536), sample(1000, 100001), sample(262145, 1), sample(1000, 0)};
    printf("%d %d %d %d\n", got[0], got[1], got[2], got[3]);
    return got[0] == QFF_ERR_UNSUPPORTED && got[1] == QFF_ERR_UNSUPPORTED && got[2] == QFF_ERR_UNSUPPORTED && got[3] == QFF_OK ? 0 : 1;
}
