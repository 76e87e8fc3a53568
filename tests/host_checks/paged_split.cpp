// How a short prompt slice is split on a chip of 256 CUs: reads lines of
// "max_ctx max_prefill_tokens start T", prints "tokens of a block, positions of a
// chunk, workgroups per kv head" of each, and checks what the kernels rely on.
#include <stdio.h>

#include <algorithm>

#include "internal.hpp"

int main() {
    qff_ctx_cfg cfg{1, 0, 0};
    int start, T, bad = 0;
    while (scanf("%d %d %d %d", &cfg.max_ctx, &cfg.max_prefill_tokens, &start, &T) == 4) {
        const int slots = 128, cap = static_cast<int>(std::min<long long>(qff::kGqaMaxChunks, qff::pf_slots(cfg) / T));
        const qff::PagedTokens tk = qff::paged_tokens_split(start, T, slots, cap);
        const int chunks = (start + T + tk.ch - 1) / tk.ch, blocks = (T + tk.per - 1) / tk.per;
        // whole tiles; as many partials as there is room for; one round of workgroups, or one chunk a block
        const bool ok = cap >= 1 && tk.ch > 0 && tk.ch % qff::kPagedTile == 0 && chunks <= cap &&
                        (tk.items() <= slots || tk.items() == blocks) && (tk.per == 8 || tk.per == 16) &&
                        (!tk.append() || blocks == 1);   // (a wave appends one token, of the one block)
        bad += !ok;
        printf("%d %d %d%s\n", tk.per, tk.ch, tk.items(), ok ? "" : " BAD");
    }
    return bad != 0;
}
