// Pairs of one page-copy launch, by the bytes of a page: at least one, no more than
// the launch's arguments hold, and a grid of fewer than 2^32 work-items.
#include <stdio.h>

#include "internal.hpp"

int main() {
    int bad = 0;
    for (size_t bytes = 16; bytes <= size_t{1} << 31; bytes = bytes < 1 << 20 ? bytes + 16 : bytes + (size_t{1} << 20)) {
        const int pairs = qff::copy_pairs(bytes);
        const size_t segs = (bytes + qff::kCopySeg - 1) / qff::kCopySeg;
        const bool full = pairs == qff::kCopyPairs || (pairs + 1) * segs * qff::kCopyThreads > 0xffffffffull;   // none fewer than need be
        if (pairs < 1 || pairs > qff::kCopyPairs || pairs * segs * qff::kCopyThreads > 0xffffffffull || !full) {
            printf("%zu bytes: %d pairs\n", bytes, pairs);
            ++bad;
        }
    }
    return bad != 0;
}
