// pages.hip -- copies of pages within pools: a fork's last page or its
// recurrent states, the moves of a compaction.
//
// pool[dst[i]] = pool[src[i]] for every pool and pair i. A pure stream: each
// source page read once, each destination written once, 16 KB a workgroup
// (four 16-byte pieces a lane, all requested before the first is stored).
// Stores are non-temporal, and loads too where no source occurs twice: 1777
// pages of 16 KB in 20 pools 231 us (5.05 TB/s read + written; 248 with
// ordinary loads and stores, 237 with ordinary loads), 7 copies of a 2 MiB
// state in 30 pools 74 us with ordinary loads, whose source then comes from the
// cache (106 with ordinary stores, 110 with non-temporal loads too). The pairs
// travel in the kernel's arguments (no upload, no workspace; a captured
// call replays the pairs it was captured with), as many as 4 KB of arguments
// hold with the pool addresses and a launch takes work-items for: more go in
// further launches.
#include <algorithm>

#include "common.hpp"
#include "internal.hpp"
#include "mfma.hpp"

namespace qff {

constexpr int kCopyPools = 32;

struct CopyArgs {
    char* pools[kCopyPools];
    int32_t src[kCopyPairs], dst[kCopyPairs];
    size_t page_bytes;
    int segs;
};
static_assert(sizeof(CopyArgs) <= 4096 - 64, "kernel arguments");

template <bool ONCE>
__global__ __launch_bounds__(kCopyThreads) void pages_copy_kernel(const CopyArgs a) {
    const int pair = static_cast<int>(blockIdx.x) / a.segs, seg = static_cast<int>(blockIdx.x) - pair * a.segs;
    char* pool = a.pools[blockIdx.y];
    const char* from = pool + static_cast<size_t>(a.src[pair]) * a.page_bytes;
    char* to = pool + static_cast<size_t>(a.dst[pair]) * a.page_bytes;
    const size_t at = seg * kCopySeg + 16 * threadIdx.x, last = a.page_bytes - 16;
    u32x4_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(from + std::min(at + 4096 * i, last));
        w[i] = ONCE ? __builtin_nontemporal_load(p) : *p;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + 4096 * i <= last) __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4_t*>(to + at + 4096 * i));
}

hipError_t launch_pages_copy(qff_ctx* ctx, hipStream_t stream, void* const* pools, int npools, size_t page_bytes,
                             const int32_t* src, const int32_t* dst, int n, bool once) {
    ProfScope prof(ctx, stream, "pages_copy");
    CopyArgs a;
    a.page_bytes = page_bytes;
    a.segs = static_cast<int>((page_bytes + kCopySeg - 1) / kCopySeg);
    const int most = copy_pairs(page_bytes);
    for (int i0 = 0; i0 < n; i0 += most) {
        const int pairs = std::min(most, n - i0);
        std::copy(src + i0, src + i0 + pairs, a.src);
        std::copy(dst + i0, dst + i0 + pairs, a.dst);
        for (int p0 = 0; p0 < npools; p0 += kCopyPools) {
            const int count = std::min(kCopyPools, npools - p0);
            for (int p = 0; p < count; ++p) a.pools[p] = static_cast<char*>(pools[p0 + p]);
            const dim3 grid(pairs * a.segs, count);
            if (once) pages_copy_kernel<true><<<grid, kCopyThreads, 0, stream>>>(a);
            else pages_copy_kernel<false><<<grid, kCopyThreads, 0, stream>>>(a);
        }
    }
    return hipGetLastError();
}

}  // namespace qff
