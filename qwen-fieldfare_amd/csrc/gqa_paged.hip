// gqa_paged.hip -- full-attention decode (16 q heads on 2 kv heads, head dim
// 256) whose K/V rows live in pages of a pool, for a batch of sequences on
// gfx950, with the positions that a group of sequences has in common read
// once for all of them.
//
// Position p of sequence b is row p % page_size of page table[b][p /
// page_size] in pools [num_pages][page_size][2][256] (bf16 or fp16). Per q
// head h (kv head j = h / 8) of a sequence at position t = positions[b]:
//   q = rope(rms(q_h) wq, t), k = rope(rms(k_j) wk, t), K[t] = k, V[t] = v,
//   o = sum_{p <= t} softmax_p(scale q . K[p]) V[p],  out = o sigmoid(gate).
// The positions are split into ranges; every range gives one partial per q
// head, its base-2 maximum m, sum d and unnormalised o, and the partials are
// joined with weights 2^(m - max m).
//
//   partial  one workgroup per (block of sequences, kv head, chunk of
//            positions): a group's shared positions for up to 8 or 16 of its
//            sequences (128 q rows), or one sequence's own positions (8 q
//            rows), whose last chunk appends the new token. K/V tiles go
//            through LDS. One launch for both, so that the few long streams of
//            a shared prefix and the many short ones behind it run together.
//   combine  one workgroup per (q head, sequence): joins the partials, gate.
//
// Both products run on 16x16x32 MFMAs in the cache's type, in which K and V
// are exact. q and the softmax weights enter as NT terms of that type (hi,
// the rest rounded again, ...): two bf16 terms carry 16 bits and two fp16
// terms 22, three bf16 terms 24. What q's terms leave out shows in proportion to
// the scores. fp32 outputs take three terms of bf16 or two of fp16 (error 2e-7 to
// 7e-7 of a row at scores of rms 1, where two bf16 terms leave 6e-6). bf16
// outputs, whose own rounding is 1.7e-3, take two of either: two bf16 terms leave 3e-6
// at scores of rms 1 and 9e-5 in the worst row at 25; one fp16 term would leave
// 3e-4 and 7e-3, more than the output's rounding once trained norm weights spread
// the scores (a 64-bit emulation over 4096 positions). fp16
// weights are scaled by 2^7 (kShift), so that weights down to 2^-21 of the row's
// largest keep all bits of their first term.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.hpp"
#include "internal.hpp"
#include "mfma.hpp"

namespace qff {

// ---- split of a call's positions ------------------------------------------------
//
// Every workgroup derives the same split from the device arrays (no host
// sync, no atomics). `positions` give each sequence's length L (0 where the
// position lies outside the table: no chunks, its output is NaN). With groups,
// consecutive sequences with the same group >= 0 (and L > 0) are a run, cut at
// every multiple of 64 sequences and into even blocks of up to 8 or 16; the
// positions before S = the least of the block's shared_len and L - 1, rounded
// down to 16, are read through the table row of the block's first sequence for
// all of it. Any values of the arrays give a valid split.
//
// A CU holds one workgroup (its LDS), which leaves the CU idle while it starts,
// so the chunk length is about the least that needs no second round of
// workgroups where such a length exists.

constexpr int kBlkSeqs = kPagedBlk;   // sequences of a block at most
constexpr int kTile = kPagedTile;   // positions of a tile
// Blocks of 8 start and end sooner and spread over more workgroups, blocks of 16
// read the prefix half as often: 8 where that makes chunks of up to
// kPagedSmallTiles (us with 8 / 16, bf16 outputs of a bf16 cache, an fp16 one within 2 %:
// 16 sequences on 6K 23.4 / 26.5, on 32K, 9 tiles, 38.5 / 41.7; 32 on 16K, 10 tiles,
// 39.8 / 40.7; 24 on 32K, 13 tiles, 47.5 / 53.4; 32 on 24K, 14 tiles, 48.0 / 47.2, on
// 32K 58.4 / 56.4; fp32 outputs 24 on 32K 55.6 / 62.5, 32 on 24K 56.3 / 54.3).
constexpr int kMinShared = 64;  // shorter shared prefixes are left to the sequences

struct PagedSeqs {
    const int32_t* positions;
    const int32_t* group;        // null: no groups
    const int32_t* shared_len;
    int batch, max_ctx;
    int slots;   // workgroups of one round, per kv head
    int cap;     // chunks allowed per sequence
};

// Sequence b0 + lane: its length, the shared positions of its block, the
// block's first sequence (as a lane) and size; shared is 0 for single
// sequences.
struct LanePlan {
    int len, shared, first, count;
    __device__ __forceinline__ int own() const { return len - shared; }
};

__device__ __forceinline__ LanePlan lane_plan(const PagedSeqs& a, int b0, int lane, int bs) {
    const int b = b0 + lane;
    LanePlan p{0, 0, lane, 1};
    int grp = -1, sh = 0;
    if (b < a.batch) {
        const int pos = a.positions[b];
        if (a.group) {
            grp = a.group[b];
            sh = a.shared_len[b];
        }
        p.len = (pos >= 0 && pos < a.max_ctx) ? pos + 1 : 0;
    }
    if (!a.group) return p;   // (uniform)
    if (p.len == 0) grp = -1;
    const int prev = __shfl_up(grp, 1, 64);
    const unsigned long long below = ~0ull >> (63 - lane);   // lanes 0 .. lane
    const unsigned long long runs = __ballot(lane == 0 || grp < 0 || grp != prev);
    const int run = 63 - __builtin_clzll(runs & below);
    // blocks as even as they can be
    const unsigned long long later = runs & ~below;
    const int members = (later ? static_cast<int>(__builtin_ctzll(later)) : 64) - run;
    // quotients of numbers up to 80, by reciprocals
    auto quotient = [](int x, int y) { return static_cast<int>((static_cast<float>(x) + 0.5f) * __builtin_amdgcn_rcpf(static_cast<float>(y))); };
    const int nblk = (members + bs - 1) / bs, size = quotient(members + nblk - 1, nblk);
    const int at = lane - run;
    const unsigned long long blocks = __ballot(at == quotient(at, size) * size);
    p.first = 63 - __builtin_clzll(blocks & below);
    const unsigned long long after = blocks & ~below;
    const int end = after ? static_cast<int>(__builtin_ctzll(after)) : 64;
    p.count = end - p.first;
    // least of the block, in its first lane (four steps reach 15 lanes on)
    int s = max(0, min(sh, p.len - 1));
#pragma unroll
    for (int off = 1; off < kBlkSeqs; off *= 2) {
        const int o = __shfl_down(s, off, 64);
        if (lane + off < end) s = min(s, o);
    }
    s = __shfl(s, p.first, 64) & ~15;
    p.shared = p.count > 1 && s >= kMinShared ? s : 0;
    return p;
}

__device__ __forceinline__ int chunks_of(int n, int ch) { return (n + ch - 1) / ch; }
// Chunk length of a sequence's own positions. A tile of a block of eight row
// blocks costs about two of a single sequence (3.5 us from L2 to 1.1 - 2.1), so
// the sequences behind such a block get chunks twice as long: 32 sequences on a
// prefix of 32K, bf16, 58.5 -> 55.8 us.
__device__ __forceinline__ int own_chunk(const LanePlan& p, int ch) { return p.shared > 0 && p.count > 8 ? 2 * ch : ch; }

// Workgroups (per kv head) of the sequence in this lane at chunk length ch:
// its own chunks, and its block's shared ones in the block's first lane.
__device__ __forceinline__ int items_of(const LanePlan& p, int ch, int lane) {
    return chunks_of(p.own(), own_chunk(p, ch)) + (p.first == lane ? chunks_of(p.shared, ch) : 0);
}

// The call's chunk length, whole tiles (0: the call has more than `most`), and whether it reads so much that
// nothing of it can still be cached when it is read again (half of the 256 MB
// that lie in front of HBM): its tiles are then copied non-temporally. 32
// sequences of up to 32K (1.1 GB) 200 -> 182 us; 8 of up to 8K (75 MB, which a
// loop over three such calls finds cached) 21.6 -> 22.5.
struct Chunk {
    int len;
    bool stream;
};
constexpr int kStreamTiles = 1024;   // of one kv head, 64 KB each

__device__ __forceinline__ Chunk chunk_length(const PagedSeqs& a, const LanePlan& p0, int lane, int bs, int most) {
    long long tiles = 0;
    int streams = 0, longest = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const LanePlan p = b0 == 0 ? p0 : lane_plan(a, b0, lane, bs);
        tiles += wave_sum_int(items_of(p, kTile, lane));
        streams += wave_sum_int((p.own() > 0) + (p.first == lane && p.shared > 0));
        longest = max(longest, wave_max_int(p.len));
    }
    if (__builtin_amdgcn_readfirstlane(static_cast<int>(tiles > most))) return Chunk{0, false};
    // sum of ceil(n / ch) is about tiles / ch + streams / 2, and at most tiles / ch + streams
    const int free = max(a.slots - streams / 2, (a.slots + 1) / 2);
    int ch = static_cast<int>((tiles + free - 1) / free);
    const int sure = streams < a.slots ? static_cast<int>((tiles + a.slots - streams - 1) / (a.slots - streams)) : ch;
    if (a.batch <= 64) {
        while (ch < sure && wave_sum_int(items_of(p0, ch * kTile, lane)) > a.slots) ch += (ch + 15) / 16;
    } else {
        ch = sure;
    }
    ch = max(max(ch, 1), (longest + (a.cap - 2) * kTile - 1) / ((a.cap - 2) * kTile));
    // (the same in every lane; the compiler has to know, for the scalar addresses that follow from it)
    return Chunk{__builtin_amdgcn_readfirstlane(ch * kTile),
                 __builtin_amdgcn_readfirstlane(static_cast<int>(tiles >= kStreamTiles)) != 0};
}

// Workgroup item g: the sequence that holds it (-1: past the last), the item's
// number among the sequence's, its plan (first: as a sequence).
__device__ __forceinline__ int find_item(const PagedSeqs& a, const LanePlan& p0, int ch, int g, int lane, int bs, int& c,
                                         LanePlan& plan) {
    int base = 0;
    c = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const LanePlan p = b0 == 0 ? p0 : lane_plan(a, b0, lane, bs);
        const int mine = items_of(p, ch, lane);
        const int incl = base + wave_inclusive_scan_int(mine);
        const unsigned long long hit = __ballot(incl > g);
        if (hit) {
            const int src = static_cast<int>(__builtin_ctzll(hit));
            c = g - (__builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane(mine, src));
            plan.len = __builtin_amdgcn_readlane(p.len, src);
            plan.shared = __builtin_amdgcn_readlane(p.shared, src);
            plan.first = __builtin_amdgcn_readlane(p.first, src) + b0;
            plan.count = __builtin_amdgcn_readlane(p.count, src);
            return b0 + src;
        }
        base = __builtin_amdgcn_readlane(incl, 63);
    }
    return -1;
}

// ---- pages -----------------------------------------------------------------------

struct PagedKv {
    uint16_t* k;
    uint16_t* v;
    const int32_t* table;   // [batch][cols]
    int num_pages, lg, cols;   // lg: log2 of the page size
};

// 64 consecutive entries of a table row, one a lane, from entry `base`; those
// outside the pool are read as page 0 and marked in `bad` (their positions get
// NaN scores: the row's output is NaN, nothing outside the pool is touched).
struct PageWindow {
    int page, base;
    unsigned long long bad;

    static __device__ __forceinline__ int entry(const int32_t* row, int first, int last, int lane) {
        return row[min(first + lane, last)];
    }
    __device__ __forceinline__ void set(int first, int p, int num_pages) {
        base = first;
        const bool out = p < 0 || p >= num_pages;
        bad = __ballot(out);
        page = out ? 0 : p;
    }
    __device__ __forceinline__ int of(int entry) const { return __builtin_amdgcn_readlane(page, entry - base); }
    __device__ __forceinline__ bool is_bad(int entry) const { return (bad >> (entry - base)) & 1; }
};

// Eight consecutive elements as fp32.
template <int DT>
__device__ __forceinline__ void load8(const void* p, size_t i, float (&x)[8]) {
    if constexpr (DT == 0) {
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i);
        const f32x4_t b = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = a[e];
            x[4 + e] = b[e];
        }
    } else {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
}

// Four consecutive elements as fp32.
template <int DT>
__device__ __forceinline__ void load4(const void* p, size_t i, float* x) {
    if constexpr (DT == 0) {
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = a[e];
    } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
}

// Sum over the four lanes l % 16 + 16 j of an MFMA column, in all of them.
__device__ __forceinline__ float quad_sum(float v) {
    v += swizzle_xor16(v);
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// 1 / sqrt(ss / 256 + eps) on the hardware's reciprocal square root (1 ulp: a
// head's scores scaled by as much; a division and a square root take 30
// instructions more for each row, 0.5 us of a block's start).
__device__ __forceinline__ float inv_rms(float ss, float eps) {
    return __builtin_amdgcn_rsqf(fmaf(ss, 1.0f / 256.0f, eps));
}

// Two floats as NT packed terms of the cache's type, each the rounding of what
// the terms before it leave.
template <int KV_F16, int NT>
__device__ __forceinline__ void split_terms(float x0, float x1, uint32_t (&w)[NT]) {
    // (x as rounded to fp32 from here on: folded into a product before it, the
    // conversion to fp16 would round the exact product, and where that gives
    // another first term than the one subtracted below, the terms are off by an
    // ulp of fp16)
    asm("" : "+v"(x0), "+v"(x1));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (KV_F16) {
            w[t] = pack_f16x2(x0, x1);
            x0 -= f16_to_f32(static_cast<uint16_t>(w[t]));
            x1 -= f16_to_f32(static_cast<uint16_t>(w[t] >> 16));
        } else {
            w[t] = pack_bf16x2(x0, x1);
            x0 -= __uint_as_float(w[t] << 16);
            x1 -= __uint_as_float(w[t] & 0xffff0000u);
        }
    }
}

template <int KV_F16>
__device__ __forceinline__ f32x4_t mfma32(u32x4_t a, u32x4_t b, f32x4_t c) {
    return KV_F16 ? mfma_16x16x32_f16(a, b, c) : mfma_16x16x32_bf16(a, b, c);
}

constexpr float kLazyMax = 8.0f;   // a row's running maximum is raised only past 2^8
template <int KV_F16> constexpr float kShift = KV_F16 ? 7.0f : 0.0f;   // (p <= 2^(8 + 7) < 65504)

struct PagedPartials {
    float* m;   // [slots][8]
    float* d;   // [slots][8]
    float* o;   // [slots][8][256]
    int32_t* count;   // [batch] partials of a sequence, per kv head (not written where the length is 0)
    int cstride;      // slots per (sequence, kv head): the shared chunks first, then its own
};

// ---- partial ------------------------------------------------------------------------
//
// grid 2 x items, 512 threads: kv head u & 1 of item u >> 1. Tiles of 64
// positions of K and V are copied straight into LDS (two stages of 64 KB,
// XOR-swizzled rows), the next one while a tile computes.
//   A block of up to 2 R sequences (R a power of two <= 8) has R row blocks of
//   16 q rows (two sequences x 8 heads): wave w takes row block w % R, and all
//   64 positions where R = 8, otherwise half w / R of them. Per 32 positions a
//   wave reads 16 KB of K and 16 KB of V operands for 32 NT MFMAs.
//   A single sequence's 8 rows: waves 0-3 take 16 positions each, the products
//   of two terms in one MFMA (see single_step).
// Waves beyond these only copy. In both
//   S^T = K Q^T   A = K rows (b128 reads), B = q in registers; a lane's scores
//                 belong to its one q row, positions 16 b + 4 kb + i
//   O^T = V^T P^T A = V^T through transposed reads (positions 4 kb + i of each
//                 16: the order the lane's weights are in), B = P.
// The waves' parts of a row are joined at the end.
// The chunk that ends with the new token norms and rotates k (wave 4), takes v
// (wave 5), writes both to their page and, once the tile that holds the
// position is in LDS, into its rows there; the rows behind them are zeroed
// (what the page holds there may be any bit pattern).
struct PartLds {
    uint16_t tile[2][2][kTile * 256];   // stage, K / V
    float md[8][16][2];                 // per wave and row: m, d
    __attribute__((aligned(16))) float sq[4][16][8];   // sums of squares: row block, row, slice of 32 dims
    __attribute__((aligned(16))) float2 turn[4][64];   // row block, angle of the two sequences: cos, sin
};

// 16-byte piece p of a tile's row r lies at p ^ tile_swz(r): the 16 pieces that 16
// rows have in one column are apart, and so are those of rows 0-3 and 12-15 from
// the next column's of rows 4-11, which b128 reads take together (with 1 in
// place of 9 a third of the LDS cycles were conflicts, now 3-5 %; the times are
// the same).
__device__ __forceinline__ int tile_swz(int r) { return ((r & 7) << 1) ^ (((r >> 3) & 1) * 9); }

template <int IN_DT, int KV_F16, int NT, bool TOKENS>
__global__ __launch_bounds__(512) void gqa_paged_partial_kernel(
    const void* __restrict__ q_gate, const void* __restrict__ k_new, const void* __restrict__ v_new,
    const float* __restrict__ q_norm_w, const float* __restrict__ k_norm_w, RopeFreqs rf, float scale, float eps,
    PagedKv kv, PagedSeqs a, PagedTokens tk, PagedPartials pp) {
    __shared__ __attribute__((aligned(1024))) PartLds L;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int kvh = blockIdx.x & 1;
    int lead, count, p_begin, p_end, slot_c, cut_from;   // cut_from: no row's limit lies before it
    bool has_new = false, stream = false;
    LanePlan plan{};
    if constexpr (TOKENS) {
        int c = static_cast<int>(blockIdx.x >> 1), blk = 0, nc;
        while (c >= (nc = chunks_of(tk.end(blk), tk.ch))) {   // (the grid is their sum)
            c -= nc;
            ++blk;
        }
        lead = tk.per * blk;
        count = min(tk.per, tk.T - lead);
        p_begin = c * tk.ch;
        p_end = min(tk.end(blk), p_begin + tk.ch);
        slot_c = c;
        cut_from = min(p_end, tk.start + lead + 1);
        if (c == 0 && kvh == 0 && static_cast<int>(threadIdx.x) < count) pp.count[lead + threadIdx.x] = nc;
    } else {
        int bs = kBlkSeqs / 2;
        LanePlan p0 = lane_plan(a, 0, lane, bs);
        Chunk chunk = chunk_length(a, p0, lane, bs, a.group ? kPagedSmallTiles * a.slots : INT_MAX);
        if (chunk.len == 0) {   // (uniform)
            bs = kBlkSeqs;
            p0 = lane_plan(a, 0, lane, bs);
            chunk = chunk_length(a, p0, lane, bs, INT_MAX);
        }
        const int ch = chunk.len;
        int item;
        lead = find_item(a, p0, ch, static_cast<int>(blockIdx.x >> 1), lane, bs, item, plan);
        if (lead < 0) return;   // (uniform over the workgroup)
        // the block's shared chunks come first among its first sequence's items
        const int npfx = chunks_of(plan.shared, ch);
        const bool pfx = lead == plan.first && item < npfx;
        int c = pfx ? item : item - (lead == plan.first ? npfx : 0);
        if (pfx && npfx >= 4) {
            // rotated so that c = g modulo 4 (but for the last few): the blocks of a
            // group then read a chunk on the same one of the 8 XCDs, through one L2
            c += (static_cast<int>(blockIdx.x >> 1) - item) & 3;
            if (c >= npfx) c -= npfx;
        }
        count = pfx ? plan.count : 1;
        const int step = pfx ? ch : own_chunk(plan, ch);
        p_begin = (pfx ? 0 : plan.shared) + c * step;
        p_end = min(pfx ? plan.shared : plan.len, p_begin + step);
        has_new = !pfx && p_end == plan.len;
        slot_c = pfx ? c : npfx + c;
        cut_from = p_end;
        stream = chunk.stream && !pfx;   // (a long prefix is read by every block of its group)
    }
    const int ntiles = (p_end - p_begin + kTile - 1) / kTile;
    const int mask = (1 << kv.lg) - 1;
    const int32_t* row = kv.table + (TOKENS ? 0 : static_cast<size_t>(lead) * kv.cols);
    const int last_entry = (p_end - 1) >> kv.lg;
    PageWindow win;

    // the page window to hold tile t
    auto window = [&](int t) {
        if ((min(p_begin + (t + 1) * kTile, p_end) - 1) >> kv.lg > win.base + 63) {
            const int first = (p_begin + t * kTile) >> kv.lg;
            win.set(first, PageWindow::entry(row, first, last_entry, lane), kv.num_pages);
        }
    };
    // K and V of tile t into stage t & 1: in round i wave wv copies rows 16 i + 2 wv,
    // + 1; 16 positions past the chunk's end repeat its last ones (masked;
    // finite, or zeroed behind the new token). Returns bit i if their page is bad.
    auto issue = [&](int t) -> unsigned {
        const int h = lane >> 5;
        const uint32_t lt = 1024u * h + 16u * ((lane & 31) ^ (2 * h) ^ tile_swz(2 * wv & 15));
        unsigned bad = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = min(p_begin + t * kTile + 16 * i, (p_end - 1) & ~15);
            const int entry = p >> kv.lg;
            const size_t at = (((static_cast<size_t>(win.of(entry)) << kv.lg) + (p & mask) + 2 * wv) * 2 + kvh) * 512;
            const char *k = reinterpret_cast<const char*>(kv.k) + at, *v = reinterpret_cast<const char*>(kv.v) + at;
            const uint32_t lk = lds_addr(&L.tile[t & 1][0][(16 * i + 2 * wv) * 256]);
            const uint32_t lv = lds_addr(&L.tile[t & 1][1][(16 * i + 2 * wv) * 256]);
            if (stream) {
                dma16_nt(k, lt, lk);
                dma16_nt(v, lt, lv);
            } else {
                dma16(k, lt, lk);
                dma16(v, lt, lv);
            }
            bad |= (win.is_bad(entry) ? 1u : 0u) << i;
        }
        return bad;
    };
    const int n = lane & 15, kb = lane >> 4;
    const int nrb = (count + 1) / 2;
    const int R = nrb <= 1 ? 1 : nrb <= 2 ? 2 : nrb <= 4 ? 4 : 8;
    const bool single = count == 1;
    const int parts = single ? 4 : R == 8 ? 1 : 2;   // of a tile's positions, one a wave
    const int rb = wv & (R - 1), part = wv / R;
    const bool active = part < parts && rb < nrb;
    const int seq = lead + min(2 * rb + (n >> 3), count - 1);   // of the lane's q row
    // the lane's row sees positions before lim
    const int lim = TOKENS ? min(p_end, tk.start + seq + 1) : p_end;
    auto position_of = [&](int s) { return TOKENS ? tk.start + s : a.positions[s]; };

    // ---- q rows: RMS norm, rotation, terms, by all waves together and handed to
    // the waves that use them through the second stage's LDS, in the operand
    // order of a 16x16x32 product. Lane (n, kb) of wave w takes two pieces of
    // four dims of row n of each row block: for kb = 0 the pairs 4 w + i and
    // 32 + 4 w + i of the rotation, for the others dims 64 + 24 w + 8 (kb - 1) +
    // i and 4 + i (turned by an angle of 0). Everything the start needs from
    // memory is requested together and waited for once, ahead of the first
    // tile's copies, which land while q is prepared.
    u32x4_t q[NT][8];             // a block's: term, step of 32 dims
    u32x4_t qs[(NT + 1) / 2][8];   // a single sequence's: term 2 k in columns l % 16 < 8, term 2 k + 1 in the others
    // dims 4 lane .. + 3 of the new k (wave 4) or v (wave 5); of a short slice's token wv, k and v
    u32x2_t fresh = u32x2_t{0u, 0u}, fresh_v = u32x2_t{0u, 0u};
    const bool append = TOKENS && tk.append() && wv < tk.T && tk.start + wv >= p_begin && tk.start + wv < p_end;
    unsigned bad_next = 0;
    auto prepare = [&](auto rr, auto one) {
        constexpr int RR = decltype(rr)::value;
        constexpr bool ONE = decltype(one)::value;   // a single sequence
        int entry0 = PageWindow::entry(row, p_begin >> kv.lg, last_entry, lane);
        const int dim0 = kb == 0 ? 4 * wv : 56 + 24 * wv + 8 * kb, dim1 = kb == 0 ? 32 + 4 * wv : dim0 + 4;
        float x[RR][8], w[8], kx[4], vx[4], kw[4];
        int page = 0;   // of the appended token
#pragma unroll
        for (int r = 0; r < RR; ++r) {
            const int s = lead + min(2 * r + (n >> 3), count - 1);
            const size_t at = (static_cast<size_t>(s) * 16 + kvh * 8 + (n & 7)) * 512;
            load4<IN_DT>(q_gate, at + dim0, &x[r][0]);
            load4<IN_DT>(q_gate, at + dim1, &x[r][4]);
        }
        load4<0>(q_norm_w, dim0, &w[0]);
        load4<0>(q_norm_w, dim1, &w[4]);
        if constexpr (ONE && !TOKENS) {   // (waves other than 4 and 5 do not use them)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                kx[i] = elem<IN_DT>::load(wv == 5 ? v_new : k_new, (static_cast<size_t>(lead) * 2 + kvh) * 256 + 4 * lane + i);
        }
        if constexpr (TOKENS) {
            if (append) {
                const size_t from = (static_cast<size_t>(wv) * 2 + kvh) * 256 + 4 * lane;
                load4<IN_DT>(k_new, from, kx);
                load4<IN_DT>(v_new, from, vx);
                load4<0>(k_norm_w, 4 * lane, kw);
                page = row[(tk.start + wv) >> kv.lg];
#pragma unroll
                for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(kx[i]), "+v"(vx[i]), "+v"(kw[i]));
                asm volatile("" : "+v"(page));
            }
        }
        int pos_a = position_of(lead + min(2 * min(wv, RR - 1) + (lane >> 5), count - 1));
        float freq = rf.f[lane & 31];   // (a load: the arguments lie in memory)
        // (consumed here, so that no load is moved behind the copies, whose
        // requests a later wait for it would wait for too)
        asm volatile("" : "+v"(entry0), "+v"(pos_a), "+v"(freq));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            asm volatile("" : "+v"(w[e]));
#pragma unroll
            for (int r = 0; r < RR; ++r) asm volatile("" : "+v"(x[r][e]));
        }
        if constexpr (ONE && !TOKENS) asm volatile("" : "+v"(kx[0]), "+v"(kx[1]), "+v"(kx[2]), "+v"(kx[3]));
        win.set(p_begin >> kv.lg, entry0, kv.num_pages);
        bad_next = issue(0);
        // cos, sin of angle l % 32 of row block wv's sequence l / 32
        if (wv < RR) {
            float s, c2;
            sincosf(static_cast<float>(pos_a) * freq, &s, &c2);
            L.turn[wv][lane] = make_float2(c2, s);
        }
#pragma unroll
        for (int r = 0; r < RR; ++r) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[r][e] * x[r][e];
            ss = quad_sum(ss);
            if (kb == 0) L.sq[r][n][wv] = ss;
        }
        __syncthreads();
        constexpr int kAtOnce = RR < 8 / NT ? RR : 8 / NT;   // row blocks that 64 KB hold
        u32x4_t* const hand = reinterpret_cast<u32x4_t*>(L.tile[1]);
        // piece of four dims d ..: step d / 32, lane 16 (d % 32 / 8) + n, half d % 8 / 4
        auto piece = [&](int d) { return 2 * (64 * (d >> 5) + 16 * ((d >> 3) & 3) + n) + ((d >> 2) & 1); };
        u32x2_t* const half0 = reinterpret_cast<u32x2_t*>(hand) + piece(dim0);
        u32x2_t* const half1 = reinterpret_cast<u32x2_t*>(hand) + piece(dim1);
#pragma unroll
        for (int r0 = 0; r0 < RR; r0 += kAtOnce) {
#pragma unroll
            for (int r = r0; r < r0 + kAtOnce; ++r) {
                const f32x4_t a0 = *reinterpret_cast<const f32x4_t*>(&L.sq[r][n][0]);
                const f32x4_t a1 = *reinterpret_cast<const f32x4_t*>(&L.sq[r][n][4]);
                const float ss = ((a0[0] + a0[1]) + (a0[2] + a0[3])) + ((a1[0] + a1[1]) + (a1[2] + a1[3]));
                const float inv = inv_rms(ss, eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[r][e] = x[r][e] * inv * w[e];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float2 cs = L.turn[r][32 * (n >> 3) + 4 * wv + i];
                    if (kb != 0) cs = make_float2(1.0f, 0.0f);
                    const float lo = x[r][i], hi = x[r][4 + i];
                    x[r][i] = lo * cs.x - hi * cs.y;
                    x[r][4 + i] = hi * cs.x + lo * cs.y;
                }
                uint32_t t[4][NT];
#pragma unroll
                for (int i = 0; i < 4; ++i) split_terms<KV_F16, NT>(x[r][2 * i], x[r][2 * i + 1], t[i]);
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    half0[((r - r0) * NT + k) * 1024] = u32x2_t{t[0][k], t[1][k]};
                    half1[((r - r0) * NT + k) * 1024] = u32x2_t{t[2][k], t[3][k]};
                }
            }
            __syncthreads();
            if constexpr (ONE) {
                const int from = 16 * kb + (n & 7);
#pragma unroll
                for (int k = 0; k < (NT + 1) / 2; ++k)
#pragma unroll
                    for (int jj = 0; jj < 8; ++jj) {
                        const u32x4_t v = hand[(min(2 * k + (n >> 3), NT - 1) * 8 + jj) * 64 + from];
                        qs[k][jj] = 2 * k + (n >> 3) < NT ? v : u32x4_t{0u, 0u, 0u, 0u};
                    }
            } else if (active && rb >= r0 && rb < r0 + kAtOnce) {
#pragma unroll
                for (int k = 0; k < NT; ++k)
#pragma unroll
                    for (int jj = 0; jj < 8; ++jj) q[k][jj] = hand[(((rb - r0) * NT + k) * 8 + jj) * 64 + lane];
            }
            if (r0 + kAtOnce < RR) __syncthreads();
        }
        if constexpr (TOKENS) {
            if (append) {   // (the angles are those of the token's q row)
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) ss += kx[i] * kx[i];
                const float inv = 1.0f / sqrtf(group_sum<64>(ss) / 256.0f + eps);
#pragma unroll
                for (int i = 0; i < 4; ++i) kx[i] = kx[i] * inv * kw[i];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float up = __shfl_down(kx[i], 8, 64), dn = __shfl_up(kx[i], 8, 64);
                    const int d = 4 * lane + i;
                    const float2 cs = L.turn[wv >> 1][32 * (wv & 1) + (d & 31)];
                    if (d < 64) kx[i] = d < 32 ? kx[i] * cs.x - up * cs.y : kx[i] * cs.x + dn * cs.y;
                }
                uint32_t w0[1], w1[1], w2[1], w3[1];
                split_terms<KV_F16, 1>(kx[0], kx[1], w0);
                split_terms<KV_F16, 1>(kx[2], kx[3], w1);
                split_terms<KV_F16, 1>(vx[0], vx[1], w2);
                split_terms<KV_F16, 1>(vx[2], vx[3], w3);
                fresh = u32x2_t{w0[0], w1[0]};
                fresh_v = u32x2_t{w2[0], w3[0]};
                if (page >= 0 && page < kv.num_pages) {
                    const size_t off = ((static_cast<size_t>(page) << kv.lg) + ((tk.start + wv) & mask)) * 512 + kvh * 256 + 4 * lane;
                    *reinterpret_cast<u32x2_t*>(kv.k + off) = fresh;
                    *reinterpret_cast<u32x2_t*>(kv.v + off) = fresh_v;
                }
            }
        }
        if constexpr (ONE && !TOKENS) {
            if (has_new && (wv == 4 || wv == 5)) {
                // dims 4 lane .. + 3; the rotation's partner of dim d < 32 is d + 32, 8 lanes on
                if (wv == 4) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) ss += kx[i] * kx[i];
                    const float inv = 1.0f / sqrtf(group_sum<64>(ss) / 256.0f + eps);
#pragma unroll
                    for (int i = 0; i < 4; ++i) kx[i] = kx[i] * inv * k_norm_w[4 * lane + i];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float up = __shfl_down(kx[i], 8, 64), dn = __shfl_up(kx[i], 8, 64);
                        const int d = 4 * lane + i;
                        const float2 cs = L.turn[0][d & 31];
                        if (d < 64) kx[i] = d < 32 ? kx[i] * cs.x - up * cs.y : kx[i] * cs.x + dn * cs.y;
                    }
                }
                uint32_t w0[1], w1[1];
                split_terms<KV_F16, 1>(kx[0], kx[1], w0);
                split_terms<KV_F16, 1>(kx[2], kx[3], w1);
                fresh = u32x2_t{w0[0], w1[0]};
                page = row[last_entry];   // (the chunk ends with the new token)
                if (page >= 0 && page < kv.num_pages) {   // (dropped where the page lies outside the pool)
                    const size_t off = ((static_cast<size_t>(page) << kv.lg) + ((plan.len - 1) & mask)) * 512 + kvh * 256 + 4 * lane;
                    *reinterpret_cast<u32x2_t*>((wv == 4 ? kv.k : kv.v) + off) = fresh;
                }
            }
        }
    };
    // Eight row blocks: each wave its own, without the hand-over.
    auto prepare_own = [&]() {
        int entry0 = PageWindow::entry(row, p_begin >> kv.lg, last_entry, lane);
        float x[8][8];
        const size_t qbase = (static_cast<size_t>(seq) * 16 + kvh * 8 + (n & 7)) * 512 + 8 * kb;
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) load8<IN_DT>(q_gate, qbase + 32 * jj, x[jj]);
        int pos_a = position_of(lead + min(2 * rb + (lane >> 5), count - 1));
        float freq = rf.f[lane & 31], w[8][8];
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) load8<0>(q_norm_w, 32 * jj + 8 * kb, w[jj]);
        asm volatile("" : "+v"(entry0), "+v"(pos_a), "+v"(freq));
#pragma unroll
        for (int jj = 0; jj < 8; ++jj)
#pragma unroll
            for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(x[jj][e]), "+v"(w[jj][e]));
        win.set(p_begin >> kv.lg, entry0, kv.num_pages);
        bad_next = issue(0);
        float cl, sl, cs[8], sn[8], ss = 0.0f;   // lane l: angle l % 32 of the row block's sequence l / 32
        sincosf(static_cast<float>(pos_a) * freq, &sl, &cl);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int from = 32 * (n >> 3) + 8 * kb + e;
            cs[e] = __shfl(cl, from, 64);
            sn[e] = __shfl(sl, from, 64);
        }
#pragma unroll
        for (int jj = 0; jj < 8; ++jj)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ss += x[jj][e] * x[jj][e];
                x[jj][e] *= w[jj][e];   // (here, so that w's registers are free before q's are filled)
                asm volatile("" : "+v"(x[jj][e]));
            }
        const float inv = inv_rms(quad_sum(ss), eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float lo = x[0][e] * inv, hi = x[1][e] * inv;
            x[0][e] = lo * cs[e] - hi * sn[e];
            x[1][e] = hi * cs[e] + lo * sn[e];
        }
#pragma unroll
        for (int jj = 0; jj < 8; ++jj)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t t[NT];
                const float f = jj < 2 ? 1.0f : inv;
                split_terms<KV_F16, NT>(x[jj][2 * i] * f, x[jj][2 * i + 1] * f, t);
#pragma unroll
                for (int k = 0; k < NT; ++k) q[k][jj][i] = t[k];
            }
    };
    if (has_new && kvh == 0 && threadIdx.x == 0) pp.count[lead] = slot_c + 1;   // the sequence's last partial

    float m_run = -INFINITY, d_run = 0.0f;
    f32x4_t oacc[16];   // O^T: dims 16 dt + 4 kb + i of the lane's row
    auto clear = [&] {
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) oacc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    };
    const float sc = scale * 1.44269504088896341f;
    const uint32_t kaddr = 512u * n + 16u * (kb ^ tile_swz(n));
    const int vr = 4 * kb + (n >> 2);
    const uint32_t vaddr = 512u * vr + 16u * (((n >> 1) & 1) ^ tile_swz(vr)) + 8u * (n & 1);

    // a ^ x next to its use: hoisted out of the loop, the operands' 24 addresses would not fit the registers
    auto at_xor = [](uint32_t a, uint32_t x) {
        uint32_t r;
        asm volatile("v_xor_b32 %0, %1, %2" : "=v"(r) : "s"(x), "v"(a));
        return r;
    };
    auto lds128 = [](uint32_t at) {
        return *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(static_cast<uintptr_t>(at));
    };
    auto lds_tr = [](uint32_t at) {
        typedef short s16x4_l __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                               (s16x4_l __attribute__((address_space(3)))*)(static_cast<uintptr_t>(at))));
    };
    // the running maximum of the lane's row against this tile's, in all four lanes of the row
    auto raise = [&](float tm) {
        tm = fmaxf(tm, swizzle_xor16(tm));
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(tm), __float_as_uint(tm), false, false);
        tm = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
        if (__any(tm > m_run + kLazyMax)) {
            const float m_new = tm > m_run + kLazyMax ? tm : m_run;
            const float alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            d_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < 16; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) oacc[dt][i] *= alpha;
        }
    };
    // what the weights' exponents count from; a token's row that sees none of the positions so far keeps weights of 0
    auto base_of = [&] { return TOKENS && m_run == -INFINITY ? 0.0f : m_run - kShift<KV_F16>; };
    // 32 positions (s0 ..) of a block's row block; sub: which half of the tile
    auto block_step = [&](uint32_t kt, uint32_t vt, int s0, int sub, unsigned bad) {
        const uint32_t ka = kt + 16384u * sub + kaddr, va0 = vt + 16384u * sub + vaddr;   // (tiles lie at multiples of 32 KB)
        f32x4_t s[2][NT];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < NT; ++k) s[b][k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        // operands two steps ahead of their products (further, and their registers spill)
        u32x4_t kf[3][2];
        auto k_read = [&](int jj) {
            const uint32_t at = at_xor(ka, 64u * jj);
            kf[jj % 3][0] = lds128(at);
            kf[jj % 3][1] = lds128(at + 8192u);
        };
        k_read(0);
        k_read(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) {
            if (jj + 2 < 8) k_read(jj + 2);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int k = 0; k < NT; ++k) s[b][k] = mfma32<KV_F16>(kf[jj % 3][b], q[k][jj], s[b][k]);
            __builtin_amdgcn_sched_barrier(0);
        }
        u32x2_t vf[4][2];
        auto v_read = [&](int dt) {
            const uint32_t at = at_xor(va0, 32u * dt);
            vf[dt % 4][0] = lds_tr(at);
            vf[dt % 4][1] = lds_tr(at + 8192u);
        };
#pragma unroll
        for (int dt = 0; dt < 3; ++dt) v_read(dt);
        float x[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = s[b][0][i];
#pragma unroll
                for (int k = 1; k < NT; ++k) v += s[b][k][i];
                x[b][i] = v * sc;
            }
        if (s0 + 32 > cut_from || (bad >> (2 * sub) & 3)) {   // (uniform)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[b][i] = s0 + 16 * b + 4 * kb + i >= lim ? -INFINITY
                              : (bad >> (2 * sub + b)) & 1     ? __builtin_nanf("")
                                                               : x[b][i];
        }
        raise(fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                    fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3]))));
        const float mb = base_of();
        u32x4_t pw[NT];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float e0 = __builtin_amdgcn_exp2f(x[b][i] - mb), e1 = __builtin_amdgcn_exp2f(x[b][i + 1] - mb);
                d_run += e0 + e1;
                uint32_t w[NT];
                split_terms<KV_F16, NT>(e0, e1, w);
#pragma unroll
                for (int k = 0; k < NT; ++k) pw[k][2 * b + i / 2] = w[k];
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) {
            if (dt + 3 < 16) v_read(dt + 3);
            const u32x2_t v0 = vf[dt % 4][0], v1 = vf[dt % 4][1];
#pragma unroll
            for (int k = 0; k < NT; ++k) oacc[dt] = mfma32<KV_F16>(u32x4_t{v0[0], v0[1], v1[0], v1[1]}, pw[k], oacc[dt]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // 16 positions (s0 ..) of a single sequence, whose 8 heads leave 8 columns
    // free: q's second term scores in those, lanes n and n ^ 8 add up. The
    // weights' first two terms share one product along its 32 positions (V's 16
    // rows twice), a third takes the free columns.
    auto single_step = [&](uint32_t kt, uint32_t vt, int s0, bool bad) {
        const uint32_t ka = kt + 8192u * part + kaddr, va0 = vt + 8192u * part + vaddr;
        f32x4_t s[(NT + 1) / 2];
#pragma unroll
        for (int k = 0; k < (NT + 1) / 2; ++k) s[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) {
            const u32x4_t kf = lds128(at_xor(ka, 64u * jj));
#pragma unroll
            for (int k = 0; k < (NT + 1) / 2; ++k) s[k] = mfma32<KV_F16>(kf, qs[k][jj], s[k]);
        }
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = s[0][i];
            if constexpr (NT == 3) v += s[1][i];
            x[i] = (v + dpp_mov<0x128>(v)) * sc;   // row_ror:8
        }
        if (s0 + 16 > p_end || bad) {   // (uniform)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = s0 + 4 * kb + i >= p_end ? -INFINITY : bad ? __builtin_nanf("") : x[i];
        }
        raise(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        const float mb = base_of();
        uint32_t w0[NT], w1[NT];
        const float e0 = __builtin_amdgcn_exp2f(x[0] - mb), e1 = __builtin_amdgcn_exp2f(x[1] - mb);
        const float e2 = __builtin_amdgcn_exp2f(x[2] - mb), e3 = __builtin_amdgcn_exp2f(x[3] - mb);
        d_run += (e0 + e1) + (e2 + e3);
        split_terms<KV_F16, NT>(e0, e1, w0);
        split_terms<KV_F16, NT>(e2, e3, w1);
        u32x4_t pw = u32x4_t{w0[0], w1[0], w0[1], w1[1]};
        if (n >= 8) pw = NT == 3 ? u32x4_t{w0[NT - 1], w1[NT - 1], 0u, 0u} : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) {
            const u32x2_t v = lds_tr(at_xor(va0, 32u * dt));
            oacc[dt] = mfma32<KV_F16>(u32x4_t{v[0], v[1], v[0], v[1]}, pw, oacc[dt]);
        }
    };

    auto arrive = [&](int t) {   // tile t is in LDS, and the other stage's readers are done
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    // four dims of row r of tile t: 4 lane .. + 3 of K (0) or V (1)
    auto tile_at = [&](int t, int which, int r) {
        return reinterpret_cast<u32x2_t*>(&L.tile[t & 1][which][r * 256 + 8 * ((lane >> 1) ^ tile_swz(r)) + 4 * (lane & 1)]);
    };
    // a short slice's tokens into their rows of tile t, over what their pages held before
    auto put_tokens = [&](int t) {
        const int t0 = p_begin + t * kTile;
        if (!TOKENS || !tk.append() || t0 + kTile <= tk.start) return;   // (uniform)
        const int r = tk.start + wv - t0;
        if (append && r >= 0 && r < kTile) {
            *tile_at(t, 0, r) = fresh;
            *tile_at(t, 1, r) = fresh_v;
        }
        __syncthreads();
    };
    // V's rows from .. to - 1 of the last tile, behind the last position (the page may hold any bit pattern there)
    auto clear_behind = [&](int t, int from, int to) {
        for (int z = from + wv; z < to; z += 8) *tile_at(t, 1, z) = u32x2_t{0u, 0u};
        __syncthreads();
    };
    // (a page outside the pool is read as page 0: rows that do not see it give V's rows weights of 0)
    auto clear_bad = [&](int t, unsigned bad) {
        if (!TOKENS || bad == 0) return;
        for (int z = wv; z < kTile; z += 8)
            if ((bad >> (z >> 4)) & 1) *tile_at(t, 1, z) = u32x2_t{0u, 0u};
        __syncthreads();
    };
    if (single) {
        prepare(std::integral_constant<int, 1>{}, std::true_type{});
        clear();
        for (int t = 0; t < ntiles; ++t) {
            arrive(t);
            const unsigned bad = bad_next;
            const int t0 = p_begin + t * kTile;
            put_tokens(t);
            if (t + 1 < ntiles) {
                window(t + 1);
                bad_next = issue(t + 1);
            } else if (TOKENS || has_new) {
                const int r = p_end - t0;
                if (!TOKENS && (wv == 4 || wv == 5)) *tile_at(t, wv - 4, r - 1) = fresh;   // the new token's row
                clear_behind(t, r, (r + 15) & ~15);
            }
            clear_bad(t, bad);
            if (active && t0 + 16 * part < p_end)
                single_step(lds_addr(L.tile[t & 1][0]), lds_addr(L.tile[t & 1][1]), t0 + 16 * part, (bad >> part) & 1);
        }
    } else {
        if (R == 1) prepare(std::integral_constant<int, 1>{}, std::false_type{});
        else if (R == 2) prepare(std::integral_constant<int, 2>{}, std::false_type{});
        else if (R == 4) prepare(std::integral_constant<int, 4>{}, std::false_type{});
        else prepare_own();
        clear();
        for (int t = 0; t < ntiles; ++t) {
            arrive(t);
            const unsigned bad = bad_next;
            const int t0 = p_begin + t * kTile;
            put_tokens(t);
            if (t + 1 < ntiles) {
                window(t + 1);
                bad_next = issue(t + 1);
            } else if (TOKENS) clear_behind(t, p_end - t0, (p_end - t0 + 31) & ~31);
            clear_bad(t, bad);
            if (!active) continue;
#pragma unroll 1
            for (int sub = parts == 2 ? part : 0; sub < (parts == 2 ? part + 1 : 2); ++sub)
                if (t0 + 32 * sub < p_end)
                    block_step(lds_addr(L.tile[t & 1][0]), lds_addr(L.tile[t & 1][1]), t0 + 32 * sub, sub, bad);
        }
    }
    d_run = quad_sum(d_run);
    // ---- the parts of a row joined through LDS, in place of the tiles
    f32x4_t* const hand = reinterpret_cast<f32x4_t*>(L.tile);
    auto slot_of = [&](int s) { return (static_cast<size_t>(s) * 2 + kvh) * pp.cstride + slot_c; };
    if (single) {
        // 8 rows, each by one wave whole (256 dims by 64 lanes): piece (dt, kb) of
        // row n lies at 64 dt + 16 kb + (n ^ dt) of its part's 16 KB, so that
        // neither side meets a bank twice
        __syncthreads();
        if (active) {
            if (NT == 3) {
#pragma unroll
                for (int dt = 0; dt < 16; ++dt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) oacc[dt][i] += dpp_mov<0x128>(oacc[dt][i]);
            }
#pragma unroll
            for (int dt = 0; dt < 16; ++dt)
                if (n < 8) hand[1024 * wv + 64 * dt + 16 * kb + (n ^ dt)] = oacc[dt];
            if (kb == 0) {
                L.md[wv][n][0] = m_run;
                L.md[wv][n][1] = d_run;
            }
        }
        __syncthreads();
        const int piece = 64 * (lane >> 2) + 16 * (lane & 3) + (wv ^ (lane >> 2));
        float mk[4], m = -INFINITY, d = 0.0f;
        f32x4_t v[4], o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            mk[k] = L.md[k][wv][0];
            v[k] = hand[1024 * k + piece];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) m = fmaxf(m, mk[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            // (a part without any position, or whose scores are all NaN, has maximum -inf)
            const float f = mk[k] == m ? 1.0f : __builtin_amdgcn_exp2f(mk[k] - m);
            d += f * L.md[k][wv][1];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += f * v[k][i];
        }
        const size_t at = slot_of(lead) * 8 + wv;
        if (lane == 0) {
            pp.m[at] = m - kShift<KV_F16>;
            pp.d[at] = d;
        }
        *reinterpret_cast<f32x4_t*>(pp.o + at * 256 + 4 * lane) = o;
        return;
    }
    // a block's rows: two parts each finish half of the dims with the other's
    // sums (dim tiles 8 part ..); without parts a wave has the whole row
    const bool mine = active && 2 * rb + (n >> 3) < count;
    const size_t at = slot_of(seq) * 8 + (n & 7);
    float* const po = pp.o + at * 256 + 4 * kb;
    auto store_md = [&](float m, float d) {
        if (mine && kb == 0) {
            pp.m[at] = m - kShift<KV_F16>;
            pp.d[at] = d;
        }
    };
    if (parts == 1) {
        store_md(m_run, d_run);
        if (mine) {
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) *reinterpret_cast<f32x4_t*>(po + 16 * dt) = oacc[dt];
        }
        return;
    }
    __syncthreads();
    auto exchange = [&](auto pc) {
        constexpr int P = decltype(pc)::value;
        if (active) {
#pragma unroll
            for (int c = 0; c < 8; ++c) hand[512 * wv + 64 * c + lane] = oacc[8 * (1 - P) + c];
            if (kb == 0) {
                L.md[wv][n][0] = m_run;
                L.md[wv][n][1] = d_run;
            }
        }
        __syncthreads();
        if (!mine) return;
        const int partner = P == 0 ? wv + R : wv - R;
        const float m1 = L.md[partner][n][0], m = fmaxf(m_run, m1);
        // (a part without any position, or whose scores are all NaN, has maximum -inf)
        const float f0 = m_run == m ? 1.0f : __builtin_amdgcn_exp2f(m_run - m);
        const float f1 = m1 == m ? 1.0f : __builtin_amdgcn_exp2f(m1 - m);
        if (P == 0) store_md(m, d_run * f0 + L.md[partner][n][1] * f1);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const f32x4_t v = hand[512 * partner + 64 * c + lane];
            f32x4_t o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = oacc[8 * P + c][i] * f0 + v[i] * f1;
            *reinterpret_cast<f32x4_t*>(po + 16 * (8 * P + c)) = o;
        }
    };
    if (part == 1) exchange(std::integral_constant<int, 1>{});
    else exchange(std::integral_constant<int, 0>{});
}

// ---- combine ----------------------------------------------------------------------------
//
// grid (16 q heads x DS dim blocks, batch), 512 threads, 256 / DS dims a
// workgroup: chunk weights one thread a chunk; 8 DS streams of float4 lanes,
// stream s adding chunks s, s + 8 DS, ... in order, then the streams in a fixed
// order (results do not depend on timing). The (m, d) of every slot, the
// gate, and the number of partials (which the partial launch leaves, so that
// the split is not derived again) are requested together, and a stream's first
// four rows before the weights; every load is unconditional, its index clamped.
template <int IN_DT, int OUT_DT, int DS>
__global__ __launch_bounds__(512) void gqa_paged_combine_kernel(const void* __restrict__ q_gate,
                                                                const int32_t* __restrict__ positions, int max_ctx,
                                                                PagedPartials pp, void* __restrict__ out) {
    constexpr int kDims = 256 / DS, kLanes = 64 / DS, kStreams = 8 * DS, kRound = 4;
    __shared__ float es[kGqaMaxChunks], red[16];
    __shared__ __attribute__((aligned(16))) float osum[kStreams][kDims];
    const int h = blockIdx.x / DS, dblk = blockIdx.x % DS, seq = blockIdx.y, t = threadIdx.x;
    const int lane = t & 63, wave = t >> 6;
    const int kvh = h >> 3, hl = h & 7, d0 = dblk * kDims;
    const size_t qi = static_cast<size_t>(seq) * 16 + h;
    const size_t base = (static_cast<size_t>(seq) * 2 + kvh) * pp.cstride;
    const int ts = min(t, pp.cstride - 1);
    const float m_slot = pp.m[(base + ts) * 8 + hl];
    const float d_slot = pp.d[(base + ts) * 8 + hl];
    const float gate = elem<IN_DT>::load(q_gate, qi * 512 + 256 + d0 + min(t, kDims - 1));
    const int pos = positions ? positions[seq] : 0, listed = pp.count[seq];
    if (pos < 0 || pos >= max_ctx) {   // (uniform over the workgroup)
        if (t < kDims) elem<OUT_DT>::store(out, qi * 256 + d0 + t, __builtin_nanf(""));
        return;
    }
    const int nc = min(listed, pp.cstride);
    const int sid = wave * DS + lane / kLanes, f = lane % kLanes;
    const float4* pr = reinterpret_cast<const float4*>(pp.o + (base * 8 + hl) * 256 + d0) + f;
    float4 v[kRound];
#pragma unroll
    for (int u = 0; u < kRound; ++u) v[u] = pr[static_cast<size_t>(min(sid + kStreams * u, nc - 1)) * 512];
    const float m = t < nc ? m_slot : -INFINITY;
    const float d = t < nc ? d_slot : 0.0f;
    const float wmax = group_max<64>(m);
    if (lane == 0) red[wave] = wmax;
    __syncthreads();
    float M = red[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) M = fmaxf(M, red[w]);
    const float e = t < nc ? __builtin_amdgcn_exp2f(m - M) : 0.0f;
    if (t < kGqaMaxChunks) es[t] = e;
    const float wd = group_sum<64>(d * e);
    if (lane == 0) red[8 + wave] = wd;
    __syncthreads();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = sid; c < nc; c += kRound * kStreams) {
        float4 cur[kRound];
#pragma unroll
        for (int u = 0; u < kRound; ++u) cur[u] = v[u];
#pragma unroll
        for (int u = 0; u < kRound; ++u)
            v[u] = pr[static_cast<size_t>(min(c + kStreams * (kRound + u), nc - 1)) * 512];
#pragma unroll
        for (int u = 0; u < kRound; ++u) {
            const int cc = c + kStreams * u;
            const float w = es[min(cc, kGqaMaxChunks - 1)];
            if (cc < nc) {
                acc.x += cur[u].x * w; acc.y += cur[u].y * w; acc.z += cur[u].z * w; acc.w += cur[u].w * w;
            }
        }
    }
    reinterpret_cast<float4*>(osum[sid])[f] = acc;
    __syncthreads();
    if (t < kDims) {
        float D = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) D += red[8 + w];
#pragma unroll
        for (int s2 = 0; s2 < kStreams; ++s2) O += osum[s2][t];
        elem<OUT_DT>::store(out, qi * 256 + d0 + t, (O / D) * sigmoid(gate));
    }
}

// ---- append ------------------------------------------------------------------------------
//
// A prompt slice's k (RMS norm, rotation) and v rows into their pages: one
// wave per (token, kv head), lane l dims 4 l .. + 3. Rows whose page lies
// outside the pool are dropped.
template <int IN_DT, int KV_F16>
__global__ __launch_bounds__(256) void gqa_paged_append_kernel(const void* __restrict__ k, const void* __restrict__ v,
                                                               const float* __restrict__ k_norm_w, RopeFreqs rf,
                                                               float eps, PagedKv kv, int start, int T) {
    const int lane = threadIdx.x & 63, unit = static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (unit >= 2 * T) return;
    const int pos = start + (unit >> 1);
    const int page = kv.table[pos >> kv.lg];
    float x[4], y[4], ss = 0.0f;
    load4<IN_DT>(k, static_cast<size_t>(unit) * 256 + 4 * lane, x);
    load4<IN_DT>(v, static_cast<size_t>(unit) * 256 + 4 * lane, y);
    float c, s;
    sincosf(static_cast<float>(pos) * rf.f[lane & 31], &s, &c);
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += x[i] * x[i];
    const float inv = 1.0f / sqrtf(group_sum<64>(ss) / 256.0f + eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = x[i] * inv * k_norm_w[4 * lane + i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // the partner of dim d < 32 is d + 32, 8 lanes on
        const float up = __shfl_down(x[i], 8, 64), dn = __shfl_up(x[i], 8, 64);
        const float ci = __shfl(c, (4 * lane + i) & 31, 64), si = __shfl(s, (4 * lane + i) & 31, 64);
        const int d = 4 * lane + i;
        if (d < 64) x[i] = d < 32 ? x[i] * ci - up * si : x[i] * ci + dn * si;
    }
    if (page < 0 || page >= kv.num_pages) return;
    uint32_t k0[1], k1[1], v0[1], v1[1];
    split_terms<KV_F16, 1>(x[0], x[1], k0);
    split_terms<KV_F16, 1>(x[2], x[3], k1);
    split_terms<KV_F16, 1>(y[0], y[1], v0);
    split_terms<KV_F16, 1>(y[2], y[3], v1);
    const size_t off = (((static_cast<size_t>(page) << kv.lg) + (pos & ((1 << kv.lg) - 1))) * 2 + (unit & 1)) * 256 + 4 * lane;
    *reinterpret_cast<u32x2_t*>(kv.k + off) = u32x2_t{k0[0], k1[0]};
    *reinterpret_cast<u32x2_t*>(kv.v + off) = u32x2_t{v0[0], v1[0]};
}

// ---- launch ---------------------------------------------------------------------------

static PagedKv paged_kv(const qff_kv_pages* kv) {
    return PagedKv{static_cast<uint16_t*>(kv->k), static_cast<uint16_t*>(kv->v), kv->table, kv->num_pages,
                   __builtin_ctz(static_cast<unsigned>(kv->page_size)), kv->table_cols};
}

// Terms of q and of the weights.
static int paged_terms(bool kv_f16, bool out16) { return kv_f16 || out16 ? 2 : 3; }

// The partial launch (a batch's step, or a slice's tokens) and the combine of
// `rows` sequences or tokens.
static void launch_partials(qff_ctx* ctx, hipStream_t stream, const qff_gqa_params* p, const void* q_gate,
                            const void* k_new, const void* v_new, qff_dtype in_dtype, const PagedKv& pk,
                            const PagedSeqs* a, const PagedTokens& tk, const PagedPartials& pp, int grid, void* out,
                            qff_dtype out_dtype, int rows) {
    const RopeFreqs rf = rope_freqs(p->rope_theta);
    const bool f16 = p->kv_f16 != 0, in16 = in_dtype == QFF_BF16, out16 = out_dtype == QFF_BF16;
    {
        ProfScope prof(ctx, stream, a ? "gqa_paged_partial" : "gqa_paged_prefill_partial");
        const PagedSeqs none{};
#define QFF_PART1(I, F, N, TOK)                                                                                     \
    gqa_paged_partial_kernel<I, F, N, TOK><<<grid, 512, 0, stream>>>(q_gate, k_new, v_new, p->q_norm_w, p->k_norm_w, rf, \
                                                                     p->scale, p->eps, pk, a ? *a : none, tk, pp)
#define QFF_PART(I, F, N) \
    if (a) QFF_PART1(I, F, N, false); else QFF_PART1(I, F, N, true)
        if (f16) {
            if (in16) { QFF_PART(1, 1, 2); } else { QFF_PART(0, 1, 2); }
        } else if (paged_terms(f16, out16) == 2) {
            if (in16) { QFF_PART(1, 0, 2); } else { QFF_PART(0, 0, 2); }
        } else {
            if (in16) { QFF_PART(1, 0, 3); } else { QFF_PART(0, 0, 3); }
        }
#undef QFF_PART
#undef QFF_PART1
    }
    ProfScope prof(ctx, stream, a ? "gqa_paged_combine" : "gqa_paged_prefill_combine");
    const int ds = rows <= 8 ? 4 : 1;   // few rows: each head's dims split over four workgroups
    const dim3 cgrid(16 * ds, rows);
    const int32_t* positions = a ? a->positions : nullptr;
    const int max_ctx = a ? a->max_ctx : 1;
#define QFF_COMB(I, O)                                                                                             \
    if (ds == 4) gqa_paged_combine_kernel<I, O, 4><<<cgrid, 512, 0, stream>>>(q_gate, positions, max_ctx, pp, out); \
    else gqa_paged_combine_kernel<I, O, 1><<<cgrid, 512, 0, stream>>>(q_gate, positions, max_ctx, pp, out)
    if (in16) {
        if (out16) { QFF_COMB(1, 1); } else { QFF_COMB(1, 0); }
    } else {
        if (out16) { QFF_COMB(0, 1); } else { QFF_COMB(0, 0); }
    }
#undef QFF_COMB
}

hipError_t launch_gqa_decode_paged(qff_ctx* ctx, hipStream_t stream, const qff_gqa_params* p, const void* q_gate,
                                   const void* k_new, const void* v_new, qff_dtype in_dtype, const qff_kv_pages* kv,
                                   const int32_t* positions, const int32_t* group, const int32_t* shared_len,
                                   void* out, qff_dtype out_dtype, int batch) {
    const PagedKv pk = paged_kv(kv);
    const int cap = gqa_chunk_cap(ctx->cfg, batch);
    const PagedSeqs a{positions, group, shared_len, batch, kv->table_cols << pk.lg, ctx->num_cu / 2, cap};
    const PagedPartials pp{ctx->gqa_m, ctx->gqa_d, ctx->gqa_o, ctx->gqa_nc, cap};
    // a round of workgroups, and one more for each stream of positions (a
    // sequence's own, a block's shared ones) that rounding up can add
    const int grid = 2 * (a.slots + batch + (group ? batch / 2 : 0));
    launch_partials(ctx, stream, p, q_gate, k_new, v_new, in_dtype, pk, &a, PagedTokens{}, pp, grid, out, out_dtype, batch);
    return hipGetLastError();
}

// A slice of few tokens takes the decode's kernels: blocks of 8 or 16 tokens read
// the pages as they are, where the other path first copies the whole cache (K as
// fp16, V transposed). Its products take a pass for each term, so the rule is
// tokens x terms <= 128 (us per call, this / the other path, behind 0, 2000, 20000
// and 60000 positions):
//   two terms    9 tokens 16 / 24, 20 / 26, 28 / 45, 46 / 86
//               64 tokens 18 / 23, 29 / 34, 57 / 61, 126 / 134
//               96 tokens 22 / 25, 34 / 34, 81 / 75, 188 / 164
//   three terms 33 tokens 18 / 23, 26 / 30, 51 / 55, 115 / 117
//               42 tokens 19 / 23, 27 / 31, 55 / 56, 126 / 118
//               64 tokens 19 / 23, 31 / 34, 67 / 61, 161 / 134
hipError_t launch_gqa_prefill_paged(qff_ctx* ctx, hipStream_t stream, const qff_gqa_params* p, const void* q_gate,
                                    const void* k, const void* v, qff_dtype in_dtype, const qff_kv_pages* kv,
                                    int start, void* out, qff_dtype out_dtype, int T) {
    // (a slice's precision follows from its tokens and types alone: a context of few
    // partial rows gives fewer chunks, pf_slots(cfg) at least one a token)
    if (T * paged_terms(p->kv_f16 != 0, out_dtype == QFF_BF16) > 2 * kPagedTokensMax)
        return launch_gqa_prefill(ctx, stream, p, q_gate, k, v, in_dtype, kv->k, kv->v, kv, start, out, out_dtype, T);
    const PagedKv pk = paged_kv(kv);
    if (!PagedTokens{start, T, kTile, kBlkSeqs}.append()) {
        ProfScope prof(ctx, stream, "gqa_paged_append");
        const RopeFreqs rf = rope_freqs(p->rope_theta);
        const int blocks = (2 * T + 3) / 4;
#define QFF_APP(I, F) gqa_paged_append_kernel<I, F><<<blocks, 256, 0, stream>>>(k, v, p->k_norm_w, rf, p->eps, pk, start, T)
        if (p->kv_f16) {
            if (in_dtype == QFF_BF16) QFF_APP(1, 1); else QFF_APP(0, 1);
        } else {
            if (in_dtype == QFF_BF16) QFF_APP(1, 0); else QFF_APP(0, 0);
        }
#undef QFF_APP
    }
    const int cap = static_cast<int>(std::min<long long>(kGqaMaxChunks, ctx->pf_slots / T));
    const PagedTokens tk = paged_tokens_split(start, T, ctx->num_cu / 2, cap);
    // partials where the sharing prefill keeps its own: m and d [T][2][cap][8], o [T][2][cap][8][256]
    const PagedPartials pp{ctx->pf_md, ctx->pf_md + static_cast<size_t>(T) * 16 * cap, ctx->pf_o, ctx->gqa_nc, cap};
    launch_partials(ctx, stream, p, q_gate, k, v, in_dtype, pk, nullptr, tk, pp, 2 * tk.items(), out, out_dtype, T);
    return hipGetLastError();
}

}  // namespace qff
