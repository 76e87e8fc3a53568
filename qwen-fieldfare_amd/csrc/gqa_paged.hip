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
//            positions): a group's shared positions for up to 16 of its
//            sequences (128 q rows), or one sequence's own positions (8 q
//            rows), whose last chunk appends the new token. K/V tiles go
//            through LDS. One launch for both, so that the few long streams of
//            a shared prefix and the many short ones behind it run together.
//   combine  one workgroup per (q head, sequence): joins the partials, gate.
//
// Both products run on 16x16x32 MFMAs in the cache's type, in which K and V
// are exact. q and the softmax weights enter as NT terms of that type (hi,
// the rest rounded again, ...): two bf16 terms carry 16 bits and two fp16
// terms 22, three bf16 terms 24. bf16 outputs take two terms; fp32 outputs
// three of bf16 or two of fp16 (error 2e-7 to 7e-7 of the exact output, where
// two bf16 terms leave 6e-6). fp16 weights are scaled by 2^7 (kShift), so that
// weights down to 2^-21 of the row's largest keep all bits of their first term.
#include "common.hpp"
#include "internal.hpp"
#include "mfma.hpp"

namespace qff {

// ---- split of a call's positions ------------------------------------------------
//
// Every workgroup derives the same split from the device arrays (no host
// sync, no atomics). `positions` give each sequence's length L (0 where the
// position lies outside the table: no chunks, its output is NaN). With groups,
// consecutive sequences with the same group >= 0 (and L > 0) are a run, cut
// every 16 sequences, and at every multiple of 64 sequences, into blocks; the
// positions before S = the least of the block's shared_len and L - 1, rounded
// down to 16, are read through the table row of the block's first sequence for
// all of it. Any values of the arrays give a valid split.
//
// A CU holds one workgroup (its LDS), which leaves the CU idle while it starts,
// so the chunk length is the least that needs no second round of workgroups
// where such a length exists.

constexpr int kBlkSeqs = 16;    // sequences of a block
constexpr int kTile = 64;       // positions of a tile
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

__device__ __forceinline__ LanePlan lane_plan(const PagedSeqs& a, int b0, int lane) {
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
    const unsigned long long blocks = __ballot(((lane - run) & (kBlkSeqs - 1)) == 0);
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

// Workgroups (per kv head) of the sequence in this lane at chunk length ch:
// its own chunks, and its block's shared ones in the block's first lane.
__device__ __forceinline__ int items_of(const LanePlan& p, int ch, int lane) {
    return chunks_of(p.own(), ch) + (p.first == lane ? chunks_of(p.shared, ch) : 0);
}

// The chunk length, whole tiles.
__device__ __forceinline__ int chunk_length(const PagedSeqs& a, const LanePlan& p0, int lane) {
    long long tiles = 0;
    int streams = 0, longest = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const LanePlan p = b0 == 0 ? p0 : lane_plan(a, b0, lane);
        tiles += wave_sum_int(items_of(p, kTile, lane));
        streams += wave_sum_int(items_of(p, 1 << 30, lane));
        longest = max(longest, wave_max_int(p.len));
    }
    // (sum of ceil(n / ch) <= (tiles / ch) + streams)
    int ch = static_cast<int>((tiles + a.slots - 1) / a.slots);
    const int sure = streams < a.slots ? static_cast<int>((tiles + a.slots - streams - 1) / (a.slots - streams)) : ch;
    if (a.batch <= 64) {
        while (ch < sure && wave_sum_int(items_of(p0, ch * kTile, lane)) > a.slots) ch += (ch + 15) / 16;
    } else {
        ch = sure;
    }
    ch = max(max(ch, 1), (longest + (a.cap - 2) * kTile - 1) / ((a.cap - 2) * kTile));
    // (the same in every lane; the compiler has to know, for the scalar addresses that follow from it)
    return __builtin_amdgcn_readfirstlane(ch * kTile);
}

// Workgroup item g: the sequence that holds it (-1: past the last), the item's
// number among the sequence's, its plan (first: as a sequence).
__device__ __forceinline__ int find_item(const PagedSeqs& a, const LanePlan& p0, int ch, int g, int lane, int& c,
                                         LanePlan& plan) {
    int base = 0;
    c = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const LanePlan p = b0 == 0 ? p0 : lane_plan(a, b0, lane);
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

    __device__ __forceinline__ void load(const int32_t* row, int first, int last, int num_pages, int lane) {
        base = first;
        const int p = row[min(first + lane, last)];
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

// Head q row of lane l's MFMA column n = l % 16, in the operand order of a
// 16x16x32 product: lane group kb = l / 16 holds dims 32 jj + 8 kb + e. The
// RMS sums over the four groups; the rotation's partner of dim d < 32 is jj = 1
// of the same lane. cs / sn: cos and sin of angle 8 kb + e.
template <int KV_F16, int NT>
__device__ __forceinline__ void q_operand(float (&x)[8][8], const float* __restrict__ w, int kb, float eps,
                                          const float (&cs)[8], const float (&sn)[8], u32x4_t (&q)[NT][8]) {
    float ss = 0.0f;
#pragma unroll
    for (int jj = 0; jj < 8; ++jj)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[jj][e] * x[jj][e];
    ss += __shfl_xor(ss, 16, 64);
    ss += __shfl_xor(ss, 32, 64);
    const float inv = 1.0f / sqrtf(ss / 256.0f + eps);
#pragma unroll
    for (int jj = 0; jj < 8; ++jj) {
        float wv[8];
        load8<0>(w, 32 * jj + 8 * kb, wv);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[jj][e] = x[jj][e] * inv * wv[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = x[0][e], b = x[1][e];
        x[0][e] = a * cs[e] - b * sn[e];
        x[1][e] = b * cs[e] + a * sn[e];
    }
#pragma unroll
    for (int jj = 0; jj < 8; ++jj)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t t[NT];
            split_terms<KV_F16, NT>(x[jj][2 * i], x[jj][2 * i + 1], t);
#pragma unroll
            for (int k = 0; k < NT; ++k) q[k][jj][i] = t[k];
        }
}

struct PagedPartials {
    float* m;   // [slots][8]
    float* d;   // [slots][8]
    float* o;   // [slots][8][256]
    int cstride;   // slots per (sequence, kv head): the shared chunks first, then its own
};

// ---- partial ------------------------------------------------------------------------
//
// grid 2 x items, 512 threads: kv head u & 1 of item u >> 1. A block of up to
// 2 R sequences (R a power of two <= 8) has R row blocks of 16 q rows (two
// sequences x 8 heads); a single sequence fills half of one. Tiles of 64
// positions of K and V are copied straight into LDS (two stages of 64 KB,
// XOR-swizzled rows), the next one while a tile computes. Wave w takes row
// block w % R: all 64 positions where R = 8, and otherwise half w / R of them
// (waves past 2 R only copy); the halves are merged at the end through LDS. Per
// 32 positions a wave reads 16 KB of K and 16 KB of V operands for 32 NT MFMAs:
//   S^T = K Q^T   A = K rows (b128 reads), B = q in registers; a lane's scores
//                 belong to its one q row, positions 16 b + 4 kb + i
//   O^T = V^T P^T A = V^T through two transposed reads (positions 4 kb + i and
//                 16 + 4 kb + i: the order the lane's weights are in), B = P.
// The chunk that ends with the new token norms and rotates k (wave 2) and takes
// v (wave 3), writes both to their page and, once the tile that holds the
// position is in LDS, into its rows there; the rows behind them are zeroed
// (what the page holds there may be any bit pattern).
struct PartLds {
    uint16_t tile[2][2][kTile * 256];   // stage, K / V
    float md[8][16][2];                 // the second halves' (m, d)
};

__device__ __forceinline__ int tile_swz(int r) { return ((r & 7) << 1) | ((r >> 3) & 1); }

template <int IN_DT, int KV_F16, int NT>
__global__ __launch_bounds__(512) void gqa_paged_partial_kernel(
    const void* __restrict__ q_gate, const void* __restrict__ k_new, const void* __restrict__ v_new,
    const float* __restrict__ q_norm_w, const float* __restrict__ k_norm_w, RopeFreqs rf, float scale, float eps,
    PagedKv kv, PagedSeqs a, PagedPartials pp) {
    __shared__ __attribute__((aligned(1024))) PartLds L;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int kvh = blockIdx.x & 1;
    const LanePlan p0 = lane_plan(a, 0, lane);
    const int ch = chunk_length(a, p0, lane);
    LanePlan plan;
    int item;
    const int found = find_item(a, p0, ch, static_cast<int>(blockIdx.x >> 1), lane, item, plan);
    if (found < 0) return;   // (uniform over the workgroup)
    // the block's shared chunks come first among its first sequence's items
    const int lead = found, npfx = chunks_of(plan.shared, ch);
    const bool pfx = found == plan.first && item < npfx;
    const int c = pfx ? item : item - (found == plan.first ? npfx : 0);
    const int count = pfx ? plan.count : 1;
    const int p_begin = (pfx ? 0 : plan.shared) + c * ch, p_end = min(pfx ? plan.shared : plan.len, p_begin + ch);
    const bool has_new = !pfx && p_end == plan.len;
    const int slot_c = pfx ? c : npfx + c;
    const int ntiles = (p_end - p_begin + kTile - 1) / kTile;
    const int mask = (1 << kv.lg) - 1;
    const int32_t* row = kv.table + static_cast<size_t>(lead) * kv.cols;
    const int last_entry = (p_end - 1) >> kv.lg;
    PageWindow win;
    win.load(row, p_begin >> kv.lg, last_entry, kv.num_pages, lane);

    // tile t into stage t & 1: wave wv copies rows 2 wv + 16 i, + 1 of K and V,
    // i < 4; 16 positions past the chunk's end repeat its last ones (masked;
    // finite, or zeroed behind the new token). Returns the tile's bad pages as
    // bits i.
    auto issue = [&](int t) -> unsigned {
        const int t0 = p_begin + t * kTile;
        if ((min(t0 + kTile, p_end) - 1) >> kv.lg > win.base + 63)
            win.load(row, t0 >> kv.lg, last_entry, kv.num_pages, lane);
        unsigned bad = 0;
        const int h = lane >> 5;
        const uint32_t lt = 1024u * h + 16u * ((lane & 31) ^ (2 * h) ^ tile_swz(2 * wv & 15));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = min(t0 + 16 * i, (p_end - 1) & ~15);
            const int entry = p >> kv.lg;
            const size_t at = (((static_cast<size_t>(win.of(entry)) << kv.lg) + (p & mask) + 2 * wv) * 2 + kvh) * 512;
            bad |= (win.is_bad(entry) ? 1u : 0u) << i;
            dma16(reinterpret_cast<const char*>(kv.k) + at, lt, lds_addr(&L.tile[t & 1][0][(16 * i + 2 * wv) * 256]));
            dma16(reinterpret_cast<const char*>(kv.v) + at, lt, lds_addr(&L.tile[t & 1][1][(16 * i + 2 * wv) * 256]));
        }
        return bad;
    };
    unsigned bad_next = issue(0);

    // ---- this wave's q rows ---------------------------------------------------
    const int n = lane & 15, kb = lane >> 4;
    const int nrb = (count + 1) / 2;
    const int R = nrb <= 1 ? 1 : nrb <= 2 ? 2 : nrb <= 4 ? 4 : 8;
    const int halves = R == 8 ? 1 : 2;
    const int rb = wv & (R - 1), half = wv / R;
    const bool active = half < halves && rb < nrb;
    const int seq = lead + min(2 * rb + (n >> 3), count - 1);
    u32x4_t q[NT][8];
    u32x2_t fresh = u32x2_t{0u, 0u};   // dims 4 lane .. + 3 of the new k (wave 2) or v (wave 3)
    if (active) {
        float x[8][8];
        const size_t qbase = (static_cast<size_t>(seq) * 16 + kvh * 8 + (n & 7)) * 512 + 8 * kb;
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) load8<IN_DT>(q_gate, qbase + 32 * jj, x[jj]);
        // lane l: angle l % 32 of the row block's sequence l / 32
        const int s2 = lead + min(2 * rb + (lane >> 5), count - 1);
        const float ang = static_cast<float>(a.positions[s2]) * rf.f[lane & 31];
        const float cl = cosf(ang), sl = sinf(ang);
        float cs[8], sn[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int from = 32 * (n >> 3) + 8 * kb + e;
            cs[e] = __shfl(cl, from, 64);
            sn[e] = __shfl(sl, from, 64);
        }
        q_operand<KV_F16, NT>(x, q_norm_w, kb, eps, cs, sn, q);
    } else if (has_new && (wv == 2 || wv == 3)) {
        // dims 4 lane .. + 3; the rotation's partner of dim d < 32 is d + 32, 8 lanes on
        const size_t at = (static_cast<size_t>(lead) * 2 + kvh) * 256 + 4 * lane;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = elem<IN_DT>::load(wv == 2 ? k_new : v_new, at + i);
        if (wv == 2) {
            const float ang = static_cast<float>(plan.len - 1) * rf.f[lane & 31];
            const float cl = cosf(ang), sl = sinf(ang);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss += x[i] * x[i];
            const float inv = 1.0f / sqrtf(group_sum<64>(ss) / 256.0f + eps);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = x[i] * inv * k_norm_w[4 * lane + i];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float up = __shfl_down(x[i], 8, 64), dn = __shfl_up(x[i], 8, 64);
                const float ci = __shfl(cl, (4 * lane + i) & 31, 64), si = __shfl(sl, (4 * lane + i) & 31, 64);
                const int d = 4 * lane + i;
                if (d < 64) x[i] = d < 32 ? x[i] * ci - up * si : x[i] * ci + dn * si;
            }
        }
        uint32_t w0[1], w1[1];
        split_terms<KV_F16, 1>(x[0], x[1], w0);
        split_terms<KV_F16, 1>(x[2], x[3], w1);
        fresh = u32x2_t{w0[0], w1[0]};
        const int page = row[(plan.len - 1) >> kv.lg];
        if (page >= 0 && page < kv.num_pages) {   // (dropped where the page lies outside the pool)
            const size_t off = ((static_cast<size_t>(page) << kv.lg) + ((plan.len - 1) & mask)) * 512 + kvh * 256 + 4 * lane;
            *reinterpret_cast<u32x2_t*>((wv == 2 ? kv.k : kv.v) + off) = fresh;
        }
    }

    float m_run = -INFINITY, d_run = 0.0f;
    f32x4_t oacc[16];   // O^T: dims 16 dt + 4 kb + i of the lane's row
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) oacc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const float sc = scale * 1.44269504088896341f;
    const uint32_t kaddr = 512u * n + 16u * (kb ^ tile_swz(n));
    const int vr = 4 * kb + (n >> 2);
    const uint32_t vaddr = 512u * vr + 16u * (((n >> 1) & 1) ^ tile_swz(vr)) + 8u * (n & 1);

    auto lds128 = [](uint32_t at) {
        return *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(static_cast<uintptr_t>(at));
    };
    auto lds_tr = [](uint32_t at) {
        typedef short s16x4_l __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                               (s16x4_l __attribute__((address_space(3)))*)(static_cast<uintptr_t>(at))));
    };

    for (int t = 0; t < ntiles; ++t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();   // the tile is in LDS, and the other stage's readers are done
        const unsigned bad = bad_next;
        const int t0 = p_begin + t * kTile;
        if (t + 1 < ntiles) {
            bad_next = issue(t + 1);
        } else if (has_new) {
            // the new token's row, and zeros behind it in the 32 positions it is among
            const int r = plan.len - 1 - t0, end = (r | 31) + 1;
            auto at = [&](int which, int rr) {
                return reinterpret_cast<u32x2_t*>(&L.tile[t & 1][which][rr * 256 + 8 * ((lane >> 1) ^ tile_swz(rr)) + 4 * (lane & 1)]);
            };
            if (wv == 2 || wv == 3) *at(wv - 2, r) = fresh;
            for (int z = r + 1 + wv; z < end; z += 8) *at(1, z) = u32x2_t{0u, 0u};
            __syncthreads();
        }
        if (!active) continue;
        const uint32_t kt = lds_addr(L.tile[t & 1][0]), vt = lds_addr(L.tile[t & 1][1]);
#pragma unroll 1
        for (int u = 0; u < 3 - halves; ++u) {
            const int sub = halves == 2 ? half : u;
            const int s0 = t0 + 32 * sub;
            if (s0 >= p_end) break;
            f32x4_t s[2][NT];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int k = 0; k < NT; ++k) s[b][k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int jj = 0; jj < 8; ++jj)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const u32x4_t kf = lds128(kt + 16384u * sub + 8192u * b + (kaddr ^ (64u * jj)));
#pragma unroll
                    for (int k = 0; k < NT; ++k) s[b][k] = mfma32<KV_F16>(kf, q[k][jj], s[b][k]);
                }
            // softmax in base 2
            const bool cut = s0 + 32 > p_end || (bad >> (2 * sub) & 3);   // (uniform)
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
            if (cut) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[b][i] = s0 + 16 * b + 4 * kb + i >= p_end ? -INFINITY
                                  : (bad >> (2 * sub + b)) & 1     ? __builtin_nanf("")
                                                                   : x[b][i];
            }
            float tm = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                             fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
            tm = fmaxf(tm, __shfl_xor(tm, 16, 64));
            tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
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
            const float mb = m_run - kShift<KV_F16>;
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
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) {
                const uint32_t va = vt + 16384u * sub + (vaddr ^ (32u * dt));
                const u32x2_t v0 = lds_tr(va), v1 = lds_tr(va + 8192u);
                const u32x4_t vf = u32x4_t{v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
                for (int k = 0; k < NT; ++k) oacc[dt] = mfma32<KV_F16>(vf, pw[k], oacc[dt]);
            }
        }
    }
    d_run += __shfl_xor(d_run, 16, 64);
    d_run += __shfl_xor(d_run, 32, 64);
    // ---- the second halves handed over in LDS, one 16-byte piece a lane and dim tile
    if (halves == 2) {   // (uniform over the workgroup)
        __syncthreads();
        f32x4_t* hand = reinterpret_cast<f32x4_t*>(&L) + rb * 1024;
        if (active && half == 1) {
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) hand[64 * dt + lane] = oacc[dt];
            if (kb == 0) {
                L.md[rb][n][0] = m_run;
                L.md[rb][n][1] = d_run;
            }
        }
        __syncthreads();
        if (active && half == 0) {
            const float m1 = L.md[rb][n][0], d1 = L.md[rb][n][1];
            const float m = fmaxf(m_run, m1);
            // (a half without any position, or whose scores are all NaN, has maximum -inf)
            const float f0 = m_run == m ? 1.0f : __builtin_amdgcn_exp2f(m_run - m);
            const float f1 = m1 == m ? 1.0f : __builtin_amdgcn_exp2f(m1 - m);
            m_run = m;
            d_run = d_run * f0 + d1 * f1;
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) {
                const f32x4_t o = hand[64 * dt + lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) oacc[dt][i] = oacc[dt][i] * f0 + o[i] * f1;
            }
        }
    }
    if (!active || half != 0 || 2 * rb + (n >> 3) >= count) return;
    const size_t slot = (static_cast<size_t>(seq) * 2 + kvh) * pp.cstride + slot_c;
    if (kb == 0) {
        pp.m[slot * 8 + (n & 7)] = m_run - kShift<KV_F16>;
        pp.d[slot * 8 + (n & 7)] = d_run;
    }
    float* o = pp.o + (slot * 8 + (n & 7)) * 256 + 4 * kb;
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) *reinterpret_cast<f32x4_t*>(o + 16 * dt) = oacc[dt];
}

// ---- combine ----------------------------------------------------------------------------
//
// grid (16 q heads x DS dim blocks, batch), 512 threads, 256 / DS dims a
// workgroup: chunk weights one thread a chunk; 8 DS streams of float4 lanes,
// stream s adding chunks s, s + 8 DS, ... in order, then the streams in a fixed
// order (results do not depend on timing). The (m, d) of every slot and the
// gate are requested before the split is known, and a stream's first four rows
// before the weights; every load is unconditional, its index clamped.
template <int IN_DT, int OUT_DT, int DS>
__global__ __launch_bounds__(512) void gqa_paged_combine_kernel(const void* __restrict__ q_gate, PagedSeqs a,
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
    const LanePlan p0 = lane_plan(a, 0, lane);
    const int ch = chunk_length(a, p0, lane);
    const LanePlan mine = seq < 64 ? p0 : lane_plan(a, seq & ~63, lane);
    const int len = __builtin_amdgcn_readlane(mine.len, seq & 63);
    const int shared = __builtin_amdgcn_readlane(mine.shared, seq & 63);
    if (len == 0) {   // (uniform over the workgroup)
        if (t < kDims) elem<OUT_DT>::store(out, qi * 256 + d0 + t, __builtin_nanf(""));
        return;
    }
    const int nc = chunks_of(shared, ch) + chunks_of(len - shared, ch);   // <= cstride
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

// ---- launch ---------------------------------------------------------------------------

hipError_t launch_gqa_decode_paged(qff_ctx* ctx, hipStream_t stream, const qff_gqa_params* p, const void* q_gate,
                                   const void* k_new, const void* v_new, qff_dtype in_dtype, const qff_kv_pages* kv,
                                   const int32_t* positions, const int32_t* group, const int32_t* shared_len,
                                   void* out, qff_dtype out_dtype, int batch) {
    const int lg = __builtin_ctz(static_cast<unsigned>(kv->page_size));
    const PagedKv pk{static_cast<uint16_t*>(kv->k), static_cast<uint16_t*>(kv->v), kv->table, kv->num_pages, lg,
                     kv->table_cols};
    const int cap = gqa_chunk_cap(ctx->cfg, batch);
    const PagedSeqs a{positions, group, shared_len, batch, kv->table_cols << lg, ctx->num_cu / 2, cap};
    const PagedPartials pp{ctx->gqa_m, ctx->gqa_d, ctx->gqa_o, cap};
    const RopeFreqs rf = rope_freqs(p->rope_theta);
    const bool f16 = p->kv_f16 != 0, in16 = in_dtype == QFF_BF16, out16 = out_dtype == QFF_BF16;
    {
        ProfScope prof(ctx, stream, "gqa_paged_partial");
        // a round of workgroups, and one more for each stream of positions (a
        // sequence's own, a block's shared ones) that rounding up can add
        const int grid = 2 * (a.slots + batch + (group ? batch / 2 : 0));
#define QFF_PART(I, F, N)                                                                                        \
    gqa_paged_partial_kernel<I, F, N><<<grid, 512, 0, stream>>>(q_gate, k_new, v_new, p->q_norm_w, p->k_norm_w, rf, \
                                                                p->scale, p->eps, pk, a, pp)
        if (f16) {
            if (in16) QFF_PART(1, 1, 2); else QFF_PART(0, 1, 2);
        } else if (out16) {
            if (in16) QFF_PART(1, 0, 2); else QFF_PART(0, 0, 2);
        } else {
            if (in16) QFF_PART(1, 0, 3); else QFF_PART(0, 0, 3);
        }
#undef QFF_PART
    }
    ProfScope prof(ctx, stream, "gqa_paged_combine");
    const int ds = batch <= 8 ? 4 : 1;   // small batches split each head's dims over four workgroups
    const dim3 cgrid(16 * ds, batch);
#define QFF_COMB(I, O)                                                                                       \
    if (ds == 4) gqa_paged_combine_kernel<I, O, 4><<<cgrid, 512, 0, stream>>>(q_gate, a, pp, out);           \
    else gqa_paged_combine_kernel<I, O, 1><<<cgrid, 512, 0, stream>>>(q_gate, a, pp, out)
    if (in16) {
        if (out16) { QFF_COMB(1, 1); } else { QFF_COMB(1, 0); }
    } else {
        if (out16) { QFF_COMB(0, 1); } else { QFF_COMB(0, 0); }
    }
#undef QFF_COMB
    return hipGetLastError();
}

}  // namespace qff
