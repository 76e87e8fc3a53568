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
//   prefix   (shared form only) one workgroup per (block of at most 16
//            sequences of a group, kv head, chunk of the shared positions):
//            up to 128 q rows over K/V tiles staged in LDS.
//   tail     one wave per (sequence, kv head, chunk of the sequence's other
//            positions); the one whose chunk holds the new token appends it.
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
// position lies outside the table: no chunks, its output is NaN). In the
// shared form, consecutive sequences with the same group >= 0 (and L > 0)
// are a run, cut every 16 sequences, and at every multiple of 64 sequences,
// into blocks; the positions before S = the least of the block's shared_len
// and L - 1, rounded down to 16, are read through the table row of the block's
// first sequence for all of it. Any values of the arrays give a valid split.

constexpr int kBlkSeqs = 16;    // sequences of a prefix block
constexpr int kPfxTile = 64;    // positions of a prefix tile
constexpr int kMinShared = 64;  // shorter shared prefixes are left to the sequences

struct PagedSeqs {
    const int32_t* positions;
    const int32_t* group;        // shared form only
    const int32_t* shared_len;   // shared form only
    int batch, max_ctx;
    int target, target_pfx;      // chunks to aim for, per kv head
    int cap, cap_pfx;            // chunks allowed per sequence: of its own positions, of the shared ones
};

// Sequence b0 + lane: its length, the shared positions of its block, the
// block's first sequence (as a lane) and size; shared is 0 for single
// sequences.
struct LanePlan {
    int len, shared, first, count;
};

template <bool SHARED>
__device__ __forceinline__ LanePlan lane_plan(const PagedSeqs& a, int b0, int lane) {
    const int b = b0 + lane;
    LanePlan p{0, 0, lane, 1};
    int grp = -1, sh = 0;
    if (b < a.batch) {
        const int pos = a.positions[b];
        if (SHARED) {
            grp = a.group[b];
            sh = a.shared_len[b];
        }
        p.len = (pos >= 0 && pos < a.max_ctx) ? pos + 1 : 0;
    }
    if (!SHARED) return p;
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

// Chunk lengths of the sequences' own positions (a multiple of 32) and of the
// shared ones (whole tiles).
struct Chunks {
    int own, pfx;
};

template <bool SHARED>
__device__ __forceinline__ Chunks chunk_lengths(const PagedSeqs& a, const LanePlan& p0, int lane) {
    long long own = 0, pfx = 0;
    int max_own = 0, max_pfx = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const LanePlan p = b0 == 0 ? p0 : lane_plan<SHARED>(a, b0, lane);
        const int mine = p.len - p.shared;
        own += wave_sum_int(mine);
        max_own = max(max_own, wave_max_int(mine));
        if (SHARED) {
            pfx += wave_sum_int(p.first == lane ? p.shared : 0);
            max_pfx = max(max_pfx, wave_max_int(p.shared));
        }
    }
    Chunks c;
    const int by_total = static_cast<int>((own + a.target - 1) / a.target), by_cap = (max_own + a.cap - 1) / a.cap;
    // (the same in every lane; the compiler has to know, for the scalar addresses that follow from them)
    c.own = __builtin_amdgcn_readfirstlane((max(max(by_total, by_cap), 1) + 31) / 32 * 32);
    c.pfx = kPfxTile;
    if (SHARED) {
        const int p_total = static_cast<int>((pfx + a.target_pfx - 1) / a.target_pfx);
        const int p_cap = (max_pfx + a.cap_pfx - 1) / a.cap_pfx;
        c.pfx = __builtin_amdgcn_readfirstlane((max(max(p_total, p_cap), 1) + kPfxTile - 1) / kPfxTile * kPfxTile);
    }
    return c;
}

// Index g among the items n(plan) of all sequences in order: the sequence that
// holds it (-1: past the last), the item's number within it, its plan.
template <bool SHARED, class N>
__device__ __forceinline__ int find_item(const PagedSeqs& a, const LanePlan& p0, int g, int lane, N n, int& c,
                                         LanePlan& plan) {
    int base = 0;
    c = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const LanePlan p = b0 == 0 ? p0 : lane_plan<SHARED>(a, b0, lane);
        const int mine = n(p);
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

__device__ __forceinline__ int chunks_of(int n, int ch) { return (n + ch - 1) / ch; }

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

__device__ __forceinline__ void paged_wave_sync() {   // orders one wave's LDS stores before its later LDS loads
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

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

// ---- prefix -------------------------------------------------------------------------
//
// grid 2 x (target_pfx + batch / 2), 512 threads: kv head u & 1 of prefix
// chunk u >> 1. A block of up to 2 R sequences (R a power of two <= 8) has R
// row blocks of 16 q rows (two sequences x 8 heads). Tiles of 64 positions of K
// and V are copied straight into LDS (two stages of 64 KB, XOR-swizzled rows),
// the next one while a tile computes. Wave w takes row block w % R: all 64
// positions where R = 8, and otherwise half w / R of them (waves past 2 R only
// copy); the halves are merged at the end through LDS. Per 32 positions a wave
// reads 16 KB of K and 16 KB of V operands for 32 NT MFMAs:
//   S^T = K Q^T   A = K rows (b128 reads), B = q in registers; a lane's scores
//                 belong to its one q row, positions 16 b + 4 kb + i
//   O^T = V^T P^T A = V^T through two transposed reads (positions 4 kb + i and
//                 16 + 4 kb + i: the order the lane's weights are in), B = P.
struct PfxLds {
    uint16_t tile[2][2][kPfxTile * 256];   // stage, K / V
    float md[8][16][2];                    // the second halves' (m, d)
};

__device__ __forceinline__ int tile_swz(int r) { return ((r & 7) << 1) | ((r >> 3) & 1); }

template <int IN_DT, int KV_F16, int NT>
__global__ __launch_bounds__(512) void gqa_paged_prefix_kernel(const void* __restrict__ q_gate,
                                                               const float* __restrict__ q_norm_w, RopeFreqs rf,
                                                               float scale, float eps, PagedKv kv, PagedSeqs a,
                                                               PagedPartials pp) {
    __shared__ __attribute__((aligned(1024))) PfxLds L;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int kvh = blockIdx.x & 1;
    const LanePlan p0 = lane_plan<true>(a, 0, lane);
    const Chunks ch = chunk_lengths<true>(a, p0, lane);
    LanePlan plan;
    int c;
    const int lead = find_item<true>(a, p0, static_cast<int>(blockIdx.x >> 1), lane, [&](const LanePlan& p) {
        return p.first == lane ? chunks_of(p.shared, ch.pfx) : 0;
    }, c, plan);
    if (lead < 0) return;   // (uniform over the workgroup)
    const int p_begin = c * ch.pfx, p_end = min(plan.shared, p_begin + ch.pfx);
    const int ntiles = (p_end - p_begin + kPfxTile - 1) / kPfxTile;
    const int32_t* row = kv.table + static_cast<size_t>(lead) * kv.cols;
    const int last_entry = (p_end - 1) >> kv.lg;
    PageWindow win;
    win.load(row, p_begin >> kv.lg, last_entry, kv.num_pages, lane);

    // tile t into stage t & 1: wave wv copies rows 2 wv + 16 i, + 1 of K and V,
    // i < 4; 16 positions past the chunk's end repeat its last ones (finite
    // data, masked). Returns the tile's bad pages as bits i.
    auto issue = [&](int t) -> unsigned {
        const int t0 = p_begin + t * kPfxTile;
        if ((min(t0 + kPfxTile, p_end) - 1) >> kv.lg > win.base + 63)
            win.load(row, t0 >> kv.lg, last_entry, kv.num_pages, lane);
        unsigned bad = 0;
        const int h = lane >> 5;
        const uint32_t lt = 1024u * h + 16u * ((lane & 31) ^ (2 * h) ^ tile_swz(2 * wv & 15));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = min(t0 + 16 * i, p_end - 16);
            const int entry = p >> kv.lg;
            const size_t at = (((static_cast<size_t>(win.of(entry)) << kv.lg) + (p & ((1 << kv.lg) - 1)) + 2 * wv) * 2 + kvh) * 512;
            bad |= (win.is_bad(entry) ? 1u : 0u) << i;
            dma16(reinterpret_cast<const char*>(kv.k) + at, lt, lds_addr(&L.tile[t & 1][0][(16 * i + 2 * wv) * 256]));
            dma16(reinterpret_cast<const char*>(kv.v) + at, lt, lds_addr(&L.tile[t & 1][1][(16 * i + 2 * wv) * 256]));
        }
        return bad;
    };
    unsigned bad_next = issue(0);

    // ---- this wave's q rows ---------------------------------------------------
    const int n = lane & 15, kb = lane >> 4;
    const int nrb = (plan.count + 1) / 2;
    const int R = nrb <= 1 ? 1 : nrb <= 2 ? 2 : nrb <= 4 ? 4 : 8;
    const int halves = R == 8 ? 1 : 2;
    const int rb = wv & (R - 1), half = wv / R;
    const bool active = half < halves && rb < nrb;
    const int seq = lead + min(2 * rb + (n >> 3), plan.count - 1);
    u32x4_t q[NT][8];
    if (active) {
        float x[8][8];
        const size_t qbase = (static_cast<size_t>(seq) * 16 + kvh * 8 + (n & 7)) * 512 + 8 * kb;
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) load8<IN_DT>(q_gate, qbase + 32 * jj, x[jj]);
        // lane l: angle l % 32 of the row block's sequence l / 32
        const int s2 = lead + min(2 * rb + (lane >> 5), plan.count - 1);
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
        if (t + 1 < ntiles) bad_next = issue(t + 1);
        if (!active) continue;
        const int t0 = p_begin + t * kPfxTile;
        const uint32_t kt = lds_addr(L.tile[t & 1][0]), vt = lds_addr(L.tile[t & 1][1]);
#pragma unroll 1
        for (int u = 0; u < 3 - halves; ++u) {
            const int sub = halves == 2 ? half : u;
            if (t0 + 32 * sub >= p_end) break;
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
            float tm = -INFINITY;
            float x[2][4];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bool gone = t0 + 32 * sub + 16 * b >= p_end, nan = (bad >> (2 * sub + b)) & 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = s[b][0][i];
#pragma unroll
                    for (int k = 1; k < NT; ++k) v += s[b][k][i];
                    v = gone ? -INFINITY : nan ? __builtin_nanf("") : v * sc;
                    x[b][i] = v;
                    tm = fmaxf(tm, v);
                }
            }
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
    if (!active || half != 0 || 2 * rb + (n >> 3) >= plan.count) return;
    const size_t slot = (static_cast<size_t>(seq) * 2 + kvh) * pp.cstride + c;
    if (kb == 0) {
        pp.m[slot * 8 + (n & 7)] = m_run - kShift<KV_F16>;
        pp.d[slot * 8 + (n & 7)] = d_run;
    }
    float* o = pp.o + (slot * 8 + (n & 7)) * 256 + 4 * kb;
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) *reinterpret_cast<f32x4_t*>(o + 16 * dt) = oacc[dt];
}

// ---- tail -----------------------------------------------------------------------------
//
// grid 2 x (target + batch), one wave each: kv head u & 1 of chunk u >> 1 of
// the sequences' own positions. The wave norms and rotates the 8 q heads into
// LDS; the one whose chunk holds the new token also norms and rotates k,
// appends k and v to their page and keeps both in LDS for its own use. Tiles of
// 16 positions (one page each: pages hold a multiple of 16), the next tile's K
// and V rows in flight while a tile computes: S^T = K Q^T with K rows straight
// from HBM (16 bytes a lane) and q's first two terms in the two 8-column halves
// of the MFMA (a third in a product of its own), the V tile through LDS and
// transposed reads, O += P V with the weights' terms in the two 8-row halves.
// The cache is read with non-temporal loads: every byte is read once a step.
constexpr int kTailTile = 16;
constexpr int kTailStride = 264;   // elements per V row in LDS: 256 + 8

struct TailTile {
    u32x4_t k[8], v[8];
};

template <int NT>
struct TailLds {
    uint16_t q[NT][8][256];
    uint16_t vs[kTailTile * kTailStride];
    uint16_t knew[256], vnew[256];
    float2 rcs[32];
};

template <int IN_DT, int KV_F16, int NT, bool SHARED>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2)))
void gqa_paged_tail_kernel(const void* __restrict__ q_gate, const void* __restrict__ k_new,
                           const void* __restrict__ v_new, const float* __restrict__ q_norm_w,
                           const float* __restrict__ k_norm_w, RopeFreqs rf, float scale, float eps, PagedKv kv,
                           PagedSeqs a, PagedPartials pp) {
    __shared__ __attribute__((aligned(16))) TailLds<NT> L;
    const int lane = threadIdx.x & 63;
    const int kvh = blockIdx.x & 1;
    const LanePlan pl0 = lane_plan<SHARED>(a, 0, lane);
    const Chunks ch = chunk_lengths<SHARED>(a, pl0, lane);
    LanePlan plan;
    int c;
    const int seq = find_item<SHARED>(a, pl0, static_cast<int>(blockIdx.x >> 1), lane, [&](const LanePlan& p) {
        return chunks_of(p.len - p.shared, ch.own);
    }, c, plan);
    if (seq < 0) return;   // past the last chunk
    const int pos = plan.len - 1;
    const int p_start = plan.shared + c * ch.own;
    const int p_end = min(pos + 1, p_start + ch.own);
    const bool has_new = pos < p_end;
    const int mask = (1 << kv.lg) - 1;
    const int32_t* row = kv.table + static_cast<size_t>(seq) * kv.cols;
    const int last_entry = (p_end - 1) >> kv.lg, last_tile = (p_end - 1) & ~(kTailTile - 1);
    PageWindow win;
    win.load(row, p_start >> kv.lg, last_entry, kv.num_pages, lane);

    // Rows past the chunk's end re-read its last row (masked below; the cache
    // past a sequence may hold any bit pattern and is never read). Every row
    // that lands on the new token's position takes the LDS copy instead, so
    // tiles may be loaded before the append. The loads are unconditional (a
    // tile past the last re-reads the last) so that the waits stay exact.
    // Returns whether the tile's page lies outside the pool.
    auto load = [&](TailTile& tl, int at) -> bool {
        const int t0 = min(at, last_tile), entry = t0 >> kv.lg;
        if (entry > win.base + 63) win.load(row, entry, last_entry, kv.num_pages, lane);
        int l = lane;
        asm volatile("" : "+v"(l));
        const size_t base = ((static_cast<size_t>(win.of(entry)) << kv.lg) + (t0 & mask)) * 512 + kvh * 256;
        const int last = p_end - 1 - t0;
        const uint16_t* krow = kv.k + base + min(l & 15, last) * 512 + 8 * (l >> 4);
#pragma unroll
        for (int jj = 0; jj < 8; ++jj)
            tl.k[jj] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(krow + 32 * jj));
        const uint16_t* vrow = kv.v + base + 8 * (l & 31);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            tl.v[i] = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4_t*>(vrow + min(2 * i + (l >> 5), last) * 512));
        return win.is_bad(entry);
    };
    // ---- q: RMS norm, rotation, terms into LDS. Lane -> head u / 32, dims
    // 8 (u % 32) .. + 7 for u = lane + 64 it; the rotation's pairs (d, d ^ 32)
    // of dims < 64 sit in lanes 4 apart. The q rows and norm weights are
    // requested first and the first tile right behind them.
    float xq[4][8], qw[8];
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const int u = 64 * it + lane;
        load8<IN_DT>(q_gate, (static_cast<size_t>(seq) * 16 + kvh * 8 + (u >> 5)) * 512 + 8 * (u & 31), xq[it]);
    }
    load8<0>(q_norm_w, 8 * (lane & 31), qw);
    __builtin_amdgcn_sched_barrier(0);
    TailTile ta, tb;
    bool bad_a = load(ta, p_start), bad_b = false;
    __builtin_amdgcn_sched_barrier(0);
    if (lane < 32) {
        const float ang = static_cast<float>(pos) * rf.f[lane];
        L.rcs[lane] = make_float2(cosf(ang), sinf(ang));
    }
    paged_wave_sync();
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        const int u = 64 * it + lane, hl = u >> 5, j = u & 31;
        float* x = xq[it];
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
        ss = group_sum<32>(ss);
        const float inv = 1.0f / sqrtf(ss / 256.0f + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * qw[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = 8 * j + i;
            const float partner = __shfl_xor(x[i], 4, 64);   // d +- 32 (used when d < 64)
            if (d < 64) {
                const float2 r = L.rcs[d & 31];
                x[i] = d < 32 ? x[i] * r.x - partner * r.y : x[i] * r.x + partner * r.y;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            uint32_t w[NT];
            split_terms<KV_F16, NT>(x[i], x[i + 1], w);
#pragma unroll
            for (int k = 0; k < NT; ++k) *reinterpret_cast<uint32_t*>(&L.q[k][hl][8 * j + i]) = w[k];
        }
    }
    // ---- the new token: k norm and rotation, k and v rounded to the cache's
    // type, into their page (dropped where the page lies outside the pool)
    if (has_new) {
        const size_t kb0 = (static_cast<size_t>(seq) * 2 + kvh) * 256 + 4 * lane;
        float kx[4], vx[4], ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            kx[i] = elem<IN_DT>::load(k_new, kb0 + i);
            vx[i] = elem<IN_DT>::load(v_new, kb0 + i);
            ss += kx[i] * kx[i];
        }
        ss = group_sum<64>(ss);
        const float inv = 1.0f / sqrtf(ss / 256.0f + eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) kx[i] = kx[i] * inv * k_norm_w[4 * lane + i];
        // dims 4 lane .. + 3; the partner of dim d < 32 is d + 32 = lane + 8
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float up = __shfl_down(kx[i], 8, 64), dn = __shfl_up(kx[i], 8, 64);
            const int d = 4 * lane + i;
            if (d < 64) {
                const float2 r = L.rcs[d & 31];
                kx[i] = d < 32 ? kx[i] * r.x - up * r.y : kx[i] * r.x + dn * r.y;
            }
        }
        uint32_t k01[1], k23[1], v01[1], v23[1];
        split_terms<KV_F16, 1>(kx[0], kx[1], k01);
        split_terms<KV_F16, 1>(kx[2], kx[3], k23);
        split_terms<KV_F16, 1>(vx[0], vx[1], v01);
        split_terms<KV_F16, 1>(vx[2], vx[3], v23);
        *reinterpret_cast<u32x2_t*>(&L.knew[4 * lane]) = u32x2_t{k01[0], k23[0]};
        *reinterpret_cast<u32x2_t*>(&L.vnew[4 * lane]) = u32x2_t{v01[0], v23[0]};
        const int page = row[pos >> kv.lg];
        if (page >= 0 && page < kv.num_pages) {
            const size_t off = ((static_cast<size_t>(page) << kv.lg) + (pos & mask)) * 512 + kvh * 256 + 4 * lane;
            *reinterpret_cast<u32x2_t*>(kv.k + off) = u32x2_t{k01[0], k23[0]};
            *reinterpret_cast<u32x2_t*>(kv.v + off) = u32x2_t{v01[0], v23[0]};
        }
    }
    paged_wave_sync();

    const int n = lane & 15, kb = lane >> 4;
    // q^T (B of 16x16x32): column n = head n & 7, first term for n < 8 and
    // second for n >= 8; the third term's columns n >= 8 are zero
    const uint16_t* qrow = n < 8 ? &L.q[0][n][8 * kb] : &L.q[1][n - 8][8 * kb];
    const uint16_t* qrow2 = &L.q[NT - 1][n & 7][8 * kb];
    const float sc = scale * 1.44269504088896341f;
    float m_run = -INFINITY, d_run = 0.0f;
    f32x4_t oacc[16];
#pragma unroll
    for (int jd = 0; jd < 16; ++jd) oacc[jd] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](TailTile& tl, int t0, bool bad) {
        if (has_new && t0 + n >= pos) {
#pragma unroll
            for (int jj = 0; jj < 8; ++jj) {
                u32x4_t w = *reinterpret_cast<const u32x4_t*>(&L.knew[32 * jj + 8 * kb]);
                asm volatile("" : "+v"(w));   // (not folded into the tile's load as one flat load)
                tl.k[jj] = w;
            }
        }
        f32x4_t s = f32x4_t{0.f, 0.f, 0.f, 0.f}, s2 = s;
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) {
            s = mfma32<KV_F16>(tl.k[jj], *reinterpret_cast<const u32x4_t*>(qrow + 32 * jj), s);
            if constexpr (NT == 3) s2 = mfma32<KV_F16>(tl.k[jj], *reinterpret_cast<const u32x4_t*>(qrow2 + 32 * jj), s2);
        }
        // lanes n and n ^ 8 add their terms' scores: both hold head n & 7's
        // (the third term's product has it in both halves)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] += dpp_mov<0x128>(s[i]);
            if constexpr (NT == 3) s[i] += s2[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 2 * i + (lane >> 5);
            u32x4_t v = tl.v[i];
            if (has_new && t0 + r >= pos) {
                v = *reinterpret_cast<const u32x4_t*>(&L.vnew[8 * (lane & 31)]);
                asm volatile("" : "+v"(v));
            }
            *reinterpret_cast<u32x4_t*>(&L.vs[r * kTailStride + 8 * (lane & 31)]) = v;
        }
        float tmax = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = t0 + 4 * kb + i >= p_end ? -INFINITY : bad ? __builtin_nanf("") : s[i] * sc;
            tmax = fmaxf(tmax, s[i]);
        }
        tmax = fmaxf(tmax, __shfl_xor(tmax, 16, 64));
        tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
        if (__any(tmax > m_run + kLazyMax)) {
            const float m_new = tmax > m_run + kLazyMax ? tmax : m_run;
            const float alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            d_run *= alpha;
            float al[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) al[i] = __shfl(alpha, 4 * kb + i, 64);
#pragma unroll
            for (int jd = 0; jd < 16; ++jd)
#pragma unroll
                for (int i = 0; i < 4; ++i) oacc[jd][i] *= al[i];
        }
        const float mb = m_run - kShift<KV_F16>;
        float pe[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pe[i] = __builtin_amdgcn_exp2f(s[i] - mb);
            d_run += pe[i];
        }
        // A of O += P V (16x16x16): row n = head n & 7, k = positions 4 kb ..
        // + 3; first term in rows 0-7, second in rows 8-15; the third in rows
        // 0-7 of a product of its own
        uint32_t w0[NT], w1[NT];
        split_terms<KV_F16, NT>(pe[0], pe[1], w0);
        split_terms<KV_F16, NT>(pe[2], pe[3], w1);
        const u32x2_t pa = n < 8 ? u32x2_t{w0[0], w1[0]} : u32x2_t{w0[1], w1[1]};
        const u32x2_t pb = n < 8 ? u32x2_t{w0[NT - 1], w1[NT - 1]} : u32x2_t{0u, 0u};
        paged_wave_sync();
        const uint16_t* vsrc = &L.vs[(4 * kb + (n >> 2)) * kTailStride + 4 * (n & 3)];
#pragma unroll
        for (int jd = 0; jd < 16; ++jd) {
            const u32x2_t vb = lds_read_tr16(vsrc + 16 * jd);
            oacc[jd] = KV_F16 ? mfma_16x16x16_f16(pa, vb, oacc[jd]) : mfma_16x16x16_bf16(pa, vb, oacc[jd]);
            if constexpr (NT == 3)
                oacc[jd] = KV_F16 ? mfma_16x16x16_f16(pb, vb, oacc[jd]) : mfma_16x16x16_bf16(pb, vb, oacc[jd]);
        }
        paged_wave_sync();
    };
    int t0 = p_start;
    for (; t0 + kTailTile < p_end; t0 += 2 * kTailTile) {
        bad_b = load(tb, t0 + kTailTile);
        compute(ta, t0, bad_a);
        bad_a = load(ta, t0 + 2 * kTailTile);
        compute(tb, t0 + kTailTile, bad_b);
    }
    if (t0 < p_end) compute(ta, t0, bad_a);

    d_run += __shfl_xor(d_run, 16, 64);
    d_run += __shfl_xor(d_run, 32, 64);
    const size_t slot = (static_cast<size_t>(seq) * 2 + kvh) * pp.cstride +
                        (SHARED ? chunks_of(plan.shared, ch.pfx) : 0) + c;
    if (lane < 8) {
        pp.m[slot * 8 + lane] = m_run - kShift<KV_F16>;
        pp.d[slot * 8 + lane] = d_run;
    }
    // rows 0-7 (lanes 0-31) and 8-15 (lanes 32-63) of O add up to the 8 heads
#pragma unroll
    for (int jd = 0; jd < 16; ++jd)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(oacc[jd][i]), __float_as_uint(oacc[jd][i]),
                                                            false, false);
            oacc[jd][i] = __uint_as_float(h[0]) + __uint_as_float(h[1]);
        }
    if (kb < 2) {
        float* o = pp.o + slot * 8 * 256;
#pragma unroll
        for (int jd = 0; jd < 16; ++jd)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[(4 * kb + i) * 256 + 16 * jd + n] = oacc[jd][i];
    }
}

// ---- combine ----------------------------------------------------------------------------
//
// grid (16 q heads x DS dim blocks, batch), 512 threads, 256 / DS dims a
// workgroup: chunk weights one thread a chunk; 8 DS streams of float4 lanes,
// stream s adding chunks s, s + 8 DS, ... in order, then the streams in a fixed
// order (results do not depend on timing). The (m, d) of every slot and the
// gate are requested before the split is known, and a stream's first four rows
// before the weights; every load is unconditional, its index clamped.
template <int IN_DT, int OUT_DT, int DS, bool SHARED>
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
    const LanePlan p0 = lane_plan<SHARED>(a, 0, lane);
    const Chunks ch = chunk_lengths<SHARED>(a, p0, lane);
    const LanePlan mine = seq < 64 ? p0 : lane_plan<SHARED>(a, seq & ~63, lane);
    const int len = __builtin_amdgcn_readlane(mine.len, seq & 63);
    const int shared = __builtin_amdgcn_readlane(mine.shared, seq & 63);
    if (len == 0) {   // (uniform over the workgroup)
        if (t < kDims) elem<OUT_DT>::store(out, qi * 256 + d0 + t, __builtin_nanf(""));
        return;
    }
    const int nc = (SHARED ? chunks_of(shared, ch.pfx) : 0) + chunks_of(len - shared, ch.own);   // <= cstride
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
    const bool shared = group != nullptr;
    const int lg = __builtin_ctz(static_cast<unsigned>(kv->page_size));
    const PagedKv pk{static_cast<uint16_t*>(kv->k), static_cast<uint16_t*>(kv->v), kv->table, kv->num_pages, lg,
                     kv->table_cols};
    const int cap = gqa_chunk_cap(ctx->cfg, batch);
    PagedSeqs a{positions, group, shared_len, batch, kv->table_cols << lg, 0, 0, cap, 0};
    a.target = batch == 1 ? ctx->num_cu : 2 * ctx->num_cu;
    if (shared) {
        a.target_pfx = ctx->num_cu / 2;
        a.cap_pfx = cap / 2;
        a.cap = cap - a.cap_pfx;
    }
    const PagedPartials pp{ctx->gqa_m, ctx->gqa_d, ctx->gqa_o, cap};
    const RopeFreqs rf = rope_freqs(p->rope_theta);
    const bool f16 = p->kv_f16 != 0, in16 = in_dtype == QFF_BF16, out16 = out_dtype == QFF_BF16;
    if (shared && batch > 1) {
        ProfScope prof(ctx, stream, "gqa_paged_prefix");
        const int grid = 2 * (a.target_pfx + batch / 2);
#define QFF_PFX(I, F, N)                                                                                             \
    gqa_paged_prefix_kernel<I, F, N><<<grid, 512, 0, stream>>>(q_gate, p->q_norm_w, rf, p->scale, p->eps, \
                                                                            pk, a, pp)
        if (f16) {
            if (in16) QFF_PFX(1, 1, 2); else QFF_PFX(0, 1, 2);
        } else if (out16) {
            if (in16) QFF_PFX(1, 0, 2); else QFF_PFX(0, 0, 2);
        } else {
            if (in16) QFF_PFX(1, 0, 3); else QFF_PFX(0, 0, 3);
        }
#undef QFF_PFX
    }
    {
        ProfScope prof(ctx, stream, "gqa_paged_tail");
        const int grid = 2 * (a.target + batch);
#define QFF_TAIL1(I, F, N, S)                                                                                \
    gqa_paged_tail_kernel<I, F, N, S><<<grid, 64, 0, stream>>>(q_gate, k_new, v_new, p->q_norm_w, p->k_norm_w, rf, \
                                                               p->scale, p->eps, pk, a, pp)
#define QFF_TAIL(I, F, N) \
    if (shared) QFF_TAIL1(I, F, N, true); else QFF_TAIL1(I, F, N, false)
        if (f16) {
            if (in16) { QFF_TAIL(1, 1, 2); } else { QFF_TAIL(0, 1, 2); }
        } else if (out16) {
            if (in16) { QFF_TAIL(1, 0, 2); } else { QFF_TAIL(0, 0, 2); }
        } else {
            if (in16) { QFF_TAIL(1, 0, 3); } else { QFF_TAIL(0, 0, 3); }
        }
#undef QFF_TAIL
#undef QFF_TAIL1
    }
    ProfScope prof(ctx, stream, "gqa_paged_combine");
    const int ds = batch <= 8 ? 4 : 1;   // small batches split each head's dims over four workgroups
    const dim3 cgrid(16 * ds, batch);
#define QFF_COMB2(I, O, D, S) gqa_paged_combine_kernel<I, O, D, S><<<cgrid, 512, 0, stream>>>(q_gate, a, pp, out)
#define QFF_COMB1(I, O, D) \
    if (shared) QFF_COMB2(I, O, D, true); else QFF_COMB2(I, O, D, false)
#define QFF_COMB(I, O)                          \
    if (ds == 4) { QFF_COMB1(I, O, 4); }        \
    else { QFF_COMB1(I, O, 1); }
    if (in16) {
        if (out16) { QFF_COMB(1, 1) } else { QFF_COMB(1, 0) }
    } else {
        if (out16) { QFF_COMB(0, 1) } else { QFF_COMB(0, 0) }
    }
#undef QFF_COMB
#undef QFF_COMB1
#undef QFF_COMB2
    return hipGetLastError();
}

}  // namespace qff
