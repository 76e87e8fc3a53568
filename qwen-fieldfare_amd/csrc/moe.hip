// moe.hip -- the expert block on affine-Q4 weights: every token through the
// matrices of its own experts (qff_moe_gate_up, qff_moe_down).
//
//   h[m, j] = silu(Wg x_m) * (Wu x_m),  W of expert indices[m, j]
//   y[m]    = residual + sum_j score[m, j] Wd h[m, j]
//
// Three forms, by how many pairs (token, slot) a call has and how many an expert
// (the figures stand at kOneUp): each pair by itself, small tiles of an expert's pairs,
// large tiles.
//
// A weight is W = s q + b, q the nibble. Pairs by themselves take the nibble as
// the bf16 1 + q / 16 (its four bits are the top ones of the mantissa:
// (q << 3) | 0x3F80, exact), so that per group of 64 columns, with
// P = sum (1 + q / 16) x and X = sum x (a product with ones, from the same
// operands),
//   sum W x = 16 s P + (b - 16 s) X,
// accumulated in fp32. Scales and biases thus enter exactly, x as its bf16
// terms: one for bf16, two for fp16 (11 bits, exact), three for fp32 (24
// bits, exact but for what lies below fp32's own last bit).
//
// Within each 8-column word the matrix-core k order is (c0, c4, c1, c5, c2, c6,
// c3, c7): dword j of a converted word is the pair (q_j, q_j+4), one shift and
// one and-or. A lane's 16-byte load holds four words of one group; lanes
// 0 .. 31 of a 16-row tile hold the first group of a 128-column span, lanes
// 32 .. 63 the second, and a permlane32 swap of two words gives every lane
// quarter kg the words 4 (kg & 1) + 2 (kg >> 1) + {0, 1} of each group: 16
// consecutive columns, which is what the lane reads of x.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "internal.hpp"
#include "mfma.hpp"

namespace qff {

namespace {

struct MoeMat {
    const uint32_t* w;
    const uint16_t* s;
    const uint16_t* b;
};

// One half of the expert block: MATS matrices (gate and up, or down) of `rows`
// x `cols` for each routed expert (m) and for the shared one (sh).
struct MoeArgs {
    MoeMat m[2], sh[2];
    const void* x;
    const int32_t* indices;
    int experts, top, slots, rows, cols, tokens;   // slots = top + 1 with a shared expert
};

// A (token, slot) pair in one int: slots are at most 17.
__device__ __forceinline__ int pair_code(int m, int j) { return m * 32 + j; }

__device__ __forceinline__ MoeMat moe_matrix(const MoeMat& routed, const MoeMat& shared, bool is_shared, int e, int rows,
                                             int cols) {
    if (is_shared) return shared;
    const size_t r = static_cast<size_t>(e) * rows;
    return MoeMat{routed.w + r * (cols / 8), routed.s + r * (cols / 64), routed.b + r * (cols / 64)};
}

// Nibble word -> the bf16 pairs 1 + q / 16 in the k order above: a shift and
// an and-or (q4_one() and the mask are kept in registers; as inline assembly the
// and-or's result could meet the late write of a matrix instruction whose
// registers it takes over, which only the compiler's own instructions wait for).
__device__ __forceinline__ uint32_t q4_one() {
    uint32_t one = 0x3F803F80u;
    asm("" : "+v"(one));
    return one;
}
__device__ __forceinline__ u32x4_t q4_to_bf16(uint32_t w, uint32_t one) {
    u32x4_t r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = ((j == 0 ? w << 3 : w >> (4 * j - 3)) & 0x00780078u) | one;
    return r;
}

// bf16 terms of a value of x that hold all of it.
constexpr int x_terms(int dtype) { return dtype == 0 ? 3 : dtype == 1 ? 1 : 2; }

// The words of a 128-column span's two groups for this lane's quarter: w[2 gi
// + step] feeds k step `step` of group gi.
__device__ __forceinline__ void span_words(const u32x4_t& u, uint32_t (&w)[4]) {
    const auto a = __builtin_amdgcn_permlane32_swap(u[0], u[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(u[1], u[3], false, false);
    w[0] = a[0];
    w[1] = b[0];
    w[2] = a[1];
    w[3] = b[1];
}

constexpr int kGroups = 4;   // groups of 64 columns that a wave requests at once: two 128-column spans

// ---- one token at a time ------------------------------------------------------
//
// A tile is 16 weight rows against one token, x as the A operand (the same
// token in all 16 rows) and the weights as B, so that a lane's accumulator is its
// own weight row's sum (lane & 15) and needs that row's scale alone. A wave takes
// 256 columns at a time: each lane splits four of them into terms, which all read
// back from the wave's own LDS (split by every lane for itself they took more
// instructions than the weights: gate and up of a token 13.4 us).
constexpr int kOneWaves = 8, kChunk = 64 * kGroups;

// A lane's four columns of x, and their terms in the k order.
template <int X_DT>
struct XFour {
    static constexpr int kTerms = x_terms(X_DT);
    float v[4];
    __device__ __forceinline__ void load(const void* x, size_t i) {
        if constexpr (X_DT == 0) {
            const f32x4_t f = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(x) + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = f[k];
        } else {
            const u32x2_t u = *reinterpret_cast<const u32x2_t*>(static_cast<const uint16_t*>(x) + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint16_t h = static_cast<uint16_t>(u[k / 2] >> (16 * (k & 1)));
                v[k] = elem<X_DT>::load(&h, 0);
            }
        }
    }
    // to: [kTerms][kChunk]. Even lanes hold columns 0-3 of a word of 8 and write its first two pairs (c0, c4), (c1, c5),
    // odd ones hold 4-7 and write the others.
    __device__ __forceinline__ void split(uint16_t* to, int lane) const {
        const bool odd = lane & 1;
        float a[2], b[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float give = odd ? v[j] : v[2 + j], take = dpp_mov<0xB1>(give);   // (the neighbour's, lane ^ 1)
            a[j] = odd ? take : v[j];
            b[j] = odd ? v[2 + j] : take;
        }
#pragma unroll
        for (int q = 0; q < kTerms; ++q) {
            u32x2_t t;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                t[j] = pack_bf16x2(a[j], b[j]);
                a[j] -= __uint_as_float(t[j] << 16);
                b[j] -= __uint_as_float(t[j] & 0xffff0000u);
            }
            *reinterpret_cast<u32x2_t*>(to + q * kChunk + 4 * lane) = t;
        }
    }
};

template <int X_DT, int SB_DT, int MATS>
struct OneStep {
    u32x4_t w[MATS][kGroups / 2];
    XFour<X_DT> x;
    u32x2_t s[MATS], b[MATS];

    // x of groups g0 .. g0 + 3 (columns past the last are requested as the row's last four and not used)
    __device__ __forceinline__ void load_x(const void* xp, size_t xrow, int cols, int g0, int lane) {
        x.load(xp, xrow + min(64 * g0 + 4 * lane, cols - 4));
    }
    // their words, scales and biases (those past the last group are requested as the last's and not used)
    __device__ __forceinline__ void load_w(const MoeMat (&m)[MATS], int row, int cols, int g0, int kg) {
        const int G = cols / 64;
        const size_t r = static_cast<size_t>(row);
#pragma unroll
        for (int i = 0; i < MATS; ++i) {
#pragma unroll
            for (int sp = 0; sp < kGroups / 2; ++sp)
                w[i][sp] = *reinterpret_cast<const u32x4_t*>(m[i].w + r * (cols / 8) +
                                                             8 * min(g0 + 2 * sp + (kg >> 1), G - 1) + 4 * (kg & 1));
            // (in one load each where rows begin on 8 bytes: two-byte ones took gate and up of a token 4 us)
            const size_t at = r * G;
            if ((G & 3) == 0 && ((reinterpret_cast<uintptr_t>(m[i].s) | reinterpret_cast<uintptr_t>(m[i].b)) & 7) == 0) {
                s[i] = *reinterpret_cast<const u32x2_t*>(m[i].s + at + g0);
                b[i] = *reinterpret_cast<const u32x2_t*>(m[i].b + at + g0);
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const size_t g = at + min(g0 + 2 * k, G - 1), h = at + min(g0 + 2 * k + 1, G - 1);
                    s[i][k] = m[i].s[g] | static_cast<uint32_t>(m[i].s[h]) << 16;
                    b[i][k] = m[i].b[g] | static_cast<uint32_t>(m[i].b[h]) << 16;
                }
            }
        }
    }
    // xs: the wave's own [kTerms][kChunk]
    __device__ __forceinline__ void add(float (&acc)[MATS], int groups, uint16_t* xs, int lane) const {
        constexpr int T = x_terms(X_DT);
        const int kg = lane >> 4;
        const uint32_t one = q4_one();
        const u32x4_t ones{one, one, one, one};
        x.split(xs, lane);
        uint32_t words[MATS][kGroups / 2][4];
#pragma unroll
        for (int i = 0; i < MATS; ++i)
#pragma unroll
            for (int sp = 0; sp < kGroups / 2; ++sp) span_words(w[i][sp], words[i][sp]);
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            if (k >= groups) break;
            f32x4_t P[MATS], X{};
#pragma unroll
            for (int i = 0; i < MATS; ++i) P[i] = f32x4_t{};
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                u32x4_t t[T];
#pragma unroll
                for (int j = 0; j < T; ++j)
                    t[j] = *reinterpret_cast<const u32x4_t*>(xs + j * kChunk + 64 * k + 32 * (kg & 1) + 16 * (kg >> 1) + 8 * st);
#pragma unroll
                for (int j = T - 1; j >= 0; --j) X = mfma_16x16x32_bf16(t[j], ones, X);
#pragma unroll
                for (int i = 0; i < MATS; ++i) {
                    const u32x4_t q = q4_to_bf16(words[i][k / 2][2 * (k % 2) + st], one);
#pragma unroll
                    for (int j = T - 1; j >= 0; --j) P[i] = mfma_16x16x32_bf16(t[j], q, P[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < MATS; ++i) {
                const uint16_t sk = static_cast<uint16_t>(s[i][k / 2] >> (16 * (k & 1)));
                const uint16_t bk = static_cast<uint16_t>(b[i][k / 2] >> (16 * (k & 1)));
                const float sc = 16.0f * elem<SB_DT>::load(&sk, 0), bi = elem<SB_DT>::load(&bk, 0);
                acc[i] = fmaf(sc, P[i][0], fmaf(bi - sc, X[0], acc[i]));
            }
        }
    }
};

// Gate and up: one workgroup per (16 rows, pair), its waves over K.
template <int X_DT, int SB_DT, int H_DT>
__global__ __launch_bounds__(64 * kOneWaves) void moe_gate_up_one_kernel(MoeArgs p, void* __restrict__ h) {
    __shared__ __attribute__((aligned(16))) uint16_t xs[kOneWaves][x_terms(X_DT) * kChunk];
    __shared__ float red[kOneWaves][2][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, kg = lane >> 4;
    const int tok = blockIdx.y / p.slots, j = blockIdx.y % p.slots, G = p.cols / 64, row0 = 16 * blockIdx.x;
    const bool shared = j >= p.top;
    const int e = shared ? 0 : p.indices[tok * p.top + j];
    OneStep<X_DT, SB_DT, 2> st;
    st.load_x(p.x, static_cast<size_t>(tok) * p.cols, p.cols, kGroups * wave, lane);   // (ahead of the expert's number)
    if (e < 0 || (!shared && e >= p.experts)) return;
    const MoeMat m[2] = {moe_matrix(p.m[0], p.sh[0], shared, e, p.rows, p.cols),
                         moe_matrix(p.m[1], p.sh[1], shared, e, p.rows, p.cols)};
    float acc[2] = {0.0f, 0.0f};
    for (int g0 = kGroups * wave; g0 < G; g0 += kGroups * kOneWaves) {
        st.load_w(m, row0 + c, p.cols, g0, kg);
        if (g0 != kGroups * wave) st.load_x(p.x, static_cast<size_t>(tok) * p.cols, p.cols, g0, lane);
        st.add(acc, G - g0, xs[wave], lane);
    }
    if (lane < 16) {
        red[wave][0][lane] = acc[0];
        red[wave][1][lane] = acc[1];
    }
    __syncthreads();
    if (threadIdx.x < 16) {
        float a = 0.0f, u = 0.0f;
#pragma unroll
        for (int w = 0; w < kOneWaves; ++w) {
            a += red[w][0][threadIdx.x];
            u += red[w][1][threadIdx.x];
        }
        elem<H_DT>::store(h, static_cast<size_t>(blockIdx.y) * p.rows + row0 + threadIdx.x, silu(a) * u);
    }
}

// Down: one workgroup per (16 rows, token), its waves over (slot, four groups);
// sums in the order of the waves and, within one, of the slots.
template <int X_DT, int SB_DT, int Y_DT>
__global__ __launch_bounds__(64 * kOneWaves) void moe_down_one_kernel(MoeArgs p, const float* __restrict__ scores,
                                                                      const float* __restrict__ coef, const void* residual,
                                                                      void* y) {
    __shared__ __attribute__((aligned(16))) uint16_t xs[kOneWaves][x_terms(X_DT) * kChunk];
    __shared__ float red[kOneWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, kg = lane >> 4;
    const int tok = blockIdx.y, row0 = 16 * blockIdx.x, G = p.cols / 64, steps = (G + kGroups - 1) / kGroups;
    const size_t o = static_cast<size_t>(tok) * p.rows + row0 + c;
    const float res = residual ? elem<Y_DT>::load(residual, o) : 0.0f;
    float acc = 0.0f;
    // the next item's loads ahead of an item's products
    struct Item {
        OneStep<X_DT, SB_DT, 1> st;
        float f;
        int g0;
        bool has;
    };
    const int items = p.slots * steps;
    auto fetch = [&](int it, Item& q) {
        const int j = it / steps;
        const bool shared = j >= p.top;
        const int e = it >= items ? -1 : shared ? 0 : p.indices[tok * p.top + j];
        q.g0 = kGroups * (it - j * steps);
        q.has = e >= 0 && (shared || e < p.experts);
        if (!q.has) return;
        const MoeMat m[1] = {moe_matrix(p.m[0], p.sh[0], shared, e, p.rows, p.cols)};
        q.f = shared ? (coef ? coef[tok] : 1.0f) : scores[tok * p.top + j];
        q.st.load_w(m, row0 + c, p.cols, q.g0, kg);
        q.st.load_x(p.x, (static_cast<size_t>(tok) * p.slots + j) * p.cols, p.cols, q.g0, lane);
    };
    Item q;
    fetch(wave, q);
    for (int it = wave; it < items; it += kOneWaves) {
        Item next;
        fetch(it + kOneWaves, next);
        if (q.has) {
            float a[1] = {0.0f};
            q.st.add(a, G - q.g0, xs[wave], lane);
            acc = fmaf(q.f, a[0], acc);
        }
        q = next;
    }
    if (lane < 16) red[wave][lane] = acc;
    __syncthreads();
    if (threadIdx.x < 16) {
        float a = res;
#pragma unroll
        for (int w = 0; w < kOneWaves; ++w) a += red[w][threadIdx.x];
        elem<Y_DT>::store(y, o, a);
    }
}

// ---- several tokens of one expert ------------------------------------------------

// Which pairs each expert has, and the tiles of up to `most` that they make: the
// pairs are counted, the counts summed up and the pairs written expert by expert
// (in no fixed order within one: a pair's sums do not depend on its place). An expert's tiles share its pairs evenly, in multiples of `unit`
// (8 to 32); the shared expert, number `experts`, has every token. Up to kPlanAlone
// pairs one workgroup does it all (6 us at 4000 pairs, 69 at 65536; by several 13);
// beyond, a workgroup for
// each kPlanShare pairs counts its own, and each then sums up those before it.
constexpr int kPlanThreads = 1024, kPlanShare = 1024, kPlanAlone = 4096;
static_assert(kMoeMaxExperts < kPlanThreads, "an expert a thread");

__global__ __launch_bounds__(kPlanThreads) void moe_count_kernel(const int32_t* __restrict__ indices, int experts, int n,
                                                                 int* __restrict__ parts) {
    __shared__ int cnt[kMoeMaxExperts];
    const int t = threadIdx.x, i = blockIdx.x * kPlanShare + t;
    if (t < experts) cnt[t] = 0;
    __syncthreads();
    const int e = i < n ? indices[i] : -1;
    if (e >= 0 && e < experts) atomicAdd(&cnt[e], 1);
    __syncthreads();
    if (t < experts) parts[static_cast<size_t>(blockIdx.x) * experts + t] = cnt[t];
}

struct PlanArgs {
    const int32_t* indices;
    int experts, top, tokens, shared, most, unit;
    const int* parts;   // or null: one workgroup
    int* count;
    int4* tiles;
    int* list;
};
__device__ __forceinline__ void moe_plan(const PlanArgs& q, int blocks) {
    const int32_t* const indices = q.indices;
    const int* const parts = q.parts;
    const int experts = q.experts, most = q.most, unit = q.unit;
    __shared__ int cnt[kMoeMaxExperts], at[kMoeMaxExperts], wsum[2][kPlanThreads / 64];
    const int t = threadIdx.x, n = q.tokens * q.top, share = parts ? kPlanShare : n, i0 = blockIdx.x * share, i1 = min(i0 + share, n);
    int mine = 0;   // pairs of expert t that other workgroups write ahead of this one's
    if (parts) {
        int all = 0;
        if (t < experts) {
#pragma unroll 8
            for (int b = 0; b < blocks; ++b) {
                const int c = parts[static_cast<size_t>(b) * experts + t];
                all += c;
                mine += b < static_cast<int>(blockIdx.x) ? c : 0;
            }
            cnt[t] = all;
        }
    } else {
        if (t < kMoeMaxExperts) cnt[t] = 0;
        __syncthreads();
        for (int i = i0 + t; i < i1; i += kPlanThreads) {
            const int e = indices[i];
            if (e >= 0 && e < experts) atomicAdd(&cnt[e], 1);
        }
    }
    __syncthreads();
    const int own = t < experts ? cnt[t] : t == experts && q.shared ? q.tokens : 0;
    const int own_tiles = (own + most - 1) / most;
    const int incl = wave_inclusive_scan_int(t < experts ? own : 0), incl_tiles = wave_inclusive_scan_int(own_tiles);
    if ((t & 63) == 63) {
        wsum[0][t >> 6] = incl;
        wsum[1][t >> 6] = incl_tiles;
    }
    __syncthreads();
    int before = incl - own, tile = incl_tiles - own_tiles;
    for (int w = 0; w < t >> 6; ++w) {
        before += wsum[0][w];
        tile += wsum[1][w];
    }
    if (t < experts) at[t] = before + mine;
    if (blockIdx.x == 0) {
        if (t == experts) {
            *q.count = tile + own_tiles;
            before = 0;   // (its pairs are the tokens themselves)
        }
        if (own_tiles > 0) {
            const int each = ((own + own_tiles - 1) / own_tiles + unit - 1) / unit * unit;
            // (rounded up, the last tiles may have fewer or none)
            for (int k = 0; k < own_tiles; ++k)
                q.tiles[tile + k] = make_int4(t, before + k * each, min(each, max(own - k * each, 0)), 0);
        }
    }
    __syncthreads();
    for (int i = i0 + t; i < i1; i += kPlanThreads) {
        const int e = indices[i];
        if (e >= 0 && e < experts) q.list[atomicAdd(&at[e], 1)] = pair_code(i / q.top, i % q.top);
    }
}
__global__ __launch_bounds__(kPlanThreads) void moe_plan_kernel(PlanArgs q) { moe_plan(q, gridDim.x); }

// y[m] = residual[m] + the rows of its pairs, in their order.
template <int Y_DT>
__global__ __launch_bounds__(256) void moe_combine_kernel(const float* __restrict__ part, const int32_t* __restrict__ indices,
                                                          int experts, int top, int slots, const void* residual, void* y,
                                                          int rows) {
    const int m = blockIdx.y, r = 4 * (blockIdx.x * 256 + threadIdx.x);
    if (r >= rows) return;
    const size_t o = static_cast<size_t>(m) * rows + r;
    f32x4_t a{};
    if (residual) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = elem<Y_DT>::load(residual, o + i);
    }
    for (int j = 0; j < slots; ++j) {
        const int e = j < top ? indices[m * top + j] : 0;
        if (e < 0 || (j < top && e >= experts)) continue;
        a += *reinterpret_cast<const f32x4_t*>(part + (static_cast<size_t>(m) * slots + j) * rows + r);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) elem<Y_DT>::store(y, o + i, a[i]);
}

// ---- many tokens ------------------------------------------------------------------
//
// The plan's tiles against the matrices on 32x32x16 fp16 products. A weight is
// s q + b = s (q - 8) + (b + 8 s); its first part is exact in fp16 where the scale has 8 significant bits (bf16): q - 8 is a power of two
// or has three bits. The nibble becomes 16 + q (its bits are the top ones of the
// mantissa), one packed FMA (16 + q) s - 24 s gives the product without a rounding,
// and the second part, constant over a group, meets the group's sums of x in a few
// products at the end. An fp16 scale (11 bits) is split into its first eight bits
// and the rest, two products a weight (WT = 2), where the output's precision needs
// it; for bf16 outputs (q - 8) s is rounded to fp16 (WT = 1).
// x enters as fp16 after a power-of-two shift that puts its row's largest
// magnitude into [2^13, 2^14), for fp32 x and F32 or F16 outputs as two terms of 11
// bits (XT = 2); fp16 rows of h are taken as they lie. The scale enters as 64 s: at 31 the
// FMA's 24 (64 s) is 47616, inside fp16 (256 s left it from 10.7 on), and at 2^-22 the last
// of eight bits is one of fp16's smallest numbers, 2^-23, which the FMA and the matrix
// cores take as they are; b + 8 s may be up to 8 in magnitude.
// So F32 and F16 outputs are sums of exact products (up to 2^-22 of x), and
// bf16 ones carry 11 bits an operand (a bf16 result has 8) from 33 tokens on.

// Rows of x for the tiles: XT fp16 terms [row][XT][cols] (each 8 columns in the
// order c0, c4, c1, c5, .., the nibbles' own) and the row's factor 2^(e - 6); and
// the sums of its groups as two fp16 terms [row][2][gp] (gp: groups rounded up to
// 16, the rest zeros), shifted as x is, with the factor that takes them back. One
// wave a row. COPY false (fp16 rows, used where they lie): the sums alone.
constexpr int kX16Waves = 4;
constexpr int kSumsPad = 16;
template <int X_DT, int XT, bool COPY>
__device__ __forceinline__ void moe_x16(const void* __restrict__ x, uint16_t* __restrict__ x16, float2* __restrict__ fac,
                                        uint16_t* __restrict__ sums, int cols, int row) {
    const int lane = threadIdx.x & 63, nb = cols / 8;
    constexpr int kMax = 8;   // 8-column blocks of a lane: cols <= 4096
    float v[kMax][8], s[kMax];
    float mx = 0.0f, ms = 0.0f;
#pragma unroll
    for (int i = 0; i < kMax; ++i) {
        s[i] = 0.0f;
        if (64 * i >= nb) continue;
        const int b = min(lane + 64 * i, nb - 1);
        const size_t o = static_cast<size_t>(row) * cols + 8 * b;
        if constexpr (X_DT == 0) {
            const f32x4_t* q = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(x) + o);
            const f32x4_t a = q[0], c = q[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[i][e] = a[e];
                v[i][4 + e] = c[e];
            }
        } else {
            const u32x4_t u = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(x) + o);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint16_t w[2] = {static_cast<uint16_t>(u[e]), static_cast<uint16_t>(u[e] >> 16)};
                v[i][2 * e] = elem<X_DT>::load(w, 0);
                v[i][2 * e + 1] = elem<X_DT>::load(w, 1);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (COPY) mx = fmaxf(mx, fabsf(v[i][e]));
            s[i] += v[i][e];
        }
        s[i] = group_sum<8>(s[i]);   // (nb is a multiple of 8: a group's eight lanes are all in or all past the end)
        ms = fmaxf(ms, fabsf(s[i]));
    }
    // (exponents of at least -127 keep their powers finite for the smallest rows)
    const auto shift = [](float m) { return m > 0.0f ? max(__builtin_amdgcn_frexp_expf(m) - 14, -127) : 0; };
    const int e = COPY ? shift(group_max<64>(mx)) : 0, es = shift(group_max<64>(ms));
    if (lane == 0) fac[row] = make_float2(ldexpf(1.0f, e - 6), ldexpf(1.0f, es - e - 6));
    const float p = ldexpf(1.0f, -e), ps = ldexpf(1.0f, -es);
    const int G = cols / 64, gp = (G + kSumsPad - 1) / kSumsPad * kSumsPad;
    uint16_t* const so = sums + static_cast<size_t>(row) * 2 * gp;
#pragma unroll
    for (int i = 0; i < kMax; ++i) {
        const int g = 8 * i + lane / 8;
        if (g < gp && (lane & 7) == 0) {
            uint32_t hi, lo;
            split_f16x2(g < G ? s[i] * ps : 0.0f, 0.0f, hi, lo);
            so[g] = static_cast<uint16_t>(hi);
            so[gp + g] = static_cast<uint16_t>(lo);
        }
        if constexpr (COPY) {
            const int b = lane + 64 * i;
            if (64 * i >= nb || b >= nb) continue;
            u32x4_t h, l;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (XT == 2) {
                    uint32_t hi, lo;
                    split_f16x2(v[i][j] * p, v[i][j + 4] * p, hi, lo);
                    h[j] = hi;
                    l[j] = lo;
                } else {
                    h[j] = pack_f16x2(v[i][j] * p, v[i][j + 4] * p);
                }
            }
            uint16_t* o = x16 + static_cast<size_t>(row) * XT * cols + 8 * b;
            *reinterpret_cast<u32x4_t*>(o) = h;
            if constexpr (XT == 2) *reinterpret_cast<u32x4_t*>(o + cols) = l;
        }
    }
}
template <int X_DT, int XT, bool COPY>
__global__ __launch_bounds__(64 * kX16Waves) void moe_x16_kernel(const void* __restrict__ x, uint16_t* __restrict__ x16,
                                                                 float2* __restrict__ fac, uint16_t* __restrict__ sums,
                                                                 int cols, int rows) {
    const int row = blockIdx.x * kX16Waves + (threadIdx.x >> 6);
    if (row < rows) moe_x16<X_DT, XT, COPY>(x, x16, fac, sums, cols, row);
}
// The same and a plan of one workgroup in one launch (a launch less is 6 us of 60
// at 32 tokens).
template <int X_DT, int XT, bool COPY>
__global__ __launch_bounds__(kPlanThreads) void moe_prepare_kernel(PlanArgs q, const void* __restrict__ x, uint16_t* __restrict__ x16,
                                                                   float2* __restrict__ fac, uint16_t* __restrict__ sums,
                                                                   int cols, int rows) {
    if (blockIdx.x == 0) return moe_plan(q, 1);
    const int row = (blockIdx.x - 1) * (kPlanThreads / 64) + (threadIdx.x >> 6);
    if (row < rows) moe_x16<X_DT, XT, COPY>(x, x16, fac, sums, cols, row);
}

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// A group's scale for one row of the tile: 64 s (its first eight bits for WT = 2)
// and the rest of it.
template <int WT>
using tile_sb = std::conditional_t<WT == 1, uint16_t, uint32_t>;
template <int SB_DT, int WT>
__device__ __forceinline__ tile_sb<WT> tile_scale(uint16_t s) {
    const float v = 64.0f * elem<SB_DT>::load(&s, 0);
    if constexpr (WT == 1) {
        return f32_to_f16(v);
    } else {
        const float hi = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
        return f32_to_f16(hi) | static_cast<uint32_t>(f32_to_f16(v - hi)) << 16;
    }
}

// Nibble word -> fp16 pairs 64 s (q - 8): the pairs (q_j, q_j+4), or with NATURAL
// (q_2j, q_2j+1) from the even and the odd nibbles' bytes.
template <bool EXACT, bool NATURAL>
__device__ __forceinline__ u32x4_t q4_to_f16(uint32_t w, f16x2_t s, f16x2_t c, uint32_t k16) {
    u32x4_t r;   // (k16: the fp16 pair 16, 16 in a register, for one and-or or shift-or a pair)
    const uint32_t even = w & 0x0f0f0f0fu, odd = w >> 4 & 0x0f0f0f0fu;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t e;
        if constexpr (NATURAL) {
            e = __builtin_amdgcn_perm(odd, even, 0x0c040c00u + 0x00010001u * j) << 6 | k16;
        } else {
            e = ((j < 2 ? w << (6 - 4 * j) : w >> (4 * j - 6)) & 0x03C003C0u) | k16;
        }
        const f16x2_t v = __builtin_bit_cast(f16x2_t, e);
        const f16x2_t q = EXACT ? __builtin_elementwise_fma(v, s, c)
                                : (v - f16x2_t{static_cast<_Float16>(24.0f), static_cast<_Float16>(24.0f)}) * s;
        r[j] = __builtin_bit_cast(uint32_t, q);
    }
    return r;
}

constexpr int kXcds = 8;
constexpr int kOutRow = 272;   // bytes of LDS for a token's outputs of one wave: 64 fp32 values and a pad
constexpr int kTileRows = 256;   // weight rows of a workgroup: four waves of 64, in two row tiles of 32

// What the tile kernel reads beside the weights.
struct TileArgs {
    const int* count;
    const int4* tiles;
    const int* list;
    const uint16_t* x16;   // [row][XT][cols]
    const float2* fac;     // [row]: of the products, of the sums' products ahead of that
    const uint16_t* sums;  // [row][2][gp]
};

// Eight consecutive 16-bit values from `at` on, those past `end` the last one.
// vec: 16-byte aligned, and `end` is a multiple of 8 further on.
__device__ __forceinline__ u32x4_t load_u16x8(const uint16_t* __restrict__ p, int at, int end, bool vec) {
    if (vec) return *reinterpret_cast<const u32x4_t*>(p + min(at, end - 8));
    uint16_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[min(at + i, end - 1)];
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = v[2 * i] | static_cast<uint32_t>(v[2 * i + 1]) << 16;
    return r;
}
__device__ __forceinline__ bool sb_vec(const MoeMat& m, int G) {
    return (G & 7) == 0 && ((reinterpret_cast<uintptr_t>(m.s) | reinterpret_cast<uintptr_t>(m.b)) & 15) == 0;
}

// Groups of x and of the weights on their way or in use: as many as LDS holds
// beside a second workgroup.
constexpr int tile_stages(int xt, int mmt) { return mmt == 4 ? 2 : mmt == 2 ? 4 - xt : 5 - xt; }
constexpr int tile_stage_bytes(int xt, int mmt) { return xt * 32 * mmt * 128 + kTileRows * 32; }

// All waves here, each with at most N of its copies still under way (the copies
// are not the compiler's own: its barrier would wait for all of them, and so
// would its reads of LDS behind them).
template <int N>
__device__ __forceinline__ void meet() {
    static_assert(N < 64, "six bits count them");   // (63: any number)
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}
template <int N, class F>
__device__ __forceinline__ void unroll(F&& f) {
    if constexpr (N > 1) unroll<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
}

// Where the constant parts' terms lie in the staging buffer: in the last stage, or
// (more than 16 groups, 32 KB at a time) from its beginning.
__device__ __forceinline__ constexpr int tile_terms_at(int xt, int mmt, int groups) {
    return groups <= 16 ? (tile_stages(xt, mmt) - 1) * tile_stage_bytes(xt, mmt) : 0;
}

// The constant parts' terms of groups k0 .. k0 + 31: (b + 8 s) 2^12 as an fp16 term and
// 2^11 times its rest as another (which meets the sums 2^-11 times), so that 8 stays inside
// fp16 (8 2^13 does not) and 22 bits are there down to 2^-26, an absolute 2^-48 below.
// Thread t forms row t's (of two matrices 32 rows of the first, 32 of the
// second, ..): [16 groups][term][row][16], a row's halves swapped in every other four
// rows. Groups past the last (which meet sums of zero) take its.
template <int MATS>
__device__ __forceinline__ int tile_row(const MoeArgs& p, int row0) {
    const int t = threadIdx.x;
    return min(MATS == 2 ? row0 + 32 * (t >> 6) + (t & 31) : row0 + t, p.rows - 1);
}
template <int SB_DT>
__device__ __forceinline__ void const_terms(const u32x4_t& s8, const u32x4_t& b8, u32x4_t& bh, u32x4_t& bl) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint16_t sq = static_cast<uint16_t>(s8[j] >> (16 * i)), bq = static_cast<uint16_t>(b8[j] >> (16 * i));
            v[i] = 4096.0f * fmaf(8.0f, elem<SB_DT>::load(&sq, 0), elem<SB_DT>::load(&bq, 0));
        }
        const f16x2_t hi = {static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1])};
        bh[j] = __builtin_bit_cast(uint32_t, hi);
        bl[j] = pack_f16x2(2048.0f * (v[0] - static_cast<float>(hi[0])), 2048.0f * (v[1] - static_cast<float>(hi[1])));
    }
}
// Eight sums for the products with bl.
__device__ __forceinline__ u32x4_t rest_sums(const u32x4_t& x) {
    constexpr _Float16 k = static_cast<_Float16>(1.0f / 2048.0f);
    u32x4_t r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, static_cast<uint32_t>(x[j])) * f16x2_t{k, k});
    return r;
}
template <int SB_DT>
__device__ __forceinline__ void put_terms(uint16_t* to, int k, const u32x4_t& s8, const u32x4_t& b8) {
    const int t = threadIdx.x;
    u32x4_t bh, bl;
    const_terms<SB_DT>(s8, b8, bh, bl);
    uint16_t* o = to + k / 16 * 32 * kTileRows + 16 * t + 8 * ((k / 8 & 1) ^ (t >> 2 & 1));
    *reinterpret_cast<u32x4_t*>(o) = bh;
    *reinterpret_cast<u32x4_t*>(o + 16 * kTileRows) = bl;
}
template <int MATS, int SB_DT>
__device__ __forceinline__ void tile_terms(const MoeArgs& p, const MoeMat& m0, const MoeMat& m1, int row0, int k0, uint16_t* to) {
    const int G = p.cols / 64;
    const MoeMat& mm = MATS == 2 && (threadIdx.x & 32) ? m1 : m0;
    const bool vec = sb_vec(m0, G) && sb_vec(m1, G);
    const size_t base = static_cast<size_t>(tile_row<MATS>(p, row0)) * G;
    for (int k = 0; k < 32 && k0 + k < (G + 15) / 16 * 16; k += 8)
        put_terms<SB_DT>(to, k, load_u16x8(mm.s + base, k0 + k, G, vec), load_u16x8(mm.b + base, k0 + k, G, vec));
}

// One tile: 256 weight rows (of gate and up: 128 of each, a wave's two row tiles the
// same rows of both) x NMT tiles of 32 tokens. Groups of x and of the words go from
// global memory into LDS, tile_stages of them in turn, one barrier a group; a
// wave converts its own rows' words in registers. Rows of x are swizzled so that
// the 32 rows of an operand read meet every bank group twice.
template <int MATS, int SB_DT, int XT, int WT, bool NATURAL, int MMT, int NMT, class Out>
__device__ __forceinline__ void tile_run(const MoeArgs& p, const TileArgs& a, const MoeMat& m0, const MoeMat& m1, int row0,
                                         const int* codes, uint16_t* Xl, const tile_sb<WT>* sbl, f32x16_t (&acc)[2][NMT], float2 (&fac)[NMT],
                                         const Out& out) {
    constexpr bool kExact = SB_DT == 1 || WT == 2;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r = lane & 31, h = lane >> 5;
    const int G = p.cols / 64;
    auto x_row = [&](int place) {
        const int code = codes[place];
        return MATS == 2 ? code >> 5 : (code >> 5) * p.slots + (code & 31);
    };
    // A stage holds a group's x [XT][32 MMT tokens][64] and words [wave][2 row tiles][64 lanes][16 bytes]. Copies of x: 8
    // tokens each, lane l the 16-byte piece l & 7 of token l >> 3, which is the token's 8-column block (l & 7) ^ ((token >>
    // 1) & 7) of the group; of words: the wave's own rows', as its lanes read them back.
    constexpr int NS = tile_stages(XT, MMT), kStage = tile_stage_bytes(XT, MMT), kXBytes = XT * 32 * MMT * 128;
    const uint32_t at = lds_addr(Xl);
    uint32_t xoff[NMT], woff[2];
#pragma unroll
    for (int i = 0; i < NMT; ++i) {
        const int tok = 8 * (NMT * wave + i) + (lane >> 3);
        xoff[i] = (static_cast<uint32_t>(x_row(tok)) * XT * p.cols + 8 * ((lane & 7) ^ ((tok >> 1) & 7))) * 2;
    }
    const int wrow = MATS == 2 ? row0 + 32 * wave + r : row0 + 64 * wave + r;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) woff[rt] = static_cast<uint32_t>(min(wrow + (MATS == 2 ? 0 : 32 * rt), p.rows - 1)) * (p.cols / 2) + 16 * h;
    auto stage = [&](int buf, int g) {
#pragma unroll
        for (int x = 0; x < XT; ++x)
#pragma unroll
            for (int i = 0; i < NMT; ++i)
                dma16(reinterpret_cast<const char*>(a.x16) + x * p.cols * 2 + 128 * g, xoff[i],
                      at + buf * kStage + (x * 32 * MMT + 8 * (NMT * wave + i)) * 128);
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
            dma16(reinterpret_cast<const char*>(rt && MATS == 2 ? m1.w : m0.w) + 32 * g, woff[rt],
                  at + buf * kStage + kXBytes + (2 * wave + rt) * 1024);
    };
    uint32_t k16 = 0x4C004C00u;
    asm("" : "+v"(k16));
    // The groups' constant parts: their terms, 32 groups at a time (the first are there already), against the rows' sums.
    // Up to 16 groups the terms lie in the last stage and the first copies are on their way meanwhile; they are asked for
    // behind the sums, since the wait for these is the compiler's, which does not count copies.
    const bool early = G <= 16;
    {
        const int gp = (G + kSumsPad - 1) / kSumsPad * kSumsPad;
        const uint16_t* S[NMT];
#pragma unroll
        for (int mt = 0; mt < NMT; ++mt) {
            const size_t row = x_row(32 * mt + r);
            S[mt] = a.sums + row * 2 * gp + 8 * h;
            fac[mt] = a.fac[row];
            fac[mt].x *= out.weight(codes[32 * mt + r]);
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[rt][mt][i] = 0.0f;
        }
        const uint16_t* const terms = Xl + tile_terms_at(XT, MMT, G) / 2;
        for (int k0 = 0; k0 < G; k0 += 16) {
            u32x4_t xh[NMT], xl[NMT], xr[NMT];
#pragma unroll
            for (int mt = 0; mt < NMT; ++mt) {
                xh[mt] = *reinterpret_cast<const u32x4_t*>(S[mt] + k0);
                xl[mt] = *reinterpret_cast<const u32x4_t*>(S[mt] + gp + k0);
            }
            if (k0 && k0 % 32 == 0) {
                __syncthreads();   // (the terms before have been read)
                tile_terms<MATS, SB_DT>(p, m0, m1, row0, k0, Xl + tile_terms_at(XT, MMT, G) / 2);
                __syncthreads();
            }
            __builtin_amdgcn_sched_barrier(0);
            if (early) {
#pragma unroll
                for (int i = 0; i < NS - 1; ++i) stage(i, min(i, G - 1));
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int mt = 0; mt < NMT; ++mt) xr[mt] = rest_sums(xh[mt]);
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
                const int q = 64 * wave + 32 * rt + r;
                const uint16_t* o = terms + k0 % 32 * 2 * kTileRows + 16 * q + 8 * (h ^ (q >> 2 & 1));
                const u32x4_t bh = *reinterpret_cast<const u32x4_t*>(o), bl = *reinterpret_cast<const u32x4_t*>(o + 16 * kTileRows);
#pragma unroll
                for (int mt = 0; mt < NMT; ++mt) {
                    acc[rt][mt] = mfma_32x32x16_f16(bl, xr[mt], acc[rt][mt]);
                    acc[rt][mt] = mfma_32x32x16_f16(bh, xl[mt], acc[rt][mt]);
                    acc[rt][mt] = mfma_32x32x16_f16(bh, xh[mt], acc[rt][mt]);
                }
            }
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int mt = 0; mt < NMT; ++mt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[rt][mt][i] *= fac[mt].y;
        if (!early) {
            meet<63>();   // (the terms have been read)
#pragma unroll
            for (int i = 0; i < NS - 1; ++i) stage(i, min(i, G - 1));
        }
    }

    // group g, in stage s, has landed once only the copies of the NS - 2 groups behind it may be under way; group g + NS - 1
    // goes where g - 1 was (past the last group, the last one again: every step copies alike)
    constexpr int kPer = NMT * XT + 2;
    auto step = [&](auto st, int g) {
        constexpr int s = decltype(st)::value;
        __builtin_amdgcn_sched_barrier(0);
        meet<(NS - 2) * kPer>();
        stage((s + NS - 1) % NS, min(g + NS - 1, G - 1));
        __builtin_amdgcn_sched_barrier(0);
        const uint16_t* const xs = Xl + s * kStage / 2;
        u32x4_t cur[2];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
            cur[rt] = *reinterpret_cast<const u32x4_t*>(xs + kXBytes / 2 + (2 * wave + rt) * 512 + 8 * lane);
        f16x2_t sv[2][WT], cv[2][WT];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const uint32_t sc = sbl[g * kTileRows + 64 * wave + 32 * rt + r];
#pragma unroll
            for (int k = 0; k < WT; ++k) {
                const uint32_t one = sc >> (16 * k) & 0xffffu;
                sv[rt][k] = __builtin_bit_cast(f16x2_t, one | one << 16);
                cv[rt][k] = sv[rt][k] * f16x2_t{static_cast<_Float16>(-24.0f), static_cast<_Float16>(-24.0f)};
            }
        }
        const int sw = (r >> 1) & 7;
        u32x4_t A[2][2][WT], B[2][NMT][XT];
        auto operands = [&](int ks) {
#pragma unroll
            for (int mt = 0; mt < NMT; ++mt)
#pragma unroll
                for (int x = 0; x < XT; ++x)
                    B[ks & 1][mt][x] = *reinterpret_cast<const u32x4_t*>(xs + (x * 32 * MMT + 32 * mt + r) * 64 + 8 * ((4 * h + ks) ^ sw));
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int k = 0; k < WT; ++k)
                    A[ks & 1][rt][k] = q4_to_f16<kExact, NATURAL>(cur[rt][ks], sv[rt][k], cv[rt][k], k16);
        };
        operands(0);
        // the next k step's reads, then its conversions between this one's products
        constexpr int kProducts = 2 * NMT * XT * WT, kBetween = (2 * WT * 16 + kProducts - 1) / kProducts;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            __builtin_amdgcn_sched_barrier(0);
            if (ks < 3) operands(ks + 1);
#pragma unroll
            for (int x = XT - 1; x >= 0; --x)
#pragma unroll
                for (int k = WT - 1; k >= 0; --k)
#pragma unroll
                    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                        for (int mt = 0; mt < NMT; ++mt)
                            acc[rt][mt] = mfma_32x32x16_f16(A[ks & 1][rt][k], B[ks & 1][mt][x], acc[rt][mt]);
            if (ks < 3) {
                __builtin_amdgcn_sched_group_barrier(0x100, NMT * XT, 0);
                unroll<kProducts>([&](auto) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, kBetween, 0);
                });
            }
        }
    };
    for (int g = 0; g < G; g += NS) unroll<NS>([&](auto i) {
        if (g + i.value < G) step(i, g + i.value);
    });
    meet<0>();   // (LDS is free: the last steps' copies have landed, their reads been made)
}

// The tile of this workgroup, its pairs and scales in LDS; body(tile, m0, m1, row0)
// where there is one.
template <int MATS, int SB_DT, int WT, int MMT, class Body>
__device__ __forceinline__ void tile_begin(const MoeArgs& p, const TileArgs& a, int* codes, tile_sb<WT>* sbl, uint16_t* terms, Body&& body) {
    constexpr int kOwn = kTileRows / MATS;   // rows of each matrix
    const int blocks = (p.rows + kOwn - 1) / kOwn, items = *a.count * blocks;
    // Workgroups go round the XCDs in turn: each XCD takes one run of the items, so that an expert's row blocks
    // and tiles meet in one L2 (the weights are read for each tile, x for each row block).
    const int run = (items + kXcds - 1) / kXcds, slot = blockIdx.x / kXcds;
    const int item = static_cast<int>(blockIdx.x % kXcds) * run + slot;
    if (slot >= run || item >= items) return;
    const int4 tile = a.tiles[item / blocks];
    if (tile.z == 0) return;
    const int row0 = kOwn * (item % blocks), G = p.cols / 64, t = threadIdx.x;
    const bool shared = tile.x >= p.experts;
    const MoeMat m0 = moe_matrix(p.m[0], p.sh[0], shared, tile.x, p.rows, p.cols);
    const MoeMat m1 = MATS == 2 ? moe_matrix(p.m[1], p.sh[1], shared, tile.x, p.rows, p.cols) : m0;
    if (t < 32 * MMT) {
        const int k = tile.y + min(t, tile.z - 1);
        codes[t] = shared ? pair_code(k, p.top) : a.list[k];
    }
    // thread t: row t's scales and the first 32 groups' terms
    const MoeMat& mm = MATS == 2 && (t & 32) ? m1 : m0;
    const bool vec = sb_vec(m0, G) && sb_vec(m1, G);
    const size_t base = static_cast<size_t>(tile_row<MATS>(p, row0)) * G;
    // (LDS has room for whole eights of groups: those past the last are not read)
    auto put = [&](int k, const u32x4_t& s8, const u32x4_t& b8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            sbl[(8 * k + i) * kTileRows + t] = tile_scale<SB_DT, WT>(static_cast<uint16_t>(s8[i / 2] >> (16 * (i & 1))));
        if (k < 4) put_terms<SB_DT>(terms, 8 * k, s8, b8);
    };
    const int eights = (G + 7) / 8;
    if (vec) {
        // 32 groups in one round of loads (one for each eight: 4096 columns of 8192 tokens 731 us instead of 719)
        for (int k0 = 0; k0 < eights; k0 += 4) {
            u32x4_t s8[4], b8[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k0 + k >= eights) break;
                s8[k] = *reinterpret_cast<const u32x4_t*>(mm.s + base + 8 * (k0 + k));
                b8[k] = *reinterpret_cast<const u32x4_t*>(mm.b + base + 8 * (k0 + k));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (k0 + k >= eights) break;
                put(k0 + k, s8[k], b8[k]);
            }
        }
    } else {
        for (int k = 0; k < eights; ++k) put(k, load_u16x8(mm.s + base, 8 * k, G, false), load_u16x8(mm.b + base, 8 * k, G, false));
    }
    if (eights < 4 && (eights & 1)) put_terms<SB_DT>(terms, 8 * eights, u32x4_t{}, u32x4_t{});   // (the half that meets sums of zero)
    __syncthreads();
    body(tile, m0, m1, row0);
}

template <int MATS, int SB_DT, int XT, int WT, bool NATURAL, int MMT, class Out>
__device__ __forceinline__ void tile_kernel(const MoeArgs& p, const TileArgs& a, const Out& out) {
    // (it first holds the constant parts' terms; behind the last group, all of them each wave's rows of outputs)
    constexpr int kStage = tile_stage_bytes(XT, MMT), kConst = 64 * kTileRows;
    constexpr int kBytes = (tile_stages(XT, MMT) - 1) * kStage + (kStage > kConst ? kStage : kConst);
    static_assert(kBytes >= 4 * 32 * kOutRow && kBytes >= 2 * kConst, "32 rows of outputs a wave; 32 groups' terms");
    __shared__ __attribute__((aligned(16))) uint16_t Xl[kBytes / 2];
    __shared__ int codes[32 * MMT];
    extern __shared__ __attribute__((aligned(16))) char sbl_bytes[];   // [G][256]
    tile_sb<WT>* const sbl = reinterpret_cast<tile_sb<WT>*>(sbl_bytes);
    tile_begin<MATS, SB_DT, WT, MMT>(p, a, codes, sbl, Xl + tile_terms_at(XT, MMT, p.cols / 64) / 2, [&](const int4& tile, const MoeMat& m0, const MoeMat& m1, int row0) {
        auto run = [&](auto n) {
            constexpr int NMT = decltype(n)::value;
            f32x16_t acc[2][NMT];
            float2 fac[NMT];
            tile_run<MATS, SB_DT, XT, WT, NATURAL, MMT, NMT>(p, a, m0, m1, row0, codes, Xl, sbl, acc, fac, out);
            const int lane = threadIdx.x & 63;
            char* const rows = reinterpret_cast<char*>(Xl) + (threadIdx.x >> 6) * 32 * kOutRow;
#pragma unroll
            for (int mt = 0; mt < NMT; ++mt) {
                out.put(acc[0][mt], acc[1][mt], fac[mt].x, row0, codes[32 * mt + (lane & 31)], rows + (lane & 31) * kOutRow);
                // a token's bytes, 16 a lane
                constexpr int kPieces = Out::kBytes / 16, kTokens = 64 / kPieces;
#pragma unroll
                for (int i = 0; i < 32 / kTokens; ++i) {
                    const int tok = kTokens * i + lane / kPieces, piece = lane % kPieces;
                    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(rows + tok * kOutRow + 16 * piece);
                    if (32 * mt + tok < tile.z) out.store(v, row0, codes[32 * mt + tok], piece);
                }
            }
        };
        const int nmt = (tile.z + 31) / 32;
        if constexpr (MMT >= 4) {
            if (nmt == 4) return run(std::integral_constant<int, 4>{});
            if (nmt == 3) return run(std::integral_constant<int, 3>{});
        }
        if constexpr (MMT >= 2) {
            if (nmt == 2) return run(std::integral_constant<int, 2>{});
        }
        run(std::integral_constant<int, 1>{});
    });
}

// What becomes of a wave's two row tiles: put() leaves a token's kBytes in its row
// of LDS (a lane holds rows 8 j + 4 h .. + 3 of its token, the column), store()
// takes 16 of them to memory. (Stored from the accumulators, 16 bytes of a row at a
// time, the pairs' rows alone took the down products of 8192 tokens 100 us.)
template <int DT>
__device__ __forceinline__ void put4(char* to, int at, f32x4_t v) {
    if constexpr (DT == 0) *reinterpret_cast<f32x4_t*>(to + 4 * at) = v;
    else if constexpr (DT == 1) *reinterpret_cast<u32x2_t*>(to + 2 * at) = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    else *reinterpret_cast<u32x2_t*>(to + 2 * at) = u32x2_t{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
}

template <int H_DT>
struct GateUpOut {
    static constexpr int kSize = H_DT == 0 ? 4 : 2, kBytes = 32 * kSize;
    const MoeArgs& p;
    void* h;
    __device__ __forceinline__ float weight(int) const { return 1.0f; }
    __device__ __forceinline__ void put(const f32x16_t& g, const f32x16_t& u, float f, int, int, char* to) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4_t v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = silu(g[4 * j + i] * f) * (u[4 * j + i] * f);
            put4<H_DT>(to, 8 * j + 4 * (threadIdx.x >> 5 & 1), v);
        }
    }
    __device__ __forceinline__ void store(u32x4_t v, int row0, int code, int piece) const {
        const int row = row0 + 32 * (threadIdx.x >> 6);
        if (row >= p.rows) return;   // (rows come in multiples of 64)
        const size_t at = (static_cast<size_t>(code >> 5) * p.slots + (code & 31)) * p.rows + row;
        *reinterpret_cast<u32x4_t*>(static_cast<char*>(h) + at * kSize + 16 * piece) = v;
    }
};
template <int SB_DT, int XT, int WT, int H_DT, int MMT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void moe_gate_up_tile_kernel(MoeArgs p, TileArgs a,
                                                                                                          void* __restrict__ h) {
    tile_kernel<2, SB_DT, XT, WT, false, MMT>(p, a, GateUpOut<H_DT>{p, h});
}

// The pairs' weighted rows: fp32, or (HALF, for bf16 y) fp16 after a power-of-two shift that
// puts the largest of each 64 into [2^14, 2^15), which stands in `exps` [pair][rows / 64]. fp16
// has 28 powers of two below that with all of its 11 bits, so a value keeps 11 bits of its
// own beside a much larger one; y has 8. It halves the rows' bytes (302 MB instead of 604 each way
// for 8192 tokens of nine pairs). Against 64 bits y is off as the plain form is (1.7e-3, its
// own rounding); from that form it differs by 5.8e-4, where the two round to different neighbours.
template <bool HALF>
struct DownOut {
    static constexpr int kBytes = HALF ? 128 : 256;
    const MoeArgs& p;
    const float* scores;
    const float* coef;
    void* part;
    float* exps;
    __device__ __forceinline__ float weight(int code) const {
        const int m = code >> 5, s = code & 31;
        return s < p.top ? scores[m * p.top + s] : coef ? coef[m] : 1.0f;
    }
    __device__ __forceinline__ void put(const f32x16_t& a0, const f32x16_t& a1, float f, int row0, int code, char* to) const {
        const int lane = threadIdx.x & 63, m = code >> 5, s = code & 31;
        float k = f;
        if constexpr (HALF) {
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fmaxf(fabsf(a0[i]), fabsf(a1[i])));
            mx = fmaxf(mx, __shfl_xor(mx, 32)) * fabsf(f);   // (the other half of the token's rows lies 32 lanes on)
            const int e = mx > 0.0f ? max(__builtin_amdgcn_frexp_expf(mx) - 15, -126) : 0, block = row0 / 64 + (threadIdx.x >> 6);
            k = f * ldexpf(1.0f, -e);
            if (lane < 32 && 64 * block < p.rows)
                exps[(static_cast<size_t>(m) * p.slots + s) * (p.rows / 64) + block] = ldexpf(1.0f, e);
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4_t v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = (rt ? a1[4 * j + i] : a0[4 * j + i]) * k;
                put4<HALF ? 2 : 0>(to, 32 * rt + 8 * j + 4 * (lane >> 5), v);
            }
    }
    __device__ __forceinline__ void store(u32x4_t v, int row0, int code, int piece) const {
        const int row = row0 + 64 * (threadIdx.x >> 6);
        if (row >= p.rows) return;
        const size_t at = (static_cast<size_t>(code >> 5) * p.slots + (code & 31)) * p.rows + row;
        *reinterpret_cast<u32x4_t*>(static_cast<char*>(part) + at * (HALF ? 2 : 4) + 16 * piece) = v;
    }
};
template <int SB_DT, int XT, int WT, bool NATURAL, bool HALF, int MMT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void moe_down_tile_kernel(
    MoeArgs p, TileArgs a, const float* __restrict__ scores, const float* __restrict__ coef, void* __restrict__ part,
    float* __restrict__ exps) {
    tile_kernel<1, SB_DT, XT, WT, NATURAL, MMT>(p, a, DownOut<HALF>{p, scores, coef, part, exps});
}

// ---- few pairs an expert ---------------------------------------------------------
//
// Where experts have a handful of pairs each, the weights' bytes bound a call, and
// the tiles above keep too few of them on their way. So the same operands in
// workgroups of 128 weight rows (of gate and up 64 of each), four waves of two row
// tiles, on 16x16x32 products; their 16 columns are 16 pairs, or 8 pairs by their
// two terms. A stage is four groups, 128 bytes of each row of words and so whole
// cache lines; three stages, 72 KB. Lane (c, kg) holds row c of a row tile and 32
// consecutive columns kg of each 128, with their group's scale: k slots may stand
// for any columns as long as both operands agree. The groups' constant parts are
// products whose k slots are 32 groups, formed from the scales and biases that the
// lane loads and leaves in LDS.
// At 32 tokens (256 experts of 512 x 2048 and a shared one, 8 a token, all fp32)
// gate and up take 50 us, 200 MB read at 4.0 TB/s with the start and the last
// round (two and a half) of workgroups, and down 36; by the large tiles 62 and 40,
// with stages of one group and two waves of 64 rows 66 and 43. Words requested ahead
// of what waits for the pairs, and workgroups that begin in different columns, gave
// nothing (52, 51).
constexpr int kSlimRows = 128, kSlimColumns = 16, kSlimStages = 3;
constexpr int kSlimWords = kSlimRows * 128, kSlimStage = kSlimWords + kSlimColumns * 512;

template <int MATS, int SB_DT, int XT, int WT, bool NATURAL, class Store>
__device__ __forceinline__ void slim_kernel(const MoeArgs& p, const TileArgs& a, const Store& store) {
    constexpr bool kExact = SB_DT == 1 || WT == 2;
    constexpr int NS = kSlimStages, kOwn = kSlimRows / MATS, kPairs = kSlimColumns / XT;
    __shared__ __attribute__((aligned(16))) char buf[NS * kSlimStage];
    extern __shared__ __attribute__((aligned(16))) char sbl_bytes[];   // [groups in whole eights][128]
    tile_sb<WT>* const sbl = reinterpret_cast<tile_sb<WT>*>(sbl_bytes);
    const int blocks = (p.rows + kOwn - 1) / kOwn, item = blockIdx.x / blocks;
    if (item >= *a.count) return;
    const int4 tile = a.tiles[item];
    if (tile.z == 0) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, kg = lane >> 4, G = p.cols / 64, steps = (G + 3) / 4;
    const bool shared = tile.x >= p.experts;
    const MoeMat m0 = moe_matrix(p.m[0], p.sh[0], shared, tile.x, p.rows, p.cols);
    const MoeMat m1 = MATS == 2 ? moe_matrix(p.m[1], p.sh[1], shared, tile.x, p.rows, p.cols) : m0;
    // the wave's rows: 16 of each of two matrices, or 32 (past the end: the last ones, whose results are left)
    const int row0 = kOwn * (blockIdx.x % blocks), own = row0 + kOwn / 4 * wave, first = min(own, p.rows - kOwn / 4);
    auto pair = [&](int col) {
        const int k = min(col & (kPairs - 1), tile.z - 1);
        return shared ? pair_code(tile.y + k, p.top) : a.list[tile.y + k];
    };
    auto x_row = [&](int code) { return static_cast<uint32_t>(MATS == 2 ? code >> 5 : (code >> 5) * p.slots + (code & 31)); };

    // Copies of words: 8 rows each, a row's 16-byte pieces p at p ^ (row / 2 % 8); of x: two columns each, a column's
    // 8-element blocks b at b ^ column: 16 lanes' reads meet every bank once. Past the last column, its last block again (the
    // scales there are zeros).
    const uint32_t lds = lds_addr(reinterpret_cast<const uint16_t*>(buf)), rbytes = p.cols / 2;
    const uint32_t wrow = (first + (lane >> 3)) * rbytes, wpiece = 16 * ((lane & 7) ^ (lane >> 4));   // (odd eights of rows: ^ 64)
    uint32_t xrow[2], xblock[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int col = 4 * wave + 2 * i + (lane >> 5);
        xrow[i] = (x_row(pair(col)) * XT + col / kPairs) * p.cols * 2;
        xblock[i] = 16 * ((lane & 31) ^ col);
    }
    auto stage = [&](int to, int g) {
        const uint32_t at = lds + to * kSlimStage;
        const uint32_t w[2] = {wrow + min(wpiece + 128 * g, rbytes - 16), wrow + min((wpiece ^ 64) + 128 * g, rbytes - 16)};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            dma16(reinterpret_cast<const char*>(MATS == 2 && i >= 2 ? m1.w : m0.w) + static_cast<size_t>(8 * (MATS == 2 ? i & 1 : i)) * rbytes,
                  w[i & 1], at + (4 * wave + i) * 1024);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            dma16(reinterpret_cast<const char*>(a.x16), xrow[i] + min(xblock[i] + 512u * g, 4 * rbytes - 16),
                  at + kSlimWords + (2 * wave + i) * 1024);
    };
    uint32_t k16 = 0x4C004C00u;
    asm("" : "+v"(k16));

    f32x4_t acc[2] = {};
    const int code = pair(c);
    float2 fac = a.fac[x_row(code)];
    fac.x *= store.weight(code);
    {
        const int gp = (G + kSumsPad - 1) / kSumsPad * kSumsPad;
        const uint16_t* const S = a.sums + static_cast<size_t>(x_row(code)) * 2 * gp;
        const bool vec = sb_vec(m0, G) && sb_vec(m1, G);
        for (int k0 = 0; k0 < G; k0 += 32) {
            const int k = k0 + 8 * kg;
            u32x4_t xh{}, xl{}, s8[2], b8[2];
            if (k < gp) {   // (16 pairs: both terms of their sums; 8: each column its own)
                xh = *reinterpret_cast<const u32x4_t*>(S + k + c / kPairs * gp);
                if constexpr (XT == 1) xl = *reinterpret_cast<const u32x4_t*>(S + gp + k);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const MoeMat& mm = MATS == 2 && j ? m1 : m0;
                const size_t at = static_cast<size_t>(first + (MATS == 2 ? 0 : 16 * j) + c) * G;
                s8[j] = load_u16x8(mm.s + at, k, G, vec);
                b8[j] = load_u16x8(mm.b + at, k, G, vec);
            }
            if (k0 == 0) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < NS - 1; ++i)
                    if (i < steps) stage(i, i);
                __builtin_amdgcn_sched_barrier(0);
            }
            const u32x4_t xr = rest_sums(xh);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (k < G) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        sbl[(k + i) * kSlimRows + 32 * wave + 16 * j + c] =
                            k + i < G ? tile_scale<SB_DT, WT>(static_cast<uint16_t>(s8[j][i / 2] >> (16 * (i & 1)))) : 0;
                }
                u32x4_t bh, bl;
                const_terms<SB_DT>(s8[j], b8[j], bh, bl);
                acc[j] = mfma_16x16x32_f16(bl, xr, acc[j]);
                if constexpr (XT == 1) acc[j] = mfma_16x16x32_f16(bh, xl, acc[j]);
                acc[j] = mfma_16x16x32_f16(bh, xh, acc[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[j] *= fac.y;
    }

    constexpr int kPer = 6;
    auto step = [&](auto st, int g) {
        constexpr int s = decltype(st)::value;
        __builtin_amdgcn_sched_barrier(0);
        if (g + NS - 2 < steps) meet<(NS - 2) * kPer>();   // (the copies of the step behind may be under way)
        else meet<0>();
        if (g + NS - 1 < steps) stage((s + NS - 1) % NS, g + NS - 1);
        __builtin_amdgcn_sched_barrier(0);
        const char* const ws = buf + s * kSlimStage + (32 * wave + c) * 128;
        const char* const xs = buf + s * kSlimStage + kSlimWords + c * 512;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            if (4 * g + 2 * d >= G) continue;
            u32x4_t words[2], B[4];
            f16x2_t sv[2][WT], cv[2][WT];
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) B[ks] = *reinterpret_cast<const u32x4_t*>(xs + 16 * ((16 * d + 4 * kg + ks) ^ c));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                words[j] = *reinterpret_cast<const u32x4_t*>(ws + 16 * j * 128 + 16 * ((4 * d + kg) ^ (c >> 1)));
                const uint32_t sc = sbl[(4 * g + 2 * d + (kg >> 1)) * kSlimRows + 32 * wave + 16 * j + c];
#pragma unroll
                for (int q = 0; q < WT; ++q) {
                    const uint32_t one = sc >> (16 * q) & 0xffffu;
                    sv[j][q] = __builtin_bit_cast(f16x2_t, one | one << 16);
                    cv[j][q] = sv[j][q] * f16x2_t{static_cast<_Float16>(-24.0f), static_cast<_Float16>(-24.0f)};
                }
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int q = WT - 1; q >= 0; --q)
                        acc[j] = mfma_16x16x32_f16(q4_to_f16<kExact, NATURAL>(words[j][ks], sv[j][q], cv[j][q], k16), B[ks], acc[j]);
        }
    };
    for (int g = 0; g < steps; g += NS) unroll<NS>([&](auto i) {
        if (g + i.value < steps) step(i, g + i.value);
    });
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (XT == 2) acc[j][i] += __shfl_xor(acc[j][i], 8);
            acc[j][i] *= fac.x;
        }
    if (c < kPairs && c < tile.z && own < p.rows) store(acc, own + 4 * kg, code);
}

// A lane's rows 4 kg .. + 3 of its wave's two row tiles, for its pair.
template <int H_DT>
struct SlimUp {
    const MoeArgs& p;
    void* h;
    __device__ __forceinline__ float weight(int) const { return 1.0f; }
    __device__ __forceinline__ void operator()(const f32x4_t (&acc)[2], int row, int code) const {
        f32x4_t v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = silu(acc[0][i]) * acc[1][i];
        put4<H_DT>(static_cast<char*>(h) + (static_cast<size_t>(code >> 5) * p.slots + (code & 31)) * p.rows * (H_DT == 0 ? 4 : 2), row, v);
    }
};
template <int SB_DT, int XT, int WT, int H_DT>
__global__ __launch_bounds__(256) void moe_gate_up_slim_kernel(MoeArgs p, TileArgs a, void* __restrict__ h) {
    slim_kernel<2, SB_DT, XT, WT, false>(p, a, SlimUp<H_DT>{p, h});
}

// The pairs' weighted rows, for moe_combine_kernel.
struct SlimDown {
    const MoeArgs& p;
    const float* scores;
    const float* coef;
    float* part;
    __device__ __forceinline__ float weight(int code) const {
        const int m = code >> 5, s = code & 31;
        return s < p.top ? scores[m * p.top + s] : coef ? coef[m] : 1.0f;
    }
    __device__ __forceinline__ void operator()(const f32x4_t (&acc)[2], int row, int code) const {
        float* const to = part + (static_cast<size_t>(code >> 5) * p.slots + (code & 31)) * p.rows + row;
#pragma unroll
        for (int j = 0; j < 2; ++j) *reinterpret_cast<f32x4_t*>(to + 16 * j) = acc[j];
    }
};
template <int SB_DT, int XT, int WT, bool NATURAL>
__global__ __launch_bounds__(256) void moe_down_slim_kernel(MoeArgs p, TileArgs a, const float* __restrict__ scores,
                                                            const float* __restrict__ coef, float* __restrict__ part) {
    slim_kernel<1, SB_DT, XT, WT, NATURAL>(p, a, SlimDown{p, scores, coef, part});
}

// y[m] = residual[m] + the rows of its pairs, in their order: a thread 8 columns.
template <int Y_DT>
__global__ __launch_bounds__(256) void moe_combine_half_kernel(const uint16_t* __restrict__ part, const float* __restrict__ exps,
                                                               const int32_t* __restrict__ indices, int experts, int top,
                                                               int slots, const void* residual, void* y, int rows) {
    const int m = blockIdx.y, r = 8 * (blockIdx.x * 256 + threadIdx.x);
    if (r >= rows) return;
    const size_t o = static_cast<size_t>(m) * rows + r;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = residual ? elem<Y_DT>::load(residual, o + i) : 0.0f;
    for (int j = 0; j < slots; ++j) {
        const int e = j < top ? indices[m * top + j] : 0;
        if (e < 0 || (j < top && e >= experts)) continue;
        const size_t pair = static_cast<size_t>(m) * slots + j;
        const u32x4_t u = *reinterpret_cast<const u32x4_t*>(part + pair * rows + r);
        const float k = exps[pair * (rows / 64) + r / 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = fmaf(f16_to_f32(static_cast<uint16_t>(u[i])), k, v[2 * i]);
            v[2 * i + 1] = fmaf(f16_to_f32(static_cast<uint16_t>(u[i] >> 16)), k, v[2 * i + 1]);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) elem<Y_DT>::store(y, o + i, v[i]);
}

MoeMat moe_mat(const qff_q4_matrices& q) {
    return MoeMat{q.w, static_cast<const uint16_t*>(q.scales), static_cast<const uint16_t*>(q.biases)};
}

// Pairs (with the shared expert's) up to which each takes its weights by itself, and
// pairs an expert (for gate and up: by the terms of x) up to which the small tiles take them; up to
// 32 tokens they always do, so the large ones have bf16 outputs of fewer terms alone.
// Measured with 256 experts of 512 x 2048 and a shared one, 8 a token, us a call with what
// stands ahead of and behind the products, other weights each time (two runs differ by up to
// 0.5, the single pairs of down by 3):
//   gate and up, pairs   36    54    63    72    81    90   an expert   6    7    8    9 (fp32 x)   14   15   16 (bf16 x)
//     by themselves    16.5  21.3  23.7  25.8  29.5  32.0
//     small tiles      18.6  22.9  23.1  23.1  30.0  29.9              86   95  101  108             91   96  101
//     large tiles                                                     109  110  111  112            100  100  101
//   down, pairs         126   144   162   180   198   216   an expert  1.5   2   2.5   3    4 (fp32 h)   1.5   2    3    4 (fp16 h, bf16 y)
//     by themselves    29.1  31.4  34.2  40.6  41.3  43.4
//     small tiles      31.7  34.4  36.5  39.5  39.5  39.1             52.5 55.8 59.8 61.9 64.2          51.4 55.6 60.3 62.6
//     large tiles                                                     53.8 54.5 60.1 60.5 61.3          54.0 55.3 61.0 61.7
constexpr int kOneUp = 60, kOneDown = 200, kSlimUp = 16, kSlimDown = 2;

template <int DT>
using Dt = std::integral_constant<int, DT>;

template <class F>
void with_dtype(qff_dtype d, F&& f) {
    if (d == QFF_F32) f(Dt<0>{});
    else if (d == QFF_BF16) f(Dt<1>{});
    else f(Dt<2>{});
}
// (x of the gate and up products, and y: F32 or BF16; scales and biases: BF16 or F16)
template <class F>
void with_io(qff_dtype d, F&& f) {
    if (d == QFF_F32) f(Dt<0>{});
    else f(Dt<1>{});
}
template <class F>
void with_sb(qff_dtype d, F&& f) {
    if (d == QFF_BF16) f(Dt<1>{});
    else f(Dt<2>{});
}

size_t dtype_size(qff_dtype d) { return d == QFF_F32 ? 4 : 2; }

struct Terms {
    int x, w;   // fp16 terms of x and of a weight
};
// (bf16 outputs of up to 32 tokens have all terms too)
Terms tile_terms(qff_dtype x, qff_dtype sb, qff_dtype out, int tokens) {
    const bool all = out != QFF_BF16 || tokens <= 32;
    return {x == QFF_F32 && all ? 2 : 1, sb == QFF_F16 && all ? 2 : 1};
}
// Tokens of a tile, in units of 32: as many as an expert has on average, within
// what fits the registers and LDS.
int tile_units(int pairs, int experts, int xt) {
    const int avg = pairs / experts;
    return xt == 1 && avg > 48 ? 4 : avg > 24 ? 2 : 1;
}

// What the tiles read: `rows` rows of p.x as fp16 terms, factors and sums (fp16 x
// stays where it is), and the plan of up to `most` pairs a tile.
TileArgs moe_prepare(qff_ctx* ctx, hipStream_t stream, const MoeArgs& p, bool shared, qff_dtype dtype, int xt, int rows, int most,
                     int unit) {
    const int n = p.tokens * p.top, blocks = n > kPlanAlone ? (n + kPlanShare - 1) / kPlanShare : 1;
    float2* fac = reinterpret_cast<float2*>(ctx->moe_xs);
    uint16_t* sums = reinterpret_cast<uint16_t*>(fac + (rows + 1) / 2 * 2);   // (16-byte aligned)
    const PlanArgs q{p.indices, p.experts, p.top, p.tokens, shared, most, unit, blocks > 1 ? ctx->moe_parts : nullptr,
                     ctx->moe_off, static_cast<int4*>(ctx->moe_tiles), ctx->moe_list};
    auto x16 = [&](auto X, auto XT, auto COPY) {
        if (blocks == 1) {
            ProfScope prof(ctx, stream, "moe_prepare");
            constexpr int kRows = kPlanThreads / 64;
            moe_prepare_kernel<X.value, XT.value, COPY.value><<<1 + (rows + kRows - 1) / kRows, kPlanThreads, 0, stream>>>(
                q, p.x, ctx->q4_x16, fac, sums, p.cols, rows);
        } else {
            ProfScope prof(ctx, stream, "moe_x16");
            moe_x16_kernel<X.value, XT.value, COPY.value><<<(rows + kX16Waves - 1) / kX16Waves, 64 * kX16Waves, 0, stream>>>(
                p.x, ctx->q4_x16, fac, sums, p.cols, rows);
        }
    };
    if (dtype == QFF_F16) x16(Dt<2>{}, Dt<1>{}, Dt<0>{});
    else if (dtype == QFF_BF16) x16(Dt<1>{}, Dt<1>{}, Dt<1>{});
    else if (xt == 1) x16(Dt<0>{}, Dt<1>{}, Dt<1>{});
    else x16(Dt<0>{}, Dt<2>{}, Dt<1>{});
    if (blocks > 1) {
        {
            ProfScope prof(ctx, stream, "moe_count");
            moe_count_kernel<<<blocks, kPlanThreads, 0, stream>>>(p.indices, p.experts, n, ctx->moe_parts);
        }
        ProfScope prof(ctx, stream, "moe_plan");
        moe_plan_kernel<<<blocks, kPlanThreads, 0, stream>>>(q);
    }
    return {ctx->moe_off, static_cast<const int4*>(ctx->moe_tiles), ctx->moe_list,
            dtype == QFF_F16 ? static_cast<const uint16_t*>(p.x) : ctx->q4_x16, fac, sums};
}

// Tokens of a slice whose `rows` rows of x each fit the workspace.
int slice_tokens(const qff_ctx* ctx, int rows, int cols, int xt, bool copy, int tokens) {
    size_t most = std::min<size_t>(tokens, 65535);
    if (copy) most = std::min(most, static_cast<size_t>(ctx->q4_xs_tokens) * 8192 / (static_cast<size_t>(rows) * xt * cols * 2));
    const size_t row = 8 + (cols / 64 + kSumsPad - 1) / kSumsPad * kSumsPad * 4;
    most = std::min(most, (size_t{1} << 31) / (static_cast<size_t>(rows) * cols * 2));   // (offsets of rows have 32 bits)
    return static_cast<int>(std::min(most, (moe_part_bytes(ctx->cfg) / 16 - 8) / (rows * row)));
}

unsigned slim_grid(const MoeArgs& p, bool shared, int xt, int own_rows) {
    const int most = kSlimColumns / xt, pairs = p.tokens * p.top;
    const unsigned tiles = pairs / most + std::min(p.experts, pairs) + (shared ? (p.tokens + most - 1) / most : 0);
    return tiles * ((p.rows + own_rows - 1) / own_rows);
}
unsigned tile_grid(const MoeArgs& p, bool shared, int units, int own_rows) {
    const int most = 32 * units, pairs = p.tokens * p.top;
    const int tiles = pairs / most + std::min(p.experts, pairs) + (shared ? (p.tokens + most - 1) / most : 0);
    const unsigned items = static_cast<unsigned>(tiles) * ((p.rows + own_rows - 1) / own_rows);
    return (items + kXcds - 1) / kXcds * kXcds;
}

template <int... V>
struct Ints {};
template <class F, int V0, int... V>
void pick(int v, Ints<V0, V...>, F&& f) {
    if constexpr (sizeof...(V) == 0) f(Dt<V0>{});
    else if (v == V0) f(Dt<V0>{});
    else pick(v, Ints<V...>{}, f);
}

}  // namespace

hipError_t launch_moe_gate_up(qff_ctx* ctx, hipStream_t stream, const qff_moe_weights* w, const void* x, qff_dtype x_dtype,
                              const int32_t* indices, int top, void* h, qff_dtype h_dtype, int tokens) {
    const bool shared = w->shared_gate.w != nullptr;
    MoeArgs p{};
    p.m[0] = moe_mat(w->gate);
    p.m[1] = moe_mat(w->up);
    p.sh[0] = moe_mat(w->shared_gate);
    p.sh[1] = moe_mat(w->shared_up);
    p.x = x;
    p.indices = indices;
    p.experts = w->experts;
    p.top = top;
    p.slots = top + shared;
    p.rows = w->inter;
    p.cols = w->hidden;
    p.tokens = tokens;
    const int G = p.cols / 64;
    if (tokens * p.slots <= kOneUp) {
        ProfScope prof(ctx, stream, "moe_gate_up_one");
        const dim3 grid(p.rows / 16, tokens * p.slots);
        with_io(x_dtype, [&](auto X) {
            with_sb(w->sb_dtype, [&](auto S) {
                with_dtype(h_dtype, [&](auto H) {
                    moe_gate_up_one_kernel<X.value, S.value, H.value><<<grid, 64 * kOneWaves, 0, stream>>>(p, h);
                });
            });
        });
        return hipGetLastError();
    }
    const Terms tm = tile_terms(x_dtype, w->sb_dtype, h_dtype, tokens);
    const int most = slice_tokens(ctx, 1, p.cols, tm.x, true, tokens);
    const size_t lds = static_cast<size_t>((G + 7) / 8 * 8) * kTileRows * 2 * tm.w;
    for (int t0 = 0; t0 < tokens; t0 += most) {
        p.tokens = std::min(most, tokens - t0);
        p.indices = indices + static_cast<size_t>(t0) * top;
        p.x = static_cast<const char*>(x) + static_cast<size_t>(t0) * p.cols * dtype_size(x_dtype);
        const bool slim = tokens <= 32 || p.tokens * top * tm.x <= kSlimUp * p.experts;
        const int units = tile_units(p.tokens * top, p.experts, tm.x), unit = slim ? kSlimColumns / tm.x : 32;
        const TileArgs a = moe_prepare(ctx, stream, p, shared, x_dtype, tm.x, p.tokens, slim ? unit : 32 * units, unit);
        void* to = static_cast<char*>(h) + static_cast<size_t>(t0) * p.slots * p.rows * dtype_size(h_dtype);
        if (slim) {
            ProfScope prof(ctx, stream, "moe_gate_up_slim");
            const unsigned grid = slim_grid(p, shared, tm.x, kSlimRows / 2);
            const size_t bytes = static_cast<size_t>((G + 7) / 8 * 8) * kSlimRows * 2 * tm.w;
            with_sb(w->sb_dtype, [&](auto S) {
                pick(tm.x, Ints<1, 2>{}, [&](auto XT) {
                    auto go = [&](auto WT) {
                        with_dtype(h_dtype, [&](auto H) {
                            moe_gate_up_slim_kernel<S.value, XT.value, WT.value, H.value><<<grid, 256, bytes, stream>>>(p, a, to);
                        });
                    };
                    if constexpr (S.value == 2) pick(tm.w, Ints<1, 2>{}, go);
                    else go(Dt<1>{});
                });
            });
            continue;
        }
        ProfScope prof(ctx, stream, "moe_gate_up_tile");
        const unsigned grid = tile_grid(p, shared, units, kTileRows / 2);
        auto launch = [&](auto S, auto XT, auto WT, auto H) {
            auto go = [&](auto U) {
                moe_gate_up_tile_kernel<S.value, XT.value, WT.value, H.value, U.value><<<grid, 256, lds, stream>>>(p, a, to);
            };
            if constexpr (XT.value == 1) pick(units, Ints<1, 2, 4>{}, go);
            else pick(units, Ints<1, 2>{}, go);
        };
        with_sb(w->sb_dtype, [&](auto S) {
            if (h_dtype == QFF_BF16) return launch(S, Dt<1>{}, Dt<1>{}, Dt<1>{});
            constexpr int WT = decltype(S)::value == 2 ? 2 : 1;
            pick(tm.x, Ints<1, 2>{}, [&](auto XT) {
                if (h_dtype == QFF_F32) launch(S, XT, Dt<WT>{}, Dt<0>{});
                else launch(S, XT, Dt<WT>{}, Dt<2>{});
            });
        });
    }
    return hipGetLastError();
}

hipError_t launch_moe_down(qff_ctx* ctx, hipStream_t stream, const qff_moe_weights* w, const void* h, qff_dtype h_dtype,
                           const int32_t* indices, const float* scores, int top, const float* coef, const void* residual,
                           void* y, qff_dtype y_dtype, int tokens) {
    const bool shared = w->shared_down.w != nullptr;
    MoeArgs p{};
    p.m[0] = moe_mat(w->down);
    p.sh[0] = moe_mat(w->shared_down);
    p.experts = w->experts;
    p.top = top;
    p.slots = top + shared;
    p.rows = w->hidden;
    p.cols = w->inter;
    const int G = p.cols / 64;
    if (tokens * p.slots <= kOneDown) {
        p.x = h;
        p.indices = indices;
        p.tokens = tokens;
        ProfScope prof(ctx, stream, "moe_down_one");
        const dim3 grid(p.rows / 16, tokens);
        with_dtype(h_dtype, [&](auto X) {
            with_sb(w->sb_dtype, [&](auto S) {
                with_io(y_dtype, [&](auto Y) {
                    moe_down_one_kernel<X.value, S.value, Y.value>
                        <<<grid, 64 * kOneWaves, 0, stream>>>(p, scores, coef, residual, y);
                });
            });
        });
        return hipGetLastError();
    }
    const Terms tm = tile_terms(h_dtype, w->sb_dtype, y_dtype, tokens);
    const bool slim = tokens <= 32 || tokens * top <= kSlimDown * p.experts, half = !slim && y_dtype == QFF_BF16;
    // as many tokens at a time as the workspace has room for
    const size_t per = static_cast<size_t>(p.slots) * p.rows * (half ? 2 : 4);
    int most = static_cast<int>(std::min<size_t>({ctx->moe_part_bytes / per, static_cast<size_t>(tokens), 65535}));
    most = std::min(most, slice_tokens(ctx, p.slots, p.cols, tm.x, h_dtype != QFF_F16, tokens));
    for (int t0 = 0; t0 < tokens; t0 += most) {
        const int n = std::min(most, tokens - t0);
        p.tokens = n;
        p.indices = indices + static_cast<size_t>(t0) * top;
        p.x = static_cast<const char*>(h) + static_cast<size_t>(t0) * p.slots * p.cols * dtype_size(h_dtype);
        const float* sc = scores + static_cast<size_t>(t0) * top;
        const float* cf = coef ? coef + t0 : nullptr;
        const size_t yo = static_cast<size_t>(t0) * p.rows * dtype_size(y_dtype);
        const void* res = residual ? static_cast<const char*>(residual) + yo : nullptr;
        void* to = static_cast<char*>(y) + yo;
        const int units = tile_units(n * top, p.experts, tm.x), unit = slim ? kSlimColumns / tm.x : 32;
        const TileArgs a = moe_prepare(ctx, stream, p, shared, h_dtype, tm.x, n * p.slots, slim ? unit : 32 * units, unit);
        if (slim) {
            ProfScope prof(ctx, stream, "moe_down_slim");
            const unsigned grid = slim_grid(p, shared, tm.x, kSlimRows);
            const size_t bytes = static_cast<size_t>((G + 7) / 8 * 8) * kSlimRows * 2 * tm.w;
            auto launch = [&](auto S, auto XT, auto NAT) {
                auto go = [&](auto WT) {
                    moe_down_slim_kernel<S.value, XT.value, WT.value, NAT.value>
                        <<<grid, 256, bytes, stream>>>(p, a, sc, cf, static_cast<float*>(ctx->moe_part));
                };
                if constexpr (S.value == 2) pick(tm.w, Ints<1, 2>{}, go);
                else go(Dt<1>{});
            };
            with_sb(w->sb_dtype, [&](auto S) {
                if (h_dtype == QFF_F16) launch(S, Dt<1>{}, Dt<1>{});
                else pick(tm.x, Ints<1, 2>{}, [&](auto XT) { launch(S, XT, Dt<0>{}); });
            });
        } else {
            ProfScope prof(ctx, stream, "moe_down_tile");
            const unsigned grid = tile_grid(p, shared, units, kTileRows);
            const size_t lds = static_cast<size_t>((G + 7) / 8 * 8) * kTileRows * 2 * tm.w;
            auto launch = [&](auto S, auto XT, auto WT, auto NAT, auto HALF) {
                auto go = [&](auto U) {
                    moe_down_tile_kernel<S.value, XT.value, WT.value, NAT.value, HALF.value, U.value>
                        <<<grid, 256, lds, stream>>>(p, a, sc, cf, ctx->moe_part, ctx->moe_exps);
                };
                if constexpr (XT.value == 1) pick(units, Ints<1, 2, 4>{}, go);
                else pick(units, Ints<1, 2>{}, go);
            };
            with_sb(w->sb_dtype, [&](auto S) {
                constexpr int WT = decltype(S)::value == 2 ? 2 : 1;
                if (half) {
                    if (h_dtype == QFF_F16) launch(S, Dt<1>{}, Dt<1>{}, Dt<1>{}, Dt<1>{});
                    else launch(S, Dt<1>{}, Dt<1>{}, Dt<0>{}, Dt<1>{});
                } else if (h_dtype == QFF_F16) {
                    launch(S, Dt<1>{}, Dt<WT>{}, Dt<1>{}, Dt<0>{});
                } else {
                    pick(tm.x, Ints<1, 2>{}, [&](auto XT) { launch(S, XT, Dt<WT>{}, Dt<0>{}, Dt<0>{}); });
                }
            });
        }
        ProfScope prof(ctx, stream, "moe_combine");
        with_io(y_dtype, [&](auto Y) {
            if (half)
                moe_combine_half_kernel<Y.value><<<dim3((p.rows + 2047) / 2048, n), 256, 0, stream>>>(
                    static_cast<const uint16_t*>(ctx->moe_part), ctx->moe_exps, p.indices, p.experts, top, p.slots, res, to, p.rows);
            else
                moe_combine_kernel<Y.value><<<dim3((p.rows + 1023) / 1024, n), 256, 0, stream>>>(
                    static_cast<const float*>(ctx->moe_part), p.indices, p.experts, top, p.slots, res, to, p.rows);
        });
    }
    return hipGetLastError();
}

}  // namespace qff
