// moe.hip -- the expert block on affine-Q4 weights: every token through the
// matrices of its own experts (qff_moe_gate_up, qff_moe_down).
//
//   h[m, j] = silu(Wg x_m) * (Wu x_m),  W of expert indices[m, j]
//   y[m]    = residual + sum_j score[m, j] Wd h[m, j]
//
// A weight is W = s q + b, q the nibble. The kernels below take the nibble as
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

// 16 consecutive columns of x in a lane, and the bf16 operands of the two k
// steps they make (columns 0-7 and 8-15), TERMS of them.
template <int X_DT>
struct XCols;
template <>
struct XCols<0> {
    static constexpr int kTerms = 3;
    f32x4_t v[4];
    __device__ __forceinline__ void load(const void* x, size_t i) {
        const f32x4_t* p = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(x) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = p[k];
    }
    __device__ __forceinline__ void terms(int step, u32x4_t (&t)[3]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = v[2 * step][j], b = v[2 * step + 1][j];
            const uint32_t h = pack_bf16x2(a, b);
            a -= __uint_as_float(h << 16);
            b -= __uint_as_float(h & 0xffff0000u);
            const uint32_t m = pack_bf16x2(a, b);
            a -= __uint_as_float(m << 16);
            b -= __uint_as_float(m & 0xffff0000u);
            t[0][j] = h;
            t[1][j] = m;
            t[2][j] = pack_bf16x2(a, b);
        }
    }
};
template <>
struct XCols<1> {
    static constexpr int kTerms = 1;
    u32x4_t v[2];
    __device__ __forceinline__ void load(const void* x, size_t i) {
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(x) + i);
        v[0] = p[0];
        v[1] = p[1];
    }
    // pairs (c0, c1), (c2, c3), (c4, c5), (c6, c7) -> (c0, c4), (c1, c5), (c2, c6), (c3, c7)
    __device__ __forceinline__ u32x4_t paired(int step) const {
        const u32x4_t u = v[step];
        return u32x4_t{__builtin_amdgcn_perm(u[2], u[0], 0x05040100u), __builtin_amdgcn_perm(u[2], u[0], 0x07060302u),
                       __builtin_amdgcn_perm(u[3], u[1], 0x05040100u), __builtin_amdgcn_perm(u[3], u[1], 0x07060302u)};
    }
    __device__ __forceinline__ void terms(int step, u32x4_t (&t)[1]) const { t[0] = paired(step); }
};
template <>
struct XCols<2> : XCols<1> {
    static constexpr int kTerms = 2;
    __device__ __forceinline__ void terms(int step, u32x4_t (&t)[2]) const {
        const u32x4_t u = paired(step);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = f16_to_f32(static_cast<uint16_t>(u[j])), b = f16_to_f32(static_cast<uint16_t>(u[j] >> 16));
            const uint32_t h = pack_bf16x2(a, b);
            a -= __uint_as_float(h << 16);
            b -= __uint_as_float(h & 0xffff0000u);
            t[0][j] = h;
            t[1][j] = pack_bf16x2(a, b);
        }
    }
};

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
// own weight row's sum (lane & 15) and needs that row's scale alone.

template <int X_DT, int SB_DT, int MATS>
struct OneStep {
    u32x4_t w[MATS][kGroups / 2];
    XCols<X_DT> x[kGroups];
    uint16_t s[MATS][kGroups], b[MATS][kGroups];

    // groups g0 .. g0 + 3 (those past the last are requested as the last and not used)
    __device__ __forceinline__ void load(const MoeMat (&m)[MATS], const void* xp, size_t xrow, int row, int cols, int g0,
                                         int kg) {
        const int G = cols / 64;
        const size_t r = static_cast<size_t>(row);
#pragma unroll
        for (int i = 0; i < MATS; ++i) {
#pragma unroll
            for (int sp = 0; sp < kGroups / 2; ++sp)
                w[i][sp] = *reinterpret_cast<const u32x4_t*>(m[i].w + r * (cols / 8) +
                                                             8 * min(g0 + 2 * sp + (kg >> 1), G - 1) + 4 * (kg & 1));
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const size_t at = r * G + min(g0 + k, G - 1);
                s[i][k] = m[i].s[at];
                b[i][k] = m[i].b[at];
            }
        }
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
            x[k].load(xp, xrow + 64 * min(g0 + k, G - 1) + 32 * (kg & 1) + 16 * (kg >> 1));
    }
    __device__ __forceinline__ void add(float (&acc)[MATS], int groups) const {
        constexpr int T = XCols<X_DT>::kTerms;
        const uint32_t one = q4_one();
        const u32x4_t ones{one, one, one, one};
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
                x[k].terms(st, t);
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
                const float sc = 16.0f * elem<SB_DT>::load(&s[i][k], 0), bi = elem<SB_DT>::load(&b[i][k], 0);
                acc[i] = fmaf(sc, P[i][0], fmaf(bi - sc, X[0], acc[i]));
            }
        }
    }
};

constexpr int kOneWaves = 8;

// Gate and up: one workgroup per (16 rows, pair), its waves over K.
template <int X_DT, int SB_DT, int H_DT>
__global__ __launch_bounds__(64 * kOneWaves) void moe_gate_up_one_kernel(MoeArgs p, void* __restrict__ h) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, kg = lane >> 4;
    const int tok = blockIdx.y / p.slots, j = blockIdx.y % p.slots;
    const bool shared = j >= p.top;
    const int e = shared ? 0 : p.indices[tok * p.top + j];
    if (e < 0 || (!shared && e >= p.experts)) return;
    const MoeMat m[2] = {moe_matrix(p.m[0], p.sh[0], shared, e, p.rows, p.cols),
                         moe_matrix(p.m[1], p.sh[1], shared, e, p.rows, p.cols)};
    const int row0 = 16 * blockIdx.x, G = p.cols / 64;
    float acc[2] = {0.0f, 0.0f};
    for (int g0 = kGroups * wave; g0 < G; g0 += kGroups * kOneWaves) {
        OneStep<X_DT, SB_DT, 2> st;
        st.load(m, p.x, static_cast<size_t>(tok) * p.cols, row0 + c, p.cols, g0, kg);
        st.add(acc, G - g0);
    }
    __shared__ float red[kOneWaves][2][16];
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
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, kg = lane >> 4;
    const int tok = blockIdx.y, row0 = 16 * blockIdx.x, G = p.cols / 64, steps = (G + kGroups - 1) / kGroups;
    float acc = 0.0f;
    for (int it = wave; it < p.slots * steps; it += kOneWaves) {
        const int j = it / steps, g0 = kGroups * (it - j * steps);
        const bool shared = j >= p.top;
        const int e = shared ? 0 : p.indices[tok * p.top + j];
        if (e < 0 || (!shared && e >= p.experts)) continue;
        const MoeMat m[1] = {moe_matrix(p.m[0], p.sh[0], shared, e, p.rows, p.cols)};
        const float f = shared ? (coef ? coef[tok] : 1.0f) : scores[tok * p.top + j];
        OneStep<X_DT, SB_DT, 1> st;
        st.load(m, p.x, (static_cast<size_t>(tok) * p.slots + j) * p.cols, row0 + c, p.cols, g0, kg);
        float a[1] = {0.0f};
        st.add(a, G - g0);
        acc = fmaf(f, a[0], acc);
    }
    __shared__ float red[kOneWaves][16];
    if (lane < 16) red[wave][lane] = acc;
    __syncthreads();
    if (threadIdx.x < 16) {
        const size_t o = static_cast<size_t>(tok) * p.rows + row0 + threadIdx.x;
        float a = residual ? elem<Y_DT>::load(residual, o) : 0.0f;
#pragma unroll
        for (int w = 0; w < kOneWaves; ++w) a += red[w][threadIdx.x];
        elem<Y_DT>::store(y, o, a);
    }
}

// ---- several tokens of one expert ------------------------------------------------

// Which pairs each expert has, for calls of many: one workgroup counts them,
// sums the counts up and writes the pairs expert by expert (in no fixed order
// within one: a pair's sums do not depend on its place).
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void moe_plan_kernel(const int32_t* __restrict__ indices, int experts, int top,
                                                                int tokens, int* __restrict__ off, int* __restrict__ list) {
    __shared__ int cnt[kMoeMaxExperts], at[kMoeMaxExperts], wsum[kPlanThreads / 64];
    const int t = threadIdx.x, n = tokens * top;
    if (t < kMoeMaxExperts) cnt[t] = 0;
    __syncthreads();
    for (int i = t; i < n; i += kPlanThreads) {
        const int e = indices[i];
        if (e >= 0 && e < experts) atomicAdd(&cnt[e], 1);
    }
    __syncthreads();
    const int own = t < experts ? cnt[t] : 0;
    const int incl = wave_inclusive_scan_int(own);
    if ((t & 63) == 63) wsum[t >> 6] = incl;
    __syncthreads();
    int before = incl - own;
    for (int w = 0; w < t >> 6; ++w) before += wsum[w];
    if (t < experts) {
        off[t] = before;
        at[t] = before;
        if (t == experts - 1) off[experts] = before + own;
    }
    __syncthreads();
    for (int i = t; i < n; i += kPlanThreads) {
        const int e = indices[i];
        if (e >= 0 && e < experts) list[atomicAdd(&at[e], 1)] = pair_code(i / top, i % top);
    }
}

constexpr int kRowsWaves = 8;
constexpr int kRowsScan = 1024;   // pairs of a call that each workgroup looks through by itself

// 16 RT rows of one expert's matrices against its tokens, 16 at a time: WK waves
// over K times RT row tiles. Outputs leave through `store(acc.., row, code)`.
template <int X_DT, int SB_DT, int MATS, int WK>
struct RowsKernel {
    static constexpr int kRt = kRowsWaves / WK, kRows = 16 * kRt;
    static constexpr int kRed = WK * kRt * MATS * 16 * 17;

    template <class Store>
    static __device__ __forceinline__ void run(const MoeArgs& p, const int* __restrict__ off, const int* __restrict__ plan,
                                               float* lds, Store&& store) {
        constexpr int T = XCols<X_DT>::kTerms;
        const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, kg = lane >> 4;
        const int wk = wave % WK, rt = wave / WK;
        const int e = blockIdx.y;
        const bool shared = e >= p.experts;
        const int G = p.cols / 64, row0 = kRows * blockIdx.x;

        __shared__ int list[kRowsScan], found;
        int n;
        const int* from = list;
        if (shared) {
            n = p.tokens;
        } else if (plan) {
            const int o = off[e];
            n = off[e + 1] - o;
            from = plan + o;
        } else {
            if (t == 0) found = 0;
            __syncthreads();
            for (int i = t; i < p.tokens * p.top; i += 64 * kRowsWaves)
                if (p.indices[i] == e) list[atomicAdd(&found, 1)] = pair_code(i / p.top, i % p.top);
            __syncthreads();
            n = found;
        }
        if (n == 0) return;

        float* const scl = lds;                              // [MATS][G][kRows] 16 s
        float* const bil = lds + MATS * G * kRows;           // [MATS][G][kRows] b - 16 s
        float* const red = lds + 2 * MATS * G * kRows;       // [WK][kRt][MATS][16 tokens][17]
        MoeMat m[MATS];
#pragma unroll
        for (int i = 0; i < MATS; ++i) {
            m[i] = moe_matrix(p.m[i], p.sh[i], shared, e, p.rows, p.cols);
            const size_t base = static_cast<size_t>(row0) * G;
            for (int k = t; k < kRows * G; k += 64 * kRowsWaves) {
                const int r = k / G, g = k - r * G;
                const size_t at = min(base + k, static_cast<size_t>(p.rows) * G - 1);
                const float s = 16.0f * elem<SB_DT>::load(m[i].s, at), b = elem<SB_DT>::load(m[i].b, at);
                scl[(i * G + g) * kRows + r] = s;
                bil[(i * G + g) * kRows + r] = b - s;
            }
        }
        const int wrow = min(row0 + 16 * rt + c, p.rows - 1);
        __syncthreads();

        for (int t0 = 0; t0 < n; t0 += 16) {
            const int place = min(t0 + c, n - 1);
            const int code = shared ? pair_code(place, p.top) : from[place];
            const size_t xrow = MATS == 2 ? static_cast<size_t>(code >> 5) * p.cols
                                          : (static_cast<size_t>(code >> 5) * p.slots + (code & 31)) * p.cols;
            f32x4_t acc[MATS];
#pragma unroll
            for (int i = 0; i < MATS; ++i) acc[i] = f32x4_t{};
            for (int g0 = kGroups * wk; g0 < G; g0 += kGroups * WK) {
                u32x4_t w[MATS][kGroups / 2];
#pragma unroll
                for (int i = 0; i < MATS; ++i)
#pragma unroll
                    for (int sp = 0; sp < kGroups / 2; ++sp)
                        w[i][sp] = *reinterpret_cast<const u32x4_t*>(
                            m[i].w + static_cast<size_t>(wrow) * (p.cols / 8) + 8 * min(g0 + 2 * sp + (kg >> 1), G - 1) +
                            4 * (kg & 1));
                XCols<X_DT> x[kGroups];
#pragma unroll
                for (int k = 0; k < kGroups; ++k)
                    x[k].load(p.x, xrow + 64 * min(g0 + k, G - 1) + 32 * (kg & 1) + 16 * (kg >> 1));
                const uint32_t one = q4_one();
                const u32x4_t ones{one, one, one, one};
                uint32_t words[MATS][kGroups / 2][4];
#pragma unroll
                for (int i = 0; i < MATS; ++i)
#pragma unroll
                    for (int sp = 0; sp < kGroups / 2; ++sp) span_words(w[i][sp], words[i][sp]);
#pragma unroll
                for (int k = 0; k < kGroups; ++k) {
                    if (g0 + k >= G) break;
                    f32x4_t P[MATS], X{};
#pragma unroll
                    for (int i = 0; i < MATS; ++i) P[i] = f32x4_t{};
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        u32x4_t tm[T];
                        x[k].terms(st, tm);
#pragma unroll
                        for (int j = T - 1; j >= 0; --j) X = mfma_16x16x32_bf16(ones, tm[j], X);
#pragma unroll
                        for (int i = 0; i < MATS; ++i) {
                            const u32x4_t q = q4_to_bf16(words[i][k / 2][2 * (k % 2) + st], one);
#pragma unroll
                            for (int j = T - 1; j >= 0; --j) P[i] = mfma_16x16x32_bf16(q, tm[j], P[i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MATS; ++i) {
                        const int at = (i * G + g0 + k) * kRows + 16 * rt + 4 * kg;
                        const f32x4_t s = *reinterpret_cast<const f32x4_t*>(scl + at);
                        const f32x4_t b = *reinterpret_cast<const f32x4_t*>(bil + at);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(s[r], P[i][r], fmaf(b[r], X[r], acc[i][r]));
                    }
                }
            }
            if (t0) __syncthreads();   // the tile before has been read
#pragma unroll
            for (int i = 0; i < MATS; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) red[(((wk * kRt + rt) * MATS + i) * 16 + c) * 17 + 4 * kg + r] = acc[i][r];
            __syncthreads();
            for (int k = t; k < 256 * kRt; k += 64 * kRowsWaves) {
                const int r = k % 16, tok = k / 16 % 16, tile = k / 256, row = row0 + 16 * tile + r;
                if (t0 + tok >= n || row >= p.rows) continue;
                float v[MATS];
#pragma unroll
                for (int i = 0; i < MATS; ++i) {
                    v[i] = 0.0f;
#pragma unroll
                    for (int q = 0; q < WK; ++q) v[i] += red[(((q * kRt + tile) * MATS + i) * 16 + tok) * 17 + r];
                }
                store(v, row, shared ? pair_code(t0 + tok, p.top) : from[t0 + tok]);
            }
        }
    }
};

template <int X_DT, int SB_DT, int H_DT, int WK>
__global__ __launch_bounds__(64 * kRowsWaves) void moe_gate_up_rows_kernel(MoeArgs p, const int* __restrict__ off,
                                                                           const int* __restrict__ plan, void* __restrict__ h) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    RowsKernel<X_DT, SB_DT, 2, WK>::run(p, off, plan, lds, [&](const float (&v)[2], int row, int code) {
        const size_t o = (static_cast<size_t>(code >> 5) * p.slots + (code & 31)) * p.rows + row;
        elem<H_DT>::store(h, o, silu(v[0]) * v[1]);
    });
}

// The weighted row of each pair, for moe_combine_kernel.
template <int X_DT, int SB_DT, int WK>
__global__ __launch_bounds__(64 * kRowsWaves) void moe_down_rows_kernel(MoeArgs p, const int* __restrict__ off,
                                                                        const int* __restrict__ plan,
                                                                        const float* __restrict__ scores,
                                                                        const float* __restrict__ coef,
                                                                        float* __restrict__ part) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    RowsKernel<X_DT, SB_DT, 1, WK>::run(p, off, plan, lds, [&](const float (&v)[1], int row, int code) {
        const int m = code >> 5, j = code & 31;
        const float f = j < p.top ? scores[m * p.top + j] : coef ? coef[m] : 1.0f;
        part[(static_cast<size_t>(m) * p.slots + j) * p.rows + row] = f * v[0];
    });
}

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

MoeMat moe_mat(const qff_q4_matrices& q) {
    return MoeMat{q.w, static_cast<const uint16_t*>(q.scales), static_cast<const uint16_t*>(q.biases)};
}

// Pairs up to which each is a workgroup row of its own (their weights are read
// for each pair).
constexpr int kOnePairs = 36;

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
    if (tokens * p.slots <= kOnePairs) {
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
    const int *off = nullptr, *plan = nullptr;
    if (tokens * top > kRowsScan) {
        ProfScope prof(ctx, stream, "moe_plan");
        moe_plan_kernel<<<1, kPlanThreads, 0, stream>>>(indices, p.experts, top, tokens, ctx->moe_off, ctx->moe_list);
        off = ctx->moe_off;
        plan = ctx->moe_list;
    }
    ProfScope prof(ctx, stream, "moe_gate_up_rows");
    const int G = p.cols / 64;
    auto launch = [&](auto X, auto S, auto H, auto K) {
        using R = RowsKernel<X.value, S.value, 2, K.value>;
        const dim3 grid((p.rows + R::kRows - 1) / R::kRows, p.experts + shared);
        const size_t lds = (4 * static_cast<size_t>(G) * R::kRows + R::kRed) * sizeof(float);
        moe_gate_up_rows_kernel<X.value, S.value, H.value, K.value>
            <<<grid, 64 * kRowsWaves, lds, stream>>>(p, off, plan, h);
    };
    with_io(x_dtype, [&](auto X) {
        with_sb(w->sb_dtype, [&](auto S) {
            with_dtype(h_dtype, [&](auto H) {
                if (G <= 8) launch(X, S, H, Dt<2>{});
                else launch(X, S, H, Dt<8>{});
            });
        });
    });
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
    if (tokens * p.slots <= kOnePairs) {
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
    // as many tokens at a time as the workspace has rows of pairs for
    const size_t per = static_cast<size_t>(p.slots) * p.rows * sizeof(float);
    const int most = static_cast<int>(std::min<size_t>({ctx->moe_part_bytes / per, static_cast<size_t>(tokens), 65535}));
    for (int t0 = 0; t0 < tokens; t0 += most) {
        const int n = std::min(most, tokens - t0);
        p.tokens = n;
        p.indices = indices + static_cast<size_t>(t0) * top;
        p.x = static_cast<const char*>(h) + static_cast<size_t>(t0) * p.slots * p.cols * dtype_size(h_dtype);
        const float* sc = scores + static_cast<size_t>(t0) * top;
        const float* cf = coef ? coef + t0 : nullptr;
        const size_t yo = static_cast<size_t>(t0) * p.rows * dtype_size(y_dtype);
        const int *off = nullptr, *plan = nullptr;
        if (n * top > kRowsScan) {
            ProfScope prof(ctx, stream, "moe_plan");
            moe_plan_kernel<<<1, kPlanThreads, 0, stream>>>(p.indices, p.experts, top, n, ctx->moe_off, ctx->moe_list);
            off = ctx->moe_off;
            plan = ctx->moe_list;
        }
        float* part = static_cast<float*>(ctx->moe_part);
        {
            ProfScope prof(ctx, stream, "moe_down_rows");
            auto launch = [&](auto X, auto S, auto K) {
                using R = RowsKernel<X.value, S.value, 1, K.value>;
                const dim3 grid((p.rows + R::kRows - 1) / R::kRows, p.experts + shared);
                const size_t lds = (2 * static_cast<size_t>(G) * R::kRows + R::kRed) * sizeof(float);
                moe_down_rows_kernel<X.value, S.value, K.value>
                    <<<grid, 64 * kRowsWaves, lds, stream>>>(p, off, plan, sc, cf, part);
            };
            with_dtype(h_dtype, [&](auto X) {
                with_sb(w->sb_dtype, [&](auto S) {
                    if (G <= 8) launch(X, S, Dt<2>{});
                    else launch(X, S, Dt<8>{});
                });
            });
        }
        ProfScope prof(ctx, stream, "moe_combine");
        const dim3 grid((p.rows + 1023) / 1024, n);
        with_io(y_dtype, [&](auto Y) {
            moe_combine_kernel<Y.value><<<grid, 256, 0, stream>>>(
                part, p.indices, p.experts, top, p.slots, residual ? static_cast<const char*>(residual) + yo : nullptr,
                static_cast<char*>(y) + yo, p.rows);
        });
    }
    return hipGetLastError();
}

}  // namespace qff
