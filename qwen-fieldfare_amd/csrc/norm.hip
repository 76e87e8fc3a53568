// norm.hip -- RMSNorm of whole tokens, the step between a layer's attention
// and its expert block:
//   y[m, c] = x[m, c] rsqrt(mean_c x[m, c]^2 + eps) w[c]
// and, in the same pass, the shared expert's coefficient
//   coef[m] = sigmoid(sum_c G[c] y[m, c]),  G one affine-Q8 row.
// Replaces qwen_rmsnorm_f32 (deltanet.metal:18-53) for callers that need the
// normalised rows themselves (the router and the experts read the same ones).
//
// One workgroup a token: thread t holds 8-column blocks t, t + 256, .. in
// registers, so x is read once; sum x^2 and sum G w x meet in one LDS round
// (the coefficient's sum takes the inverse RMS afterwards, the unrounded y).
#include "common.hpp"
#include "internal.hpp"
#include "mfma.hpp"

namespace qff {

constexpr int kNormThreads = 256;

template <int DT>
__device__ __forceinline__ void load8(const void* p, size_t i, float (&v)[8]) {
    if constexpr (DT == 1) {
        const u32x4_t u = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(u[j] << 16);
            v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        }
    } else {
        const f32x4_t* q = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i);
        const f32x4_t a = q[0], b = q[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = a[j];
            v[4 + j] = b[j];
        }
    }
}

// (x may be y: neither is declared to overlap nothing)
template <int X_DT, int Y_DT, int W_DT, int NB>
__global__ __launch_bounds__(kNormThreads) void rms_norm_kernel(const void* x, const void* __restrict__ w, float eps,
                                                                const uint32_t* __restrict__ gw,
                                                                const uint16_t* __restrict__ gs,
                                                                const uint16_t* __restrict__ gb, int g_bf16,
                                                                void* y, float* __restrict__ coef, int cols) {
    const int t = threadIdx.x, nb = cols / 8;
    const size_t row = static_cast<size_t>(blockIdx.x) * cols;
    float v[NB][8], wn[NB][8];
    float ss = 0.0f, dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int b = min(t + kNormThreads * i, nb - 1);
        load8<X_DT>(x, row + 8 * b, v[i]);
        load8<W_DT>(w, 8 * b, wn[i]);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int b = t + kNormThreads * i;
        if (b >= nb) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ss = fmaf(v[i][e], v[i][e], ss);
            v[i][e] *= wn[i][e];
        }
        if (gw) {
            const u32x2_t q = *reinterpret_cast<const u32x2_t*>(gw + 2 * b);
            const float s = g_bf16 ? bf16_to_f32(gs[b / 8]) : f16_to_f32(gs[b / 8]);
            const float c = g_bf16 ? bf16_to_f32(gb[b / 8]) : f16_to_f32(gb[b / 8]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                dot = fmaf(fmaf(static_cast<float>(q[e / 4] >> (8 * (e % 4)) & 0xffu), s, c), v[i][e], dot);
        }
    }
    __shared__ float2 part[kNormThreads / 64];
    ss = group_sum<64>(ss);
    dot = group_sum<64>(dot);
    if ((t & 63) == 0) part[t >> 6] = make_float2(ss, dot);
    __syncthreads();
    ss = (part[0].x + part[1].x) + (part[2].x + part[3].x);
    const float rs = 1.0f / sqrtf(ss / static_cast<float>(cols) + eps);
    if (gw && t == 0) coef[blockIdx.x] = sigmoid(rs * ((part[0].y + part[1].y) + (part[2].y + part[3].y)));
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int b = t + kNormThreads * i;
        if (b >= nb) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= rs;
        if constexpr (Y_DT == 1) {
            *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(y) + row + 8 * b) =
                u32x4_t{pack_bf16x2(v[i][0], v[i][1]), pack_bf16x2(v[i][2], v[i][3]), pack_bf16x2(v[i][4], v[i][5]),
                        pack_bf16x2(v[i][6], v[i][7])};
        } else {
            f32x4_t* o = reinterpret_cast<f32x4_t*>(static_cast<float*>(y) + row + 8 * b);
            o[0] = f32x4_t{v[i][0], v[i][1], v[i][2], v[i][3]};
            o[1] = f32x4_t{v[i][4], v[i][5], v[i][6], v[i][7]};
        }
    }
}

template <int X_DT, int Y_DT, int W_DT>
static void rms_norm_launch(hipStream_t stream, const void* x, const void* w, float eps, const uint32_t* gw,
                            const uint16_t* gs, const uint16_t* gb, int g_bf16, void* y, float* coef, int cols, int tokens) {
    constexpr int kMost = static_cast<int>(((1ll << 32) - 1) / kNormThreads);   // a grid has fewer than 2^32 work-items
    for (int t0 = 0; t0 < tokens; t0 += kMost) {
        const int n = tokens - t0 < kMost ? tokens - t0 : kMost;
        const size_t at = static_cast<size_t>(t0) * cols;
        const void* const from = static_cast<const char*>(x) + at * (X_DT == 0 ? 4 : 2);
        void* const to = static_cast<char*>(y) + at * (Y_DT == 0 ? 4 : 2);
        float* const c = gw ? coef + t0 : nullptr;
#define QFF_NORM(NB) rms_norm_kernel<X_DT, Y_DT, W_DT, NB><<<n, kNormThreads, 0, stream>>>(from, w, eps, gw, gs, gb, g_bf16, to, c, cols)
        if (cols <= 8 * kNormThreads) QFF_NORM(1);
        else if (cols <= 16 * kNormThreads) QFF_NORM(2);
        else QFF_NORM(4);
#undef QFF_NORM
        if (tokens - t0 <= kMost) break;   // (t0 stays within an int)
    }
}

hipError_t launch_rms_norm(qff_ctx* ctx, hipStream_t stream, const void* x, qff_dtype x_dtype, const void* norm_w,
                           qff_dtype norm_dtype, float eps, const qff_q4_matrices* gate, qff_dtype gate_sb, void* y,
                           qff_dtype y_dtype, float* coef, int cols, int tokens) {
    ProfScope prof(ctx, stream, "rms_norm");
    const uint32_t* gw = gate ? gate->w : nullptr;
    const uint16_t* gs = gate ? static_cast<const uint16_t*>(gate->scales) : nullptr;
    const uint16_t* gb = gate ? static_cast<const uint16_t*>(gate->biases) : nullptr;
    const int gbf = gate_sb == QFF_BF16;
    const int kind = (x_dtype == QFF_BF16) * 4 + (y_dtype == QFF_BF16) * 2 + (norm_dtype == QFF_BF16);
    switch (kind) {
#define QFF_KIND(K) \
    case K: rms_norm_launch<(K) / 4, (K) / 2 % 2, (K) % 2>(stream, x, norm_w, eps, gw, gs, gb, gbf, y, coef, cols, tokens); break
        QFF_KIND(0); QFF_KIND(1); QFF_KIND(2); QFF_KIND(3);
        QFF_KIND(4); QFF_KIND(5); QFF_KIND(6); QFF_KIND(7);
#undef QFF_KIND
    }
    return hipGetLastError();
}

}  // namespace qff
