// sample.hip -- the next token of each sequence from its logits (qff_sample).
// Counterpart of QwenLogitSelector (QwenGenerationSupport.swift:228-362),
// which runs on the host.
//
// A token weighs e_i = exp((l_i - l_max) / t), held as the whole number of
// 2^-44 nearest to it (a row of 2^18 tokens sums to at most 2^62): sums of
// whole numbers do not depend on their order, so neither do the borders of
// top-p nor the token that u falls on, however a row is cut up. Every filter
// keeps a head of the order (l descending, index ascending), so what is kept is
// all tokens down to one (l*, index*). Tokens that weigh 0 are never kept or
// drawn and are left out of everything.
//
// Four launches, a row's tokens cut into chunks, a workgroup each:
//   max     each chunk's largest and least finite logit
//   bins    each chunk's weights, and the row's weights and counts, in 256 bins of
//           equal width in l
//   gather  every chunk finds the row's bins [lo, hi] that hold the
//           borders of top-k and top-p, and lists its tokens in them in order;
//           the tokens of the bins before lo are kept
//   pick    one workgroup a row: the borders among the listed tokens, kept in LDS,
//           by an 8-bit radix selection over the bits of l in which they differ (by
//           count, then by weight), the chunk that u falls into, its 64 tokens and
//           the token there
// A row is read four times at most (three from the caches: 0.6 MB at 151936
// logits); rows that need no border or no draw skip what they do not need.
//
// At 151936 fp32 logits (a read of all takes 0.1 us a row): one row 34 us, of
// them max 4, bins 8, gather 6, pick 17; 32 rows with settings of their own
// 7 + 16 + 17 + 23. What bounds it: the chain of dependent steps, for one row;
// for 32 also the exponentials, one in 64 bits a token (an exact border needs a
// weight that does not depend on who computes it), twice where min_p asks: the bins'
// 16.4 us are 10.6 without them, 15.8 without the additions in LDS (which lie behind
// them), 9.4 without either; for one row 7.7, 6.6, 5.8 and 4.6. The row's bins are added up by atomics in the second launch (of
// whole numbers, so in any order): by every chunk in the third, one row's gather
// took 28 us and its bins 5.
#include <algorithm>

#include "common.hpp"
#include "internal.hpp"

namespace qff {

namespace {

typedef unsigned long long u64;

constexpr int kBins = kSampleBins, kCopies = 8;   // LDS copies of a chunk's bins: lanes of equal logits meet in fewer of them
constexpr int kSampleThreads = 256, kPickThreads = 1024;
static_assert(kBins == kSampleThreads, "a bin a thread");
// Listed tokens that the last launch keeps in LDS; groups of 64 tokens of a chunk.
constexpr int kPickCache = 15872, kGroups = kSampleVocab / 8 / 64;
constexpr double kUnit = 17592186044416.0;   // 2^44

struct SampleArgs {
    const void* logits;
    const float* u;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* tokens;
    float* probs;
    int vocab, chunks, per;   // per: tokens of a chunk
    SampleWork w;
};

// What a row asks for.
struct Row {
    float t, top_p, min_p;
    int top_k;
    bool first;   // the first of the order, without a draw
};
__device__ __forceinline__ Row row_of(const SampleArgs& a, int b) {
    Row r;
    r.t = a.temperature ? a.temperature[b] : 1.0f;
    r.top_k = a.top_k ? a.top_k[b] : 0;
    r.top_p = a.top_p ? a.top_p[b] : 1.0f;
    r.min_p = a.min_p ? a.min_p[b] : 0.0f;
    r.first = !(r.t > 0.0f) || r.top_p <= 0.0f || r.min_p > 1.0f;
    return r;
}

template <int DT>
__device__ __forceinline__ float logit(const SampleArgs& a, int b, int i) {
    const float l = elem<DT>::load(a.logits, static_cast<size_t>(b) * a.vocab + i);
    return l != l ? -INFINITY : l;
}

// Tokens at, at + step, .. of a row, all requested at once; those from `end` on: -inf.
constexpr int kBatch = 16;
template <int DT>
__device__ __forceinline__ void load_logits(const SampleArgs& a, int b, int at, int step, int end, float (&l)[kBatch]) {
#pragma unroll
    for (int q = 0; q < kBatch; ++q) l[q] = logit<DT>(a, b, min(at + q * step, end - 1));
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
        if (at + q * step >= end) l[q] = -INFINITY;
}

// Monotone in l: larger logits have larger keys.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t u = __float_as_uint(l == 0.0f ? 0.0f : l);   // (-0 and 0 are equal)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// e^d for d in (-32, 0]: d = k ln 2 + r, |r| <= ln 2 / 2, with ln 2 in two parts (Cody and
// Waite's reduction), e^r by its Taylor series to r^13 / 13! (what follows is 4e-18 of
// it). The library's, which serves other ranges too, made 32 rows' bins 18 us instead of 16.
__device__ __forceinline__ double exp_head(double d) {
    const double k = rint(d * 1.4426950408889634);
    const double r = fma(k, -2.3190468138462996e-17, fma(k, -0.6931471805599453, d));
    double p = 1.0 / 6227020800.0;
    constexpr double kTerms[] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0,
                                 1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
    for (double c : kTerms) p = fma(p, r, c);
    return ldexp(p, static_cast<int>(k));
}

// e^((l - best) / t) and its weight.
struct Weigher {
    double best, inv, min_p;
    float bestf;
    __device__ __forceinline__ Weigher(const Row& r, float best_) : best(best_), inv(1.0 / r.t), min_p(r.min_p), bestf(best_) {}
    __device__ __forceinline__ double e(float l) const {
        if (l == bestf) return 1.0;
        const double d = (static_cast<double>(l) - best) * inv;
        return d > -31.3 ? exp_head(d) : 0.0;   // (e^-31.3 rounds to no unit)
    }
    // (e <= 1: added to 2^52, whose last bit is 1, it is rounded to the nearest unit and stands in the low bits)
    static __device__ __forceinline__ u64 units(double e) {
        return static_cast<u64>(__double_as_longlong(fma(e, kUnit, 4503599627370496.0))) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 mass(float l) const { return units(e(l)); }
    __device__ __forceinline__ bool passes(double e) const { return !(min_p > 0.0) || e >= min_p; }
};

// Bins of equal width in l over what the row spans, or over the 32 t below its
// largest, beyond which nothing weighs anything.
struct Binner {
    float best, scale;
    __device__ __forceinline__ Binner(const Row& r, float best_, float least) : best(best_) {
        const float span = fminf(32.0f * r.t, best_ - least);
        scale = static_cast<float>(kBins) / span;
    }
    __device__ __forceinline__ int operator()(float l) const {
        if (l == best) return 0;
        return static_cast<int>(fminf((best - l) * scale, static_cast<float>(kBins - 1)));
    }
};

__device__ __forceinline__ float2 row_range(const SampleArgs& a, int b) {
    // (every lane of a wave reads one chunk's; 64 chunks at most)
    const int lane = threadIdx.x & 63;
    const float2 m = a.w.range[b * kSampleChunks + min(lane, a.chunks - 1)];
    return make_float2(group_max<64>(m.x), -group_max<64>(-m.y));
}

// The lane's value (the same lane for the whole wave).
__device__ __forceinline__ u64 lane_u64(u64 v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane);
    return static_cast<u64>(hi) << 32 | lo;
}
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ u64 dpp_u64(u64 v) {
    const uint32_t lo = dpp_int<CTRL, ROW_MASK>(static_cast<int>(v)), hi = dpp_int<CTRL, ROW_MASK>(static_cast<int>(v >> 32));
    return static_cast<u64>(hi) << 32 | lo;
}
// Sum over the lanes before and up to this one (as wave_inclusive_scan_int), and over all.
__device__ __forceinline__ u64 wave_scan_u64(u64 v) {
    v += dpp_u64<0x111>(v);
    v += dpp_u64<0x112>(v);
    v += dpp_u64<0x114>(v);
    v += dpp_u64<0x118>(v);
    v += dpp_u64<0x142, 0xa>(v);
    v += dpp_u64<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) { return lane_u64(wave_scan_u64(v), 63); }

// Where chunk c's bins stand; kSampleChunks: the row's.
__device__ __forceinline__ size_t bins_at(int b, int c) { return (static_cast<size_t>(b) * (kSampleChunks + 1) + c) * kBins; }

template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_max_kernel(SampleArgs a) {
    const int b = blockIdx.y, i0 = blockIdx.x * a.per, i1 = min(i0 + a.per, a.vocab);
    float hi = -INFINITY, lo = INFINITY;
    if (blockIdx.x == 0) {   // (for the next launch's sums)
        a.w.bin_mass[bins_at(b, kSampleChunks) + threadIdx.x] = 0;
        a.w.bin_count[b * kBins + threadIdx.x] = 0;
    }
    for (int j = i0; j < i1; j += kBatch * kSampleThreads) {
        float l[kBatch];
        load_logits<DT>(a, b, j + threadIdx.x, kSampleThreads, i1, l);
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            hi = fmaxf(hi, l[q]);
            if (l[q] > -INFINITY) lo = fminf(lo, l[q]);
        }
    }
    __shared__ float2 part[kSampleThreads / 64];
    hi = group_max<64>(hi);
    lo = -group_max<64>(-lo);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = make_float2(hi, lo);
    __syncthreads();
    if (threadIdx.x == 0) {
        float2 m = part[0];
        for (int w = 1; w < kSampleThreads / 64; ++w) m = make_float2(fmaxf(m.x, part[w].x), fminf(m.y, part[w].y));
        a.w.range[b * kSampleChunks + blockIdx.x] = m;
    }
}

template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_bins_kernel(SampleArgs a) {
    const int b = blockIdx.y, t = threadIdx.x, i0 = blockIdx.x * a.per, i1 = min(i0 + a.per, a.vocab);
    float l[kBatch];   // (the first tokens are on their way beside what the row asks for)
    load_logits<DT>(a, b, i0 + t, kSampleThreads, i1, l);
    const Row r = row_of(a, b);
    const float2 range = row_range(a, b);
    if (r.first || range.x == -INFINITY) return;
    __shared__ u64 mass[kBins][kCopies];
    __shared__ uint32_t count[kBins][kCopies];
    for (int i = t; i < kBins * kCopies; i += kSampleThreads) {
        (&mass[0][0])[i] = 0;
        (&count[0][0])[i] = 0;
    }
    __syncthreads();
    const Weigher weigh(r, range.x);
    const Binner bin(r, range.x, range.y);
    for (int j = i0; j < i1; j += kBatch * kSampleThreads) {
        if (j > i0) load_logits<DT>(a, b, j + t, kSampleThreads, i1, l);
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const u64 m = weigh.mass(l[q]);
            if (m == 0) continue;
            const int k = bin(l[q]);
            atomicAdd(&mass[k][t % kCopies], m);
            atomicAdd(&count[k][t % kCopies], 1u);
        }
    }
    __syncthreads();
    u64 m = 0;
    uint32_t n = 0;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
        m += mass[t][(c + t) % kCopies];
        n += count[t][(c + t) % kCopies];
    }
    a.w.bin_mass[bins_at(b, blockIdx.x) + t] = m;
    if (n) {   // (whole numbers: any order)
        atomicAdd(&a.w.bin_mass[bins_at(b, kSampleChunks) + t], m);
        atomicAdd(&a.w.bin_count[b * kBins + t], n);
    }
}

// The bins that hold the borders, the same in every chunk's workgroup: bins
// before lo are kept whole, those past hi not at all. lo > hi: there is no border.
// A bin a thread.
struct CutWork {
    u64 mass[kSampleThreads / 64];
    uint32_t count[kSampleThreads / 64];
    u64 least;
    int by_count, last;
    u64 mass_before;
    int count_before;
};
__device__ __forceinline__ SampleCut find_cut(const SampleArgs& a, const Row& r, int b, CutWork& w) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const u64 mass = a.w.bin_mass[bins_at(b, kSampleChunks) + t];
    const uint32_t count = a.w.bin_count[b * kBins + t];
    u64 mass_to = wave_scan_u64(mass);
    int count_to = wave_inclusive_scan_int(static_cast<int>(count));
    if (lane == 63) {
        w.mass[wave] = mass_to;
        w.count[wave] = count_to;
    }
    if (t == 0) w.last = 0;
    __syncthreads();
    u64 total = 0;
    int tokens = 0;
#pragma unroll
    for (int i = 0; i < kSampleThreads / 64; ++i) {
        if (i < wave) {
            mass_to += w.mass[i];
            count_to += w.count[i];
        }
        total += w.mass[i];
        tokens += w.count[i];
    }
    const u64 mass_ahead = mass_to - mass;
    const int count_ahead = count_to - static_cast<int>(count);
    SampleCut cut;
    cut.total = total;
    cut.by_count = r.top_k > 0 && r.top_k < tokens;
    cut.by_mass = r.top_p < 1.0f;
    cut.lo = kBins;
    cut.hi = -1;
    u64 least = total;   // of what the top_k's tokens weigh
    if (cut.by_count) {
        // the first bin with which there are top_k
        if (count_ahead < r.top_k && count_to >= r.top_k) {
            w.by_count = t;
            w.least = mass_ahead;
        }
        __syncthreads();
        cut.lo = cut.hi = w.by_count;
        least = w.least;
    }
    if (cut.by_mass) {
        // the last bin before which less than top_p of it lies; where the
        // top_k's weight is not known yet, from the least that it can be
        const double aim = static_cast<double>(r.top_p) * static_cast<double>(least);
        if (count > 0 && static_cast<double>(mass_ahead) < aim) atomicMax(&w.last, t);
        __syncthreads();
        if (cut.by_count) cut.lo = min(cut.lo, w.last);
        else cut.lo = cut.hi = w.last;
    }
    if (t == min(cut.lo, kBins - 1)) {
        w.mass_before = cut.lo < kBins ? mass_ahead : total;
        w.count_before = cut.lo < kBins ? count_ahead : tokens;
    }
    __syncthreads();
    cut.mass_before = w.mass_before;
    cut.count_before = w.count_before;
    return cut;
}

template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_gather_kernel(SampleArgs a) {
    const int b = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int i0 = blockIdx.x * a.per, i1 = min(i0 + a.per, a.vocab);
    float l[kBatch];
    load_logits<DT>(a, b, i0 + wave * kBatch * 64 + lane, 64, i1, l);
    const Row r = row_of(a, b);
    const float2 range = row_range(a, b);
    if (r.first || range.x == -INFINITY) return;
    __shared__ CutWork cut_work;
    __shared__ int wcount[kSampleThreads / 64];
    __shared__ u64 wmass[kSampleThreads / 64];
    const SampleCut cut = find_cut(a, r, b, cut_work);
    if (blockIdx.x == 0 && t == 0) a.w.cut[b] = cut;
    const Weigher weigh(r, range.x);
    const Binner bin(r, range.x, range.y);
    const bool border = cut.lo <= cut.hi, sift = r.min_p > 0.0f;
    u64 base = 0;   // what the chunk's tokens of the bins before lo weigh
    int listed = 0;
    if (border || sift) {
        int32_t* const list = a.w.list + static_cast<size_t>(b) * a.vocab + i0;
        // a wave's tokens of a batch follow one another
        for (int j = i0; j < i1; j += kBatch * kSampleThreads) {
            const int at0 = j + wave * kBatch * 64 + lane;
            if (j > i0) load_logits<DT>(a, b, at0, 64, i1, l);
            uint64_t m[kBatch];
            int own = 0;
#pragma unroll
            for (int q = 0; q < kBatch; ++q) {
                const int k = l[q] > -INFINITY ? bin(l[q]) : kBins;
                bool mine = false;
                if (k < cut.lo && k < kBins) {
                    if (sift) {
                        const double e = weigh.e(l[q]);
                        if (weigh.passes(e)) base += Weigher::units(e);
                    }
                } else if (k <= cut.hi) {
                    mine = weigh.mass(l[q]) > 0;
                }
                m[q] = __ballot(mine);
                own += __popcll(m[q]);
            }
            if (!border) continue;
            if (lane == 0) wcount[wave] = own;
            __syncthreads();
            int at = listed;
            for (int w = 0; w < kSampleThreads / 64; ++w) {
                if (w < wave) at += wcount[w];
                listed += wcount[w];
            }
#pragma unroll
            for (int q = 0; q < kBatch; ++q) {
                if (m[q] >> lane & 1) list[at + __popcll(m[q] & ((1ull << lane) - 1))] = at0 + 64 * q;
                at += __popcll(m[q]);
            }
            __syncthreads();
        }
    }
    if (!sift && t < cut.lo) base = a.w.bin_mass[bins_at(b, blockIdx.x) + t];
    base = wave_sum_u64(base);
    if (lane == 0) wmass[wave] = base;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < kSampleThreads / 64; ++w) base += wmass[w];
        a.w.base[b * kSampleChunks + blockIdx.x] = base;
        a.w.listed[b * kSampleChunks + blockIdx.x] = listed;
    }
}

// A border among the listed tokens: those with a larger key are kept, and the
// first `ties` of those with this one.
struct Border {
    uint32_t key;
    long long ties;
};

template <int DT>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs a) {
    constexpr int kWaves = kPickThreads / 64;
    const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const Row r = row_of(a, b);
    const float2 range = row_range(a, b);
    __shared__ int found;
    __shared__ u64 sums[256];
    __shared__ uint32_t counts[256];
    __shared__ int first[kSampleChunks + 1];
    __shared__ u64 kept[kSampleChunks];
    __shared__ Border pass;
    __shared__ u64 carry, digit_mass;
    __shared__ int wcount[kWaves];

    if (range.x == -INFINITY) {
        if (t == 0) {
            a.tokens[b] = -1;
            if (a.probs) a.probs[b] = 0.0f;
        }
        return;
    }
    if (r.first) {
        // the first chunk with the largest logit, the first token there
        const float m = a.w.range[b * kSampleChunks + min(lane, a.chunks - 1)].x;
        const int chunk = static_cast<int>(__builtin_ctzll(__ballot(m == range.x)));
        if (t == 0) found = a.vocab;
        __syncthreads();
        const int i0 = chunk * a.per, i1 = min(i0 + a.per, a.vocab);
        for (int i = i0 + t; i < i1; i += kPickThreads)
            if (logit<DT>(a, b, i) == range.x) {
                atomicMin(&found, i);
                break;
            }
        __syncthreads();
        if (t == 0) {
            a.tokens[b] = found;
            if (a.probs) a.probs[b] = 1.0f;
        }
        return;
    }
    const Weigher weigh(r, range.x);
    const SampleCut cut = a.w.cut[b];
    const bool border = cut.lo <= cut.hi;

    // where each chunk's listed tokens begin, end to end
    if (wave == 0) {
        const int n = border && lane < a.chunks ? a.w.listed[b * kSampleChunks + lane] : 0;
        const int to = wave_inclusive_scan_int(n);
        first[lane] = to - n;
        if (lane == 63) first[64] = to;
        kept[lane] = lane < a.chunks ? a.w.base[b * kSampleChunks + lane] : 0;
    }
    __syncthreads();
    const int n = first[a.chunks];
    const int32_t* const lists = a.w.list + static_cast<size_t>(b) * a.vocab;
    auto chunk_of = [&](int k) {   // the last chunk that begins at or before k
        int lo = 0, hi = a.chunks;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            (first[mid] <= k ? lo : hi) = mid;
        }
        return lo;
    };
    // a listed token: its key, then its index
    auto read_entry = [&](int k) {
        const int c = chunk_of(k), i = lists[static_cast<size_t>(c) * a.per + (k - first[c])];
        return static_cast<u64>(key_of(logit<DT>(a, b, i))) << 32 | static_cast<uint32_t>(i);
    };
    __shared__ u64 cache[kPickCache];
    const bool cached = n <= kPickCache;
    uint32_t differ = 0;   // the keys' bits that are not all alike
    if (n > 0) {
        const uint32_t any = read_entry(0) >> 32;
#pragma unroll 4
        for (int k = t; k < n; k += kPickThreads) {
            const u64 e = read_entry(k);
            if (cached) cache[k] = e;
            differ |= static_cast<uint32_t>(e >> 32) ^ any;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) differ |= __shfl_xor(static_cast<int>(differ), d);
        if (t == 0) found = 0;
        __syncthreads();
        if (lane == 0 && differ) atomicOr(&found, static_cast<int>(differ));
        __syncthreads();
        differ = found;
    }
    auto entry = [&](int k) { return cached ? cache[k] : read_entry(k); };
    // the selections' digits begin at the highest of these bits; those above it are the first token's
    const int bits = 32 - (differ ? __builtin_clz(differ) : 32), top = bits > 8 ? bits : 8;
    const uint32_t alike = n > 0 && top < 32 ? static_cast<uint32_t>(entry(0) >> 32) & (~0u << top) : 0u;

    // The border where `by_mass`: the last token before which (with `before` ahead of
    // the listed ones) less than `aim` lies; else: the aim-th token. Only keys
    // above `least`, and the first `least_ties` of that one, count. Returns what is
    // kept and weighs: `before`, and what the listed tokens to the border weigh.
    auto select = [&](bool by_mass, double aim_mass, long long aim_count, u64 before, uint32_t least, long long least_ties,
                      Border& out) {
        uint32_t prefix = alike;
        u64 ahead = before;
        long long rank = aim_count;   // still to be taken
        for (int end = top; end > 0; end = max(end - 8, 0)) {   // bits [sh, end), eight or (the last) the rest
            const int sh = max(end - 8, 0);
            __syncthreads();   // (the scan before has been read)
            for (int i = t; i < 256; i += kPickThreads) {
                sums[i] = 0;
                counts[i] = 0;
            }
            __syncthreads();
            const uint32_t mask = end < 32 ? ~0u << end : 0u;
            for (int k = t; k < n; k += kPickThreads) {
                const uint32_t key = entry(k) >> 32;
                if ((key & mask) != prefix || key < least) continue;
                const int d = key >> sh & ((1 << (end - sh)) - 1);
                atomicAdd(&counts[d], 1u);
                atomicAdd(&sums[d], weigh.mass(logit_of(key)));
            }
            __syncthreads();
            if (wave == 0) {
                // digits in descending order, four a lane
                u64 m[4], own = 0;
                uint32_t c[4], ownc = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 255 - (4 * lane + i);
                    m[i] = sums[d];
                    c[i] = counts[d];
                    own += m[i];
                    ownc += c[i];
                }
                u64 am = ahead + wave_scan_u64(own) - own, ac = wave_inclusive_scan_int(static_cast<int>(ownc)) - ownc;
                int mine = -1;
                u64 mine_ahead = 0, mine_count = 0, mine_mass = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = c[i] > 0 && (by_mass ? static_cast<double>(am) < aim_mass : ac < static_cast<u64>(rank));
                    if (in) {
                        mine = 255 - (4 * lane + i);
                        mine_ahead = am;
                        mine_count = ac;
                        mine_mass = m[i];
                    }
                    am += m[i];
                    ac += c[i];
                }
                const uint64_t who = __ballot(mine >= 0);
                if (who && lane == 63 - static_cast<int>(__builtin_clzll(who))) {
                    pass.key = prefix | static_cast<uint32_t>(mine) << sh;
                    pass.ties = rank - static_cast<long long>(mine_count);
                    carry = mine_ahead;
                    digit_mass = mine_mass;
                    found = counts[mine];
                }
            }
            __syncthreads();
            prefix = pass.key;
            ahead = carry;
            if (!by_mass) rank = pass.ties;
        }
        // the tokens with this key weigh the same
        const long long same = found;
        const u64 each = digit_mass / static_cast<u64>(same);
        long long ties = same;
        if (by_mass) {
            // those before which less than the aim lies: the first does
            if (each) {
                const double room = aim_mass - static_cast<double>(ahead);
                ties = static_cast<long long>(fmin(ceil(room / static_cast<double>(each)), static_cast<double>(same)));
                while (ties > 1 && !(static_cast<double>(ahead + (ties - 1) * each) < aim_mass)) --ties;
                while (ties < same && static_cast<double>(ahead + ties * each) < aim_mass) ++ties;
                if (ties < 1) ties = 1;
            }
        } else {
            ties = rank < same ? rank : same;
        }
        if (prefix == least && ties > least_ties) ties = least_ties;
        out.key = prefix;
        out.ties = ties;
        __syncthreads();
        return ahead + static_cast<u64>(ties) * each;
    };

    Border last{0, 1ll << 40};
    if (border) {
        u64 weight = cut.total;
        if (cut.by_count) weight = select(false, 0.0, r.top_k - cut.count_before, cut.mass_before, 0, 1ll << 40, last);
        if (cut.by_mass) {
            const Border by_count = last;
            select(true, static_cast<double>(r.top_p) * static_cast<double>(weight), 0, cut.mass_before, by_count.key,
                   by_count.ties, last);
        }
    }
    // the index up to which tokens with the border's key are kept
    int last_index = a.vocab;
    if (border) {
        if (t == 0) found = a.vocab;
        long long seen = 0;
        __syncthreads();
        for (int k0 = 0; k0 < n; k0 += kPickThreads) {
            const int k = k0 + t;
            const u64 e = k < n ? entry(k) : 0;
            const bool tie = k < n && static_cast<uint32_t>(e >> 32) == last.key;
            const uint64_t m = __ballot(tie);
            if (lane == 0) wcount[wave] = __popcll(m);
            __syncthreads();
            long long at = seen + __popcll(m & ((1ull << lane) - 1));
            for (int w = 0; w < kWaves; ++w) {
                if (w < wave) at += wcount[w];
                seen += wcount[w];
            }
            if (tie && at == last.ties - 1) found = static_cast<uint32_t>(e);
            __syncthreads();
            if (seen >= last.ties) break;
        }
        last_index = found;
    }
    auto keeps = [&](uint32_t key, int i) { return key > last.key || (key == last.key && i <= last_index); };
    // each chunk's kept weight
    for (int k = t; k < n; k += kPickThreads) {
        const u64 at = entry(k);
        const uint32_t key = at >> 32;
        if (!keeps(key, static_cast<int>(static_cast<uint32_t>(at)))) continue;
        const double e = weigh.e(logit_of(key));
        if (weigh.passes(e)) atomicAdd(&kept[chunk_of(k)], Weigher::units(e));
    }
    __syncthreads();
    // the chunk that u falls into, the same in every wave
    const u64 own = lane < a.chunks ? kept[lane] : 0, to = wave_scan_u64(own), total = lane_u64(to, 63);
    const double u = fmin(fmax(static_cast<double>(a.u[b]), 0.0), 1.0);
    u64 aim = static_cast<u64>(floor(u * static_cast<double>(total)));
    if (aim > total - 1) aim = total - 1;
    const int chunk = static_cast<int>(__builtin_ctzll(__ballot(to > aim)));
    u64 before = lane_u64(to - own, chunk);
    // the 64 tokens of it that hold this one, and the token there
    __shared__ u64 groups[kGroups];
    const int i0 = chunk * a.per, i1 = min(i0 + a.per, a.vocab), n64 = (i1 - i0 + 63) / 64;
    auto mass_at = [&](int i, float l) -> u64 {
        if (!(l > -INFINITY) || !keeps(key_of(l), i)) return 0;
        const double e = weigh.e(l);
        return weigh.passes(e) ? Weigher::units(e) : 0;
    };
    for (int g0 = wave; g0 < n64; g0 += 4 * kWaves) {
        float l[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) l[q] = logit<DT>(a, b, min(i0 + 64 * (g0 + q * kWaves) + lane, i1 - 1));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int g = g0 + q * kWaves, i = i0 + 64 * g + lane;
            const u64 m = wave_sum_u64(i < i1 ? mass_at(i, l[q]) : 0);
            if (lane == 0 && g < n64) groups[g] = m;
        }
    }
    __syncthreads();
    if (wave != 0) return;
    const int each = (n64 + 63) / 64;
    u64 sum = 0;
    for (int k = 0; k < each; ++k)
        if (each * lane + k < n64) sum += groups[each * lane + k];
    u64 upto = before + wave_scan_u64(sum);
    const int src = static_cast<int>(__builtin_ctzll(__ballot(upto > aim) | 1ull << 63));
    before = lane_u64(upto - sum, src);
    int g = each * src;
    while (g + 1 < n64 && before + groups[g] <= aim) before += groups[g++];
    const int i = i0 + 64 * g + lane;
    const u64 m = i < i1 ? mass_at(i, logit<DT>(a, b, i)) : 0;
    const u64 at = before + wave_scan_u64(m);
    if (m && at > aim && at - m <= aim) {
        a.tokens[b] = i;
        if (a.probs) a.probs[b] = static_cast<float>(static_cast<double>(m) / static_cast<double>(total));
    }
}

}  // namespace

hipError_t launch_sample(qff_ctx* ctx, hipStream_t stream, const void* logits, qff_dtype dtype, const float* u,
                         const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         int32_t* tokens, float* probs, int vocab, int batch) {
    SampleArgs a{logits, u, temperature, top_k, top_p, min_p, tokens, probs, vocab, 0, 0, ctx->sample};
    // four workgroups a CU over all rows, 64 a row at most (32 rows of 151936: 66 us, with two a CU 70)
    const int chunks = std::min(std::max(4 * ctx->num_cu / batch, 8), kSampleChunks);
    a.per = (vocab + chunks - 1) / chunks;
    a.chunks = (vocab + a.per - 1) / a.per;
    const dim3 grid(a.chunks, batch);
#define QFF_SAMPLE(KERNEL, GRID, THREADS)                                            \
    {                                                                                \
        ProfScope prof(ctx, stream, #KERNEL);                                        \
        if (dtype == QFF_BF16) KERNEL##_kernel<1><<<GRID, THREADS, 0, stream>>>(a);  \
        else KERNEL##_kernel<0><<<GRID, THREADS, 0, stream>>>(a);                    \
    }
    QFF_SAMPLE(sample_max, grid, kSampleThreads)
    QFF_SAMPLE(sample_bins, grid, kSampleThreads)
    QFF_SAMPLE(sample_gather, grid, kSampleThreads)
    QFF_SAMPLE(sample_pick, batch, kPickThreads)
#undef QFF_SAMPLE
    return hipGetLastError();
}

}  // namespace qff
