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
//   bins    each chunk's counts and weights in 64 bins of equal width in l
//   gather  every chunk adds the bins up, finds the bins [lo, hi] that hold the
//           borders of top-k and top-p, and lists its tokens in them in order;
//           the tokens of the bins before lo are kept
//   pick    one workgroup a row: the borders among the listed tokens by an
//           8-bit radix selection over the bits of l (by count, then by weight),
//           the chunk that u falls into and the token in it
// A row is read four times at most (three from the caches: 0.6 MB at 151936
// logits); rows that need no border or no draw skip what they do not need.
#include <algorithm>

#include "common.hpp"
#include "internal.hpp"

namespace qff {

namespace {

typedef unsigned long long u64;

constexpr int kBins = 64, kCopies = 16;   // LDS copies of a chunk's bins: lanes of equal logits meet in fewer of them
constexpr int kSampleThreads = 256, kPickThreads = 1024;
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

// Monotone in l: larger logits have larger keys.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t u = __float_as_uint(l == 0.0f ? 0.0f : l);   // (-0 and 0 are equal)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// e^((l - best) / t) and its weight.
struct Weigher {
    double best, t, min_p;
    float bestf;
    __device__ __forceinline__ Weigher(const Row& r, float best_) : best(best_), t(r.t), min_p(r.min_p), bestf(best_) {}
    __device__ __forceinline__ double e(float l) const {
        if (l == bestf) return 1.0;
        const double d = (static_cast<double>(l) - best) / t;
        return d > -31.3 ? exp(d) : 0.0;   // (e^-31.3 rounds to no unit)
    }
    static __device__ __forceinline__ u64 units(double e) { return static_cast<u64>(rint(e * kUnit)); }
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

__device__ __forceinline__ u64 shfl_u64(u64 v, int src) {
    const uint32_t lo = __shfl(static_cast<int>(v), src), hi = __shfl(static_cast<int>(v >> 32), src);
    return static_cast<u64>(hi) << 32 | lo;
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += shfl_u64(v, (threadIdx.x & 63) ^ d);
    return v;
}
// Sum over the lanes before and up to this one.
__device__ __forceinline__ u64 wave_scan_u64(u64 v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = shfl_u64(v, lane - d & 63);
        if (lane >= d) v += o;
    }
    return v;
}

template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_max_kernel(SampleArgs a) {
    const int b = blockIdx.y, i0 = blockIdx.x * a.per, i1 = min(i0 + a.per, a.vocab);
    float hi = -INFINITY, lo = INFINITY;
    for (int i = i0 + threadIdx.x; i < i1; i += kSampleThreads) {
        const float l = logit<DT>(a, b, i);
        hi = fmaxf(hi, l);
        if (l > -INFINITY) lo = fminf(lo, l);
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
    for (int i = i0 + t; i < i1; i += kSampleThreads) {
        const float l = logit<DT>(a, b, i);
        const u64 m = weigh.mass(l);
        if (m == 0) continue;
        const int k = bin(l);
        atomicAdd(&mass[k][t % kCopies], m);
        atomicAdd(&count[k][t % kCopies], 1u);
    }
    __syncthreads();
    if (t < kBins) {
        u64 m = 0;
        uint32_t n = 0;
        for (int c = 0; c < kCopies; ++c) {
            m += mass[t][(c + t) % kCopies];
            n += count[t][(c + t) % kCopies];
        }
        const size_t o = (static_cast<size_t>(b) * kSampleChunks + blockIdx.x) * kBins + t;
        a.w.bin_mass[o] = m;
        a.w.bin_count[o] = n;
    }
}

// The bins that hold the borders, the same in every chunk's workgroup: bins
// before lo are kept whole, those past hi not at all. lo > hi: there is no border.
__device__ __forceinline__ SampleCut find_cut(const SampleArgs& a, const Row& r, int b, u64 (&ms)[kBins], uint32_t (&cs)[kBins]) {
    const int t = threadIdx.x;
    if (t < kBins) {
        ms[t] = 0;
        cs[t] = 0;
    }
    __syncthreads();
    {
        u64 m = 0;
        uint32_t n = 0;
        for (int c = t / kBins; c < a.chunks; c += kSampleThreads / kBins) {
            const size_t o = (static_cast<size_t>(b) * kSampleChunks + c) * kBins + t % kBins;
            m += a.w.bin_mass[o];
            n += a.w.bin_count[o];
        }
        atomicAdd(&ms[t % kBins], m);
        atomicAdd(&cs[t % kBins], n);
    }
    __syncthreads();
    const int lane = t & 63;
    const u64 mass = ms[lane], mass_to = wave_scan_u64(mass);
    const uint32_t count = cs[lane];
    const u64 count_to = wave_scan_u64(count);
    const u64 total = shfl_u64(mass_to, 63), tokens = shfl_u64(count_to, 63);
    SampleCut cut;
    cut.total = total;
    cut.by_count = r.top_k > 0 && static_cast<u64>(r.top_k) < tokens;
    cut.by_mass = r.top_p < 1.0f;
    cut.lo = kBins;
    cut.hi = -1;
    u64 least = total;   // of what the top_k's tokens weigh
    if (cut.by_count) {
        // the first bin with which there are top_k
        const uint64_t m = __ballot(count_to >= static_cast<u64>(r.top_k));
        cut.lo = cut.hi = static_cast<int>(__builtin_ctzll(m));
        least = shfl_u64(mass_to, cut.hi) - shfl_u64(mass, cut.hi);
    }
    if (cut.by_mass) {
        // the last bin before which less than top_p of it lies; where the
        // top_k's weight is not known yet, from the least that it can be
        const double aim = static_cast<double>(r.top_p) * static_cast<double>(least);
        const uint64_t m = __ballot(count > 0 && static_cast<double>(mass_to - mass) < aim) | 1;
        const int last = 63 - static_cast<int>(__builtin_clzll(m));
        if (cut.by_count) {
            cut.lo = min(cut.lo, last);
        } else {
            cut.lo = cut.hi = last;
        }
    }
    const int at = min(cut.lo, kBins - 1);
    const u64 mb = shfl_u64(mass_to - mass, at), cb = shfl_u64(count_to - count, at);
    cut.mass_before = cut.lo < kBins ? mb : total;
    cut.count_before = static_cast<int>(cut.lo < kBins ? cb : tokens);
    return cut;
}

template <int DT>
__global__ __launch_bounds__(kSampleThreads) void sample_gather_kernel(SampleArgs a) {
    const int b = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int i0 = blockIdx.x * a.per, i1 = min(i0 + a.per, a.vocab);
    const Row r = row_of(a, b);
    const float2 range = row_range(a, b);
    if (r.first || range.x == -INFINITY) return;
    __shared__ u64 ms[kBins];
    __shared__ uint32_t cs[kBins];
    __shared__ int wcount[kSampleThreads / 64];
    __shared__ u64 wmass[kSampleThreads / 64];
    const SampleCut cut = find_cut(a, r, b, ms, cs);
    if (blockIdx.x == 0 && t == 0) a.w.cut[b] = cut;
    const Weigher weigh(r, range.x);
    const Binner bin(r, range.x, range.y);
    const bool border = cut.lo <= cut.hi, sift = r.min_p > 0.0f;
    u64 base = 0;   // what the chunk's tokens of the bins before lo weigh
    int listed = 0;
    if (border || sift) {
        int32_t* const list = a.w.list + static_cast<size_t>(b) * a.vocab + i0;
        for (int j = i0; j < i1; j += kSampleThreads) {
            const int i = j + t;
            const float l = i < i1 ? logit<DT>(a, b, i) : -INFINITY;
            const int k = l > -INFINITY ? bin(l) : kBins;
            bool mine = false;
            if (k < cut.lo && k < kBins) {
                if (sift) {
                    const double e = weigh.e(l);
                    if (weigh.passes(e)) base += Weigher::units(e);
                }
            } else if (k <= cut.hi) {
                mine = weigh.mass(l) > 0;
            }
            if (border) {
                const uint64_t m = __ballot(mine);
                if (lane == 0) wcount[wave] = __popcll(m);
                __syncthreads();
                int at = listed + __popcll(m & ((1ull << lane) - 1));
                for (int w = 0; w < kSampleThreads / 64; ++w) {
                    if (w < wave) at += wcount[w];
                    listed += wcount[w];
                }
                if (mine) list[at] = i;
                __syncthreads();
            }
        }
    }
    if (!sift && t < kBins && t < cut.lo)
        base = a.w.bin_mass[(static_cast<size_t>(b) * kSampleChunks + blockIdx.x) * kBins + t];
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
    auto token_at = [&](int k) {
        const int c = chunk_of(k);
        return lists[static_cast<size_t>(c) * a.per + (k - first[c])];
    };

    // The border where `by_mass`: the last token before which (with `before` ahead of
    // the listed ones) less than `aim` lies; else: the aim-th token. Only keys
    // above `least`, and the first `least_ties` of that one, count. Returns what is
    // kept and weighs: `before`, and what the listed tokens to the border weigh.
    auto select = [&](bool by_mass, double aim_mass, long long aim_count, u64 before, uint32_t least, long long least_ties,
                      Border& out) {
        uint32_t prefix = 0;
        u64 ahead = before;
        long long rank = aim_count;   // still to be taken
        for (int sh = 24; sh >= 0; sh -= 8) {
            for (int i = t; i < 256; i += kPickThreads) {
                sums[i] = 0;
                counts[i] = 0;
            }
            __syncthreads();
            const uint32_t mask = sh == 24 ? 0u : ~0u << (sh + 8);
            for (int k = t; k < n; k += kPickThreads) {
                const float l = logit<DT>(a, b, token_at(k));
                const uint32_t key = key_of(l);
                if ((key & mask) != prefix || key < least) continue;
                const int d = key >> sh & 255;
                atomicAdd(&counts[d], 1u);
                atomicAdd(&sums[d], weigh.mass(l));
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
                u64 am = ahead + wave_scan_u64(own) - own, ac = wave_scan_u64(ownc) - ownc;
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
            __syncthreads();
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
            const int i = k < n ? token_at(k) : -1;
            const bool tie = i >= 0 && key_of(logit<DT>(a, b, i)) == last.key;
            const uint64_t m = __ballot(tie);
            if (lane == 0) wcount[wave] = __popcll(m);
            __syncthreads();
            long long at = seen + __popcll(m & ((1ull << lane) - 1));
            for (int w = 0; w < kWaves; ++w) {
                if (w < wave) at += wcount[w];
                seen += wcount[w];
            }
            if (tie && at == last.ties - 1) found = i;
            __syncthreads();
            if (seen >= last.ties) break;
        }
        last_index = found;
    }
    auto keeps = [&](float l, int i) {
        const uint32_t key = key_of(l);
        return key > last.key || (key == last.key && i <= last_index);
    };
    // each chunk's kept weight
    for (int c = wave; c < a.chunks && border; c += kWaves) {
        u64 m = 0;
        for (int k = first[c] + lane; k < first[c + 1]; k += 64) {
            const int i = lists[static_cast<size_t>(c) * a.per + (k - first[c])];
            const float l = logit<DT>(a, b, i);
            const double e = weigh.e(l);
            if (keeps(l, i) && weigh.passes(e)) m += Weigher::units(e);
        }
        m = wave_sum_u64(m);
        if (lane == 0) kept[c] += m;
    }
    __syncthreads();
    // the chunk that u falls into, the same in every wave
    const u64 own = lane < a.chunks ? kept[lane] : 0, to = wave_scan_u64(own), total = shfl_u64(to, 63);
    const double u = fmin(fmax(static_cast<double>(a.u[b]), 0.0), 1.0);
    u64 aim = static_cast<u64>(floor(u * static_cast<double>(total)));
    if (aim > total - 1) aim = total - 1;
    const int chunk = static_cast<int>(__builtin_ctzll(__ballot(to > aim)));
    u64 before = shfl_u64(to - own, chunk);
    // and the token there: a wave's 64 tokens after the other
    __shared__ u64 wsum[kWaves];
    const int i0 = chunk * a.per, i1 = min(i0 + a.per, a.vocab);
    for (int j = i0; j < i1; j += kPickThreads) {
        const int i = j + t;
        u64 m = 0;
        if (i < i1) {
            const float l = logit<DT>(a, b, i);
            if (l > -INFINITY && keeps(l, i)) {
                const double e = weigh.e(l);
                if (weigh.passes(e)) m = Weigher::units(e);
            }
        }
        const u64 upto = wave_scan_u64(m);
        if (lane == 63) wsum[wave] = upto;
        __syncthreads();
        u64 at = before + upto, all = 0;
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) at += wsum[w];
            all += wsum[w];
        }
        if (m && at > aim && at - m <= aim) {
            a.tokens[b] = i;
            if (a.probs) a.probs[b] = static_cast<float>(static_cast<double>(m) / static_cast<double>(total));
        }
        before += all;
        if (before > aim) break;
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_sample(qff_ctx* ctx, hipStream_t stream, const void* logits, qff_dtype dtype, const float* u,
                         const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         int32_t* tokens, float* probs, int vocab, int batch) {
    SampleArgs a{logits, u, temperature, top_k, top_p, min_p, tokens, probs, vocab, 0, 0, ctx->sample};
    // two workgroups a CU over all rows, 64 a row at most
    const int chunks = std::min(std::max(2 * ctx->num_cu / batch, 8), kSampleChunks);
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
