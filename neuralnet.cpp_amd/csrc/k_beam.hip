// k_beam.hip — beam search's selection: of each group's beams * vocab
// continuations, with totals score + logit - log(sum exp(logits of the beam)),
// the best `take`, equal totals in the order of their index beam * vocab + token.
//
// One pass over the logits leaves, for every segment of neighbouring tokens of
// a beam, the largest logit and the sum of exp(logit - largest): the sums make
// the beam's log-sum-exp, and the best `take` candidates lie in the best
// `take` segments (a segment that ranks behind `take` others, by its largest
// total and then its index, holds nothing that ranks before the best of each
// of those). Only these segments are read again. Totals are formed in float64,
// so that candidates of different beams compare as exactly as the sums allow.
#include "common.hpp"
#include "kv_pages.hpp"

namespace nnhip
{
namespace
{

constexpr unsigned kSegColumn = 64;   // tokens that a thread loads at once, (vocab, beams) logits
constexpr unsigned kSegRow = 256;     // tokens that 16 lanes load at once, (beams, vocab) logits
constexpr unsigned kSegMost = 4096;
constexpr unsigned kSegments = 32768; // segments of a group that the selection looks at, unless they grew to kSegMost
constexpr unsigned kStored = 8192;    // segments of a group whose bins the selection keeps in LDS
constexpr int kMaxTake = 256;
constexpr int kMaxBeams = 1024;
constexpr int kList = 512;        // candidates that are ranked one against another
constexpr unsigned kFew = 128;    // segments of a group that are ranked at once
constexpr int kLog2Bins = 10, kBins = 1 << kLog2Bins;
constexpr int kPickThreads = 1024;

struct BeamArgs
{
    const float *logits, *scores, *done;
    size_t ld;
    unsigned groups, beams, vocab, take, eos, n_seg, seg;
    unsigned log2_seg;
    FastDiv by_n_seg;
    int beam_major;
    float2* part;   // per (beam of all groups, segment): largest logit, sum of exp(logit - largest)
    float *out_score, *out_beam, *out_token;
};

// exp(x - m) of a logit and its segment's largest, m as 0 where that is -inf. The product with log2(e) is kept
// in two parts: its rounding alone would be off by up to 2^-24 |x - m|.
__device__ __forceinline__ float exp_below(float x, float m)
{
    constexpr float kHi = 1.44269502e+0f, kLo = 1.92596299e-8f, kLn2 = 6.93147182e-1f;   // log2(e) = kHi + kLo
    const float d = x - m, y = d * kHi;
    const float r = __builtin_fmaf(d, kHi, -y) + d * kLo;
    const float e = __builtin_amdgcn_exp2f(y);
    return e == 0.0f ? 0.0f : __builtin_fmaf(e, r * kLn2, e);   // r is NaN for d = -inf
}

// Takes a further part of a segment (largest m2, sum s2 of exp(logit - m2), m2 as 0 where it is -inf) in.
__device__ __forceinline__ void take_in(float& m, float& s, float m2, float s2)
{
    const float mn = fmax_std(m, m2), base = mn == -__builtin_inff() ? 0.0f : mn;
    // an all -inf part has the sum 0 (or NaN), whatever its factor is
    s = s * exp_below(m, base) + s2 * exp_below(m2, base);
    m = mn;
}

// Bound by HBM and its latency: 7 us for 32000 x 16 logits in columns, 16.6 us for 224 rows of 100003 (90 MB,
// 5.4 TB/s).
//
// (vocab, beams) logits: a thread takes one segment of one beam, neighbouring threads neighbouring beams.
__global__ __launch_bounds__(256) void k_beam_segments_column(BeamArgs a)
{
    const unsigned all = a.groups * a.beams;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)all * a.n_seg) return;
    const unsigned seg = (unsigned)(i / all), n = (unsigned)(i % all);
    if (a.done && a.done[n] != 0.0f) return;
    float m = -__builtin_inff(), s = 0.0f;
    const unsigned v1 = min((seg + 1) * a.seg, a.vocab);
    for (unsigned v0 = seg * a.seg; v0 < v1; v0 += kSegColumn)
    {
        const unsigned nv = min(kSegColumn, v1 - v0);
        const float* p = a.logits + (size_t)v0 * a.ld + n;
        float x[kSegColumn], mc = -__builtin_inff(), sc = 0.0f;
#pragma unroll
        for (unsigned k = 0; k < kSegColumn; ++k) x[k] = k < nv ? p[(size_t)k * a.ld] : -__builtin_inff();
#pragma unroll
        for (unsigned k = 0; k < kSegColumn; ++k) mc = fmax_std(mc, x[k]);
        const float base = mc == -__builtin_inff() ? 0.0f : mc;
#pragma unroll
        for (unsigned k = 0; k < kSegColumn; ++k) sc += exp_below(x[k], base);
        if (v0 == seg * a.seg)
        {
            m = mc;
            s = sc;
        }
        else take_in(m, s, mc, sc);
    }
    a.part[(size_t)n * a.n_seg + seg] = make_float2(m, s);
}

// (beams, vocab) logits: 16 lanes take one segment of one beam.
__global__ __launch_bounds__(256) void k_beam_segments_row(BeamArgs a)
{
    constexpr int kPer = kSegRow / 16;
    const unsigned lane = threadIdx.x & 15, i = blockIdx.x * 16 + (threadIdx.x >> 4), n = a.by_n_seg.div(i);
    if (n >= a.groups * a.beams || (a.done && a.done[n] != 0.0f)) return;   // whole groups of 16 lanes
    const unsigned seg = i - n * a.n_seg;
    const float* p = a.logits + (size_t)n * a.ld;
    float m = -__builtin_inff(), s = 0.0f;
    const unsigned v1 = min((seg + 1) * a.seg, a.vocab);
    for (unsigned v0 = seg * a.seg; v0 < v1; v0 += kSegRow)
    {
        float x[kPer], mc = -__builtin_inff(), sc = 0.0f;
#pragma unroll
        for (int k = 0; k < kPer; ++k)
        {
            const unsigned v = v0 + 16 * k + lane;
            x[k] = v < v1 ? p[v] : -__builtin_inff();
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) mc = fmax_std(mc, x[k]);
        for (int o = 8; o > 0; o >>= 1) mc = fmax_std(mc, __shfl_xor(mc, o, 16));
        const float base = mc == -__builtin_inff() ? 0.0f : mc;
#pragma unroll
        for (int k = 0; k < kPer; ++k) sc += exp_below(x[k], base);
        for (int o = 8; o > 0; o >>= 1) sc += __shfl_xor(sc, o, 16);
        if (v0 == seg * a.seg)
        {
            m = mc;
            s = sc;
        }
        else take_in(m, s, mc, sc);
    }
    if (lane == 0) a.part[(size_t)n * a.n_seg + seg] = make_float2(m, s);
}

typedef unsigned long long u64;

// Totals as whole numbers of the same order; NaN as -inf, -0 as 0.
__device__ __forceinline__ u64 key_of(double x)
{
    if (x != x) x = -__builtin_inf();
    const u64 b = __builtin_bit_cast(u64, x + 0.0);
    return (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double value_of(u64 k)
{
    return __builtin_bit_cast(double, (k >> 63) ? k & ~(1ull << 63) : ~k);
}

struct PickShared
{
    double lse[kMaxBeams], best[kMaxBeams], sum[kMaxBeams];   // sum, top: of a wave's segments of a beam
    float score[kMaxBeams], top[kMaxBeams];
    unsigned char ended[kMaxBeams];
    u64 key[kList];
    unsigned idx[kList];
    unsigned hist[kBins];
    unsigned wave[kPickThreads / 64];
    u64 red[2][kPickThreads / 64];
    unsigned count, bin, above, wide;
    unsigned order[kMaxTake];   // items of the list by rank
    unsigned seg_beam[kMaxTake], seg_token[kMaxTake];   // of the best segments: beam and first token
    unsigned short bins[kStored];
};

// The bin in which the running count, from bin 0 on (or from the last one down), reaches k: s.bin, and the
// count before it, s.above; s.bin = kBins where it never does. The first wave's work, 16 bins a lane.
__device__ __forceinline__ void find_bin(PickShared& s, unsigned k, bool down)
{
    constexpr int kEach = kBins / 64;
    const int lane = threadIdx.x;
    if (lane < 64)
    {
        unsigned h[kEach], own = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
        {
            h[i] = s.hist[down ? kBins - 1 - (lane * kEach + i) : lane * kEach + i];
            own += h[i];
        }
        unsigned sum = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1)
        {
            const unsigned up = __shfl_up(sum, o, 64);
            if (lane >= o) sum += up;
        }
        if (lane == 63 && sum < k) s.bin = kBins;
        unsigned before = sum - own;
        if (sum >= k && before < k)
        {
            unsigned at = 0, above = before;
#pragma unroll
            for (int i = 0; i < kEach; ++i)
            {
                if (before < k)
                {
                    at = i;
                    above = before;
                }
                before += h[i];
            }
            s.bin = down ? kBins - 1 - (lane * kEach + at) : lane * kEach + at;
            s.above = above;
        }
    }
    __syncthreads();
}

// Puts into the list at most kList of n items, the first k by (key descending, index ascending) among them; k
// <= n, k <= kMaxTake. key(i) and index(i) give item i's; indices differ. A histogram over the keys' range
// narrows it to the bin that holds the k-th; where keys are equal, one over the indices follows. This takes any
// keys; the selection comes here where its quick way does not end in a short list.
template <class Key, class Index> __device__ __noinline__ void pick(PickShared& s, unsigned n, unsigned k, Key key, Index index)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const u64 neg_inf = key_of(-__builtin_inf());
    auto each = [&](auto&& f) {
        for (unsigned i = t; i < n; i += kPickThreads) f(i, key(i));
    };
    // Range of the keys above -inf, if those suffice.
    u64 lo = ~0ull, hi = 0;
    unsigned above_inf = 0;
    each([&](unsigned, u64 x) {
        hi = x > hi ? x : hi;
        if (x > neg_inf)
        {
            lo = x < lo ? x : lo;
            ++above_inf;
        }
    });
    for (int o = 32; o > 0; o >>= 1)
    {
        const u64 l2 = __shfl_xor(lo, o, 64), h2 = __shfl_xor(hi, o, 64);
        lo = l2 < lo ? l2 : lo;
        hi = h2 > hi ? h2 : hi;
        above_inf += __shfl_xor(above_inf, o, 64);
    }
    __syncthreads();
    if (lane == 0)
    {
        s.red[0][wave] = lo;
        s.red[1][wave] = hi;
        s.wave[wave] = above_inf;
    }
    __syncthreads();
    above_inf = 0;
    for (int w = 0; w < kPickThreads / 64; ++w)
    {
        lo = s.red[0][w] < lo ? s.red[0][w] : lo;
        hi = s.red[1][w] > hi ? s.red[1][w] : hi;
        above_inf += s.wave[w];
    }
    if (above_inf < k) lo = neg_inf;
    unsigned base = 0, ilo = 0, ihi = ~0u;   // base: items before the range
    bool by_index = false;
    for (;;)
    {
        __syncthreads();
        s.hist[t] = 0;
        __syncthreads();
        const u64 range = by_index ? (u64)(ihi - ilo) : hi - lo;
        const int shift = range ? max(0, 64 - __clzll((long long)range) - kLog2Bins) : 0;   // range >> shift < kBins
        each([&](unsigned i, u64 x) {
            if (x < lo || x > hi) return;
            if (!by_index) atomicAdd(&s.hist[(x - lo) >> shift], 1u);
            else
            {
                const unsigned idx = index(i);
                if (idx >= ilo && idx <= ihi) atomicAdd(&s.hist[(idx - ilo) >> shift], 1u);
            }
        });
        __syncthreads();
        find_bin(s, k - base, !by_index);
        const unsigned bin = s.bin, here = s.hist[bin];
        base += s.above;
        if (by_index)
        {
            const unsigned l2 = ilo + (bin << shift);
            const u64 h2 = (u64)l2 + ((1ull << shift) - 1);
            ilo = l2;
            ihi = h2 < ihi ? (unsigned)h2 : ihi;
        }
        else
        {
            const u64 l2 = lo + ((u64)bin << shift), h2 = l2 + ((1ull << shift) - 1);
            lo = l2;
            hi = h2 < hi && h2 >= l2 ? h2 : hi;
        }
        if (base + here <= kList) break;
        if (!by_index && lo == hi)
        {
            by_index = true;
            ilo = 0;
            ihi = ~0u;
        }
    }
    if (t == 0) s.count = 0;
    __syncthreads();
    each([&](unsigned i, u64 x) {
        if (x < lo) return;
        const unsigned idx = index(i);
        if (x > hi || !by_index || idx <= ihi)
        {
            const unsigned at = atomicAdd(&s.count, 1u);
            s.key[at] = x;
            s.idx[at] = idx;
        }
    });
    __syncthreads();
}

// order[r] = the list's item of rank r, r < k (whatever order the items came in: indices differ). 16 lanes an item.
__device__ __forceinline__ void rank_list(PickShared& s, unsigned k)
{
    const unsigned n = s.count, part = threadIdx.x & 15;
    for (unsigned i = threadIdx.x >> 4; i < n; i += kPickThreads / 16)
    {
        const u64 key = s.key[i];
        const unsigned idx = s.idx[i];
        unsigned r = 0;
#pragma unroll 4
        for (unsigned j = part; j < n; j += 16) r += s.key[j] > key || (s.key[j] == key && s.idx[j] < idx) ? 1u : 0u;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) r += __shfl_xor(r, o, 16);
        if (part == 0 && r < k) s.order[r] = i;
    }
    __syncthreads();
}

// One workgroup a group. The kernel runs once over little data, so its time is that of the loads it waits for one
// after another, of its instructions (one CU's) and of fetching them: loads go several at a time, loops stay loops,
// and most items are put aside by a float32 distance from the best total, before any 64-bit total is formed. 13 us for
// 4 x 1024 logits, 20 for 16 x 32000 and for 32 groups of 8 x 100003. Of these, by the cycle counter (2.4 GHz): the
// sums 4.9, 5.6 and 5.6, log-sum-exps and distances 1.8, 1.5 and 1.8, the best segments 0.6 (64 are ranked at once), 5.1
// and 4.1, their rank 1.3, 1.2 and 1.2, the best segments' tokens 2.3, 3.9 and 4.3, the last rank 0.7, and the launch.
__global__ __launch_bounds__(kPickThreads) void k_beam_pick(BeamArgs a)
{
    constexpr unsigned kWaves = kPickThreads / 64;
    __shared__ PickShared s;
    const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const unsigned b0 = blockIdx.x * a.beams, n_all = a.beams * a.n_seg, k_seg = min(a.take, n_all);
    const bool stored = n_all <= kStored;
    // A unit is a beam's segments, or where there are fewer beams than waves every 2^log2_slices-th 64 of them.
    unsigned log2_slices = 0;
    while ((a.beams << (log2_slices + 1)) <= kWaves) ++log2_slices;
    const unsigned slices = 1u << log2_slices, units = a.beams << log2_slices, step = 64 << log2_slices;
    const float2* part = a.part + (size_t)b0 * a.n_seg;
    s.hist[t] = 0;
    if (t == 0) s.count = s.wide = 0;
    static_assert(kMaxBeams <= kPickThreads);
    float score = 0.0f, done = 0.0f;   // of beam t, on their way with the segments
    if (t < a.beams)
    {
        score = a.scores[b0 + t];
        if (a.done) done = a.done[b0 + t];
    }
    // f(first of 8 segments, each step apart, their values) over a unit's segments.
    auto over_unit = [&](unsigned u, auto&& f) {
        const unsigned w = u >> log2_slices;
        const float2* p = part + (size_t)w * a.n_seg;
#pragma unroll 1
        for (unsigned i = (u - (w << log2_slices)) * 64 + lane; i < a.n_seg; i += 8 * step)
        {
            float2 x[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = p[min(i + step * r, a.n_seg - 1)];
            f(w, i, x);
        }
    };
#pragma unroll 1
    for (unsigned u = wave; u < units; u += kWaves)
    {
        // Lanes past the last segment have none: -inf and 0.
        float m = -__builtin_inff();
        double sum = 0.0;
        over_unit(u, [&](unsigned, unsigned i, const float2(&x)[8]) {
            float mn = m;
#pragma unroll
            for (int r = 0; r < 8; ++r) mn = fmax_std(mn, x[r].x);
            const float base = mn == -__builtin_inff() ? 0.0f : mn;
            if (m != mn) sum *= (double)exp_below(m, base);
            m = mn;
#pragma unroll
            for (int r = 0; r < 8; ++r)
            {
                const float e = x[r].y * exp_below(x[r].x, base);   // NaN where m is +inf, and so is the total
                sum += i + step * r < a.n_seg ? (double)e : 0.0;
            }
        });
        const float top = wave_max(m);
        sum *= (double)exp_below(m, top == -__builtin_inff() ? 0.0f : top);
#pragma unroll 1
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0)
        {
            s.top[u] = top;
            s.sum[u] = sum;
        }
    }
    __syncthreads();
    const bool ended = done != 0.0f;   // whose segments' sums are anything, and not used
    double lse = 0.0;
    if (t < a.beams)
    {
        const unsigned w = t;
        float m = -__builtin_inff();
#pragma unroll 1
        for (unsigned i = 0; i < slices; ++i) m = fmax_std(m, s.top[w * slices + i]);
        double sum = 0.0;
#pragma unroll 1
        for (unsigned i = 0; i < slices; ++i)
            sum += s.sum[w * slices + i] * (double)exp_below(s.top[w * slices + i], m == -__builtin_inff() ? 0.0f : m);
        lse = (double)m + log(sum);
        const double best = ended ? (double)score : (double)score + ((double)m - lse);
        s.score[w] = score;
        s.ended[w] = ended;
        s.lse[w] = lse;
        s.best[w] = best == best ? best : -__builtin_inf();
    }
    __syncthreads();
    double hi = -__builtin_inf();   // the best total
#pragma unroll 1
    for (unsigned w = lane; w < a.beams; w += 64) hi = s.best[w] > hi ? s.best[w] : hi;
#pragma unroll 1
    for (int o = 32; o > 0; o >>= 1)
    {
        const double h2 = __shfl_xor(hi, o, 64);
        hi = h2 > hi ? h2 : hi;
    }
    // A candidate lies near[w] - logit below the best, to within half a bin of 1/32 while near[w] is at most 2^16.
    float* near = s.top;
    __syncthreads();
    if (t < a.beams)
    {
        const float d = (float)(hi - (ended ? (double)score : (double)score - lse));
        near[t] = d;
        if (!(fabsf(d) <= 0x1p16f) && d != __builtin_inff()) s.wide = 1;
    }
    __syncthreads();
    // Totals, NaN as -inf.
    auto total = [&](unsigned w, bool is_eos, float logit) {
        const double sc = (double)s.score[w], x = s.ended[w] ? (is_eos ? sc : -__builtin_inf()) : sc + ((double)logit - s.lse[w]);
        return x == x ? x : -__builtin_inf();
    };
    const unsigned eos_seg = a.eos / a.seg;
    auto of_segment = [&](unsigned i) {
        const unsigned w = a.by_n_seg.div(i);
        return key_of(total(w, eos_seg == i - w * a.n_seg, part[i].x));
    };

    // The best segments. Bins of 1/32 over the 32 below the best total hold them, as a rule; the bin behind the
    // one where their count is reached is taken too, for the half bin that a distance may be off. Behind the last
    // bin there is none: a count that is reached there is left to pick.
    auto bin_of = [&](float distance) {
        const float d = distance * 32.0f;
        return d > -1.0f && d < (float)kBins ? (unsigned)(int)d : (unsigned)kBins;
    };
    // f(segment, bin) over all.
    auto over_bins = [&](auto&& f) {
#pragma unroll 1
        for (unsigned u = wave; u < units; u += kWaves)
        {
            const unsigned beam = u >> log2_slices;
            const bool over = s.ended[beam];
            const float dist = near[beam];
            over_unit(u, [&](unsigned w, unsigned i, const float2(&x)[8]) {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                {
                    const unsigned g = i + step * r;
                    if (g < a.n_seg)
                        f(w * a.n_seg + g, !over ? bin_of(dist - x[r].x) : g == eos_seg ? bin_of(dist) : (unsigned)kBins);
                }
            });
        }
    };
    auto list_segment = [&](unsigned i) {
        const unsigned at = atomicAdd(&s.count, 1u);
        s.key[at] = of_segment(i);
        s.idx[at] = i;
    };
    bool listed = n_all <= kFew;
    if (listed)
    {
        for (unsigned i = t; i < n_all; i += kPickThreads) list_segment(i);
        __syncthreads();
    }
    else
    {
        over_bins([&](unsigned i, unsigned bin) {
            if (bin < kBins) atomicAdd(&s.hist[bin], 1u);
            if (stored) s.bins[i] = (unsigned short)bin;
        });
        __syncthreads();
        find_bin(s, k_seg, false);
        const unsigned last = s.bin + 1;
        listed = !s.wide && last < kBins && s.above + s.hist[s.bin] + s.hist[last] <= kList;
        if (listed)
        {
            if (stored)
            {
#pragma unroll 4
                for (unsigned i = t; i < n_all; i += kPickThreads)
                    if (s.bins[i] <= last) list_segment(i);
            }
            else
                over_bins([&](unsigned i, unsigned bin) {
                    if (bin <= last) list_segment(i);
                });
            __syncthreads();
        }
    }
    if (!listed) pick(s, n_all, k_seg, of_segment, [](unsigned i) { return i; });
    rank_list(s, k_seg);
    if (t < k_seg)
    {
        const unsigned g = s.idx[s.order[t]], w = a.by_n_seg.div(g);
        s.seg_beam[t] = w;
        s.seg_token[t] = (g - w * a.n_seg) * a.seg;
    }
    // The k_seg segments' best are as many candidates from this total on. Those of -inf are left out, unless the
    // others do not suffice.
    const u64 above = key_of(-__builtin_inf()) + 1, kth = s.key[s.order[k_seg - 1]];
    const u64 least = n_all >= a.take && kth > above ? kth : above;
    const float reach = (float)(hi - value_of(least));
    __syncthreads();
    if (t == 0) s.count = 0;
    __syncthreads();

    // The best candidates of theirs. Places past the vocabulary have key 0, behind every candidate's.
    auto place = [&](unsigned i, unsigned& w, unsigned& v) {
        const unsigned q = i >> a.log2_seg;
        w = s.seg_beam[q];
        v = s.seg_token[q] + (i & (a.seg - 1));
    };
    auto logit = [&](unsigned w, unsigned v) {
        const size_t n = b0 + w, at = min(v, a.vocab - 1);
        return a.logits[a.beam_major ? n * a.ld + at : at * a.ld + n];
    };
    auto of_token = [&](unsigned w, unsigned v, float x) { return v < a.vocab ? key_of(total(w, v == a.eos, x)) : 0; };
    const unsigned n_tok = k_seg * a.seg;
#pragma unroll 1
    for (unsigned i = t; i < n_tok; i += 4 * kPickThreads)
    {
        float x[4];
        unsigned w[4], v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            place(min(i + r * kPickThreads, n_tok - 1), w[r], v[r]);
            x[r] = logit(w[r], v[r]);
        }
#pragma unroll 1
        for (int r = 0; r < 4; ++r)
        {
            const float xr = r == 0 ? x[0] : r == 1 ? x[1] : r == 2 ? x[2] : x[3];
            const unsigned wr = r == 0 ? w[0] : r == 1 ? w[1] : r == 2 ? w[2] : w[3];
            const unsigned vr = r == 0 ? v[0] : r == 1 ? v[1] : r == 2 ? v[2] : v[3];
            if (i + r * kPickThreads >= n_tok) break;
            // The distances are off by less than 2^-20 of their terms.
            const float d = near[wr];
            if (!s.ended[wr] && d - xr > reach + 0x1p-20f * (fabsf(d) + fabsf(xr) + fabsf(reach))) continue;
            const u64 key = of_token(wr, vr, xr);
            if (key < least) continue;
            const unsigned at = atomicAdd(&s.count, 1u);
            if (at >= kList) continue;
            s.key[at] = key;
            s.idx[at] = wr * a.vocab + vr;
        }
    }
    __syncthreads();
    if (s.count > kList || s.count < a.take)
        pick(
            s, n_tok, a.take,
            [&](unsigned i) {
                unsigned w, v;
                place(i, w, v);
                return of_token(w, v, logit(w, v));
            },
            [&](unsigned i) {
                unsigned w, v;
                place(i, w, v);
                return v < a.vocab ? w * a.vocab + v : a.beams * a.vocab + i;
            });
    rank_list(s, a.take);
    if (t < a.take)
    {
        const unsigned i = s.order[t], idx = s.idx[i];
        const size_t o = (size_t)blockIdx.x * a.take + t;
        a.out_score[o] = (float)value_of(s.key[i]);
        a.out_beam[o] = (float)(b0 + idx / a.vocab);
        a.out_token[o] = (float)(idx % a.vocab);
    }
}

// Tokens of a segment: as few as the loads take at once, unless the group's segments then take the selection, which
// is one workgroup a group, longer than reading the best ones again.
unsigned segment_of(bool beam_major, size_t beams, size_t vocab)
{
    unsigned seg = beam_major ? kSegRow : kSegColumn;
    while (seg < kSegMost && beams * ((vocab + seg - 1) / seg) > kSegments) seg *= 2;
    return seg;
}

bool beam_sizes_ok(size_t groups, size_t beams, size_t vocab, size_t take)
{
    return groups > 0 && beams > 0 && beams <= kMaxBeams && vocab > 0 && vocab <= kMaxIndex &&
           groups <= kMaxIndex && groups * beams <= kMaxIndex && beams * vocab < (size_t)0x80000000u - (1u << 20) &&
           take > 0 && take <= kMaxTake && take <= beams * vocab;
}

} // namespace
} // namespace nnhip

using namespace nnhip;

extern "C" size_t nnhip_beam_select_workspace_bytes(size_t groups, size_t beams, size_t vocab, size_t take)
{
    if (!beam_sizes_ok(groups, beams, vocab, take)) return 0;
    return groups * beams * ((vocab + kSegColumn - 1) / kSegColumn) * sizeof(float2);
}

extern "C" int nnhip_beam_select(const float* logits, size_t ld, int beam_major, const float* scores,
                                 const float* done, size_t groups, size_t beams, size_t vocab, size_t take, size_t eos,
                                 float* out_score, float* out_beam, float* out_token, void* workspace,
                                 size_t workspace_bytes, void* stream)
{
    if (groups == 0) return 0;
    if (!beam_sizes_ok(groups, beams, vocab, take) || !logits || !scores || !out_score || !out_beam || !out_token ||
        ld < (beam_major ? vocab : groups * beams) || (done && eos >= vocab) || !workspace ||
        workspace_bytes < nnhip_beam_select_workspace_bytes(groups, beams, vocab, take) ||
        reinterpret_cast<uintptr_t>(workspace) % sizeof(float2) != 0)
        return -1;
    if (groups * beams == 1 && !beam_major && ld == 1)   // one column without gaps is a row
    {
        beam_major = 1;
        ld = vocab;
    }
    const unsigned seg = segment_of(beam_major != 0, beams, vocab);
    const unsigned n_seg = static_cast<unsigned>((vocab + seg - 1) / seg), all = static_cast<unsigned>(groups * beams);
    BeamArgs a{logits, scores, done, ld, static_cast<unsigned>(groups), static_cast<unsigned>(beams),
               static_cast<unsigned>(vocab), static_cast<unsigned>(take), static_cast<unsigned>(done ? eos : 0), n_seg, seg,
               static_cast<unsigned>(__builtin_ctz(seg)), FastDiv(n_seg), beam_major, static_cast<float2*>(workspace), out_score, out_beam, out_token};
    auto s = static_cast<hipStream_t>(stream);
    const size_t segments = (size_t)all * n_seg;
    if (segments + 16 > 0x7fffffffu) return -1;
    if (beam_major)
        hipLaunchKernelGGL(k_beam_segments_row, dim3(static_cast<unsigned>((segments + 15) / 16)), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(k_beam_segments_column, dim3(static_cast<unsigned>((segments + 255) / 256)), dim3(256), 0, s, a);
    if (int rc = launch_status()) return rc;
    hipLaunchKernelGGL(k_beam_pick, dim3(all / a.beams), dim3(kPickThreads), 0, s, a);
    return launch_status();
}
