// k_verify.hip — verification of drafted tokens (speculative sampling: Leviathan,
// Kalman and Matias, "Fast Inference from Transformers via Speculative
// Decoding", ICML 2023).
//
// Three launches. The first leaves, for every row of logits and segment of the
// vocabulary, the largest logit and the sum of exp((logit - largest) /
// temperature). From these the second decides for every sequence which row is
// the first whose token does not stand, and leaves that row's sums of
// max(p - q, 0) by segment. The third finds the segment that the random number
// falls into, and the token within it. Sums, probabilities and comparisons are
// in float64, of exponentials good to 2^-37: float32's would move the border
// between two tokens by 2^-24 of the whole, far more than most tokens'
// probability.
//
// The first launch is bound by its exponentials (144 rows of 100003 of either
// model: 32 us, 3.5 TB/s; 144 of 32000 by columns 17), the others by latency:
// a sequence's decision, a scan of its row's sums and a search by one
// workgroup, 9 to 17 us each.
#include "kv_pages.hpp"

namespace nnhip
{
namespace
{

constexpr int kThreads = 256;
constexpr unsigned kMostSegments = 1024;
constexpr size_t kMostRows = 1024;   // of a sequence

// The decision on a sequence: the row whose distribution the next token is from, -1 without rows; whether it is a drafted
// token's; the largest logits and the sums of both models' row.
struct Decision
{
    int row, accepted, drafted, token;
    float mt, md;
    double pt, pd;   // 1 / the sums, 0 where these are
};

struct VerifyArgs
{
    const float *target, *draft, *fed, *start, *accept, *pick;
    size_t t_row, t_col, d_row, d_col;   // floats from a row's logits to the next row's, and from one logit to the next
    unsigned vocab, tokens, batch, most, seg, n_seg, left_seg, n_left;   // tokens of a segment, segments: of the sums, of what is left
    int log2_cols;                       // logits by columns: 2^log2_cols of them to a workgroup
    FastDiv by_seg, by_left;
    double scale;                        // 32 / (temperature ln 2); 0: the largest logit
    float* part_m;                       // per (model, row, segment): largest logit; and sum, or the largest one's index
    double* part_s;
    Decision* decision;                  // per sequence
    double* left;                        // per (sequence, piece): sum of max(p - q, 0)
    float *out_accepted, *out_token;
};

// 2^(i / 32), by the exponential's series.
struct Powers
{
    double p[32];
    constexpr Powers() : p{}
    {
        for (int i = 0; i < 32; ++i)
        {
            const double x = i * 0.6931471805599453 / 32;
            double term = 1.0, sum = 0.0;
            for (int k = 1; k < 30; ++k)
            {
                sum += term;
                term *= x / k;
            }
            p[i] = sum;
        }
    }
};
__constant__ const Powers kPowers;

// exp((z - m) / temperature) for m >= z; NaN counts as -inf, and +inf beside +inf as equal. With x = (z - m) / temperature
// in units of ln 2 / 32 and n the nearest whole number this is 2^(n / 32), from a table, times exp of (x - n) ln 2 / 32,
// which is below 0.011: 1 + r + r^2 (1/2 + r/6 + r^2/24), the last in float32. Off by 2^-37 at most. No branch, so that a
// thread's values go side by side. 144 rows of 100003 twice, first launch: 40 us with the series to r^13 in float64, 33 so;
// the library's exp, one value after another, took 54.
using Table = double[32];
__device__ __forceinline__ double term(const VerifyArgs& a, const Table& powers, float z, float m)
{
    constexpr double kUnit = 0.6931471805599453 / 32;
    const double d = z == m ? 0.0 : (double)z - (double)m;
    const double x = z > -__builtin_inff() ? fmax(d * a.scale, -36932.0) : -36932.0;   // exp(-800), as every number below -746: 0
    const double n = rint(x), left = x - n;
    const int i = (int)n;
    const float r = (float)left * (float)kUnit;
    const float square = r * r * __builtin_fmaf(r, __builtin_fmaf(r, 1.0f / 24, 1.0f / 6), 0.5f);
    const double p = powers[i & 31];
    return __builtin_ldexp(__builtin_fma(p, __builtin_fma(left, kUnit, (double)square), p), i >> 5);
}
__device__ __forceinline__ void load_powers(Table& powers)   // a barrier follows
{
    if (threadIdx.x < 32) powers[threadIdx.x] = kPowers.p[threadIdx.x];
}
__device__ __forceinline__ float larger(float m, float z) { return z > m ? z : m; }   // of NaN and m, m

struct Sum
{
    float m;
    double s;   // or the index of m
};

// What f makes of the values of all threads that have the thread's column: lanes at distances of 2^log2_cols, then waves.
template <int NT, class T, class F> __device__ __forceinline__ T of_column(const VerifyArgs& a, T x, T (&wave_s)[NT / 2], F&& f)
{
    const int t = threadIdx.x, cols = 1 << a.log2_cols, col = t & (cols - 1);
    for (int o = 32; o >= cols; o >>= 1) x = f(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if ((t & 63) < cols) wave_s[(t >> 6) * cols + col] = x;
    __syncthreads();
    x = wave_s[col];
    for (int w = 1; w < NT / 64; ++w) x = f(x, wave_s[w * cols + col]);
    return x;
}

// One segment of a row (logits by rows) or of up to 32 rows' columns; a thread takes PER logits of a row at once, on their
// way together. blockIdx.y: the target's, the draft's.
template <bool GREEDY, int PER, int NT> __global__ __launch_bounds__(NT) void k_verify_sums(VerifyArgs a)
{
    __shared__ float m_s[NT / 2];
    __shared__ double s_s[NT / 2];
    __shared__ Table powers;
    load_powers(powers);   // of_column has barriers
    const int t = threadIdx.x;
    const unsigned outer = a.by_seg.div(blockIdx.x), seg = blockIdx.x - outer * a.n_seg;
    const unsigned cols = 1u << a.log2_cols, parts = NT >> a.log2_cols;
    const unsigned part = t >> a.log2_cols, n = outer * cols + (t & (cols - 1));
    const float* p = blockIdx.y ? a.draft : a.target;
    const size_t row = blockIdx.y ? a.d_row : a.t_row, col = blockIdx.y ? a.d_col : a.t_col;
    const unsigned v0 = seg * a.seg, end = min(v0 + a.seg, a.vocab);
    const float* x = p + (size_t)min(n, a.tokens - 1) * row;
    Sum r{-__builtin_inff(), GREEDY ? (double)v0 : 0.0};
    for (unsigned v = v0; v < end; v += PER * parts)
    {
        float z[PER], m = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < PER; ++k) z[k] = x[(size_t)min(v + part + k * parts, end - 1) * col];
#pragma unroll
        for (int k = 0; k < PER; ++k) z[k] = v + part + k * parts < end ? z[k] : -__builtin_inff();
#pragma unroll
        for (int k = 0; k < PER; ++k) m = larger(m, z[k]);
        m = larger(r.m, of_column<NT>(a, m, m_s, larger));
        if constexpr (GREEDY)
        {
            double at = a.vocab;
#pragma unroll
            for (int k = PER - 1; k >= 0; --k)
                if (z[k] == m) at = v + part + k * parts;
            at = of_column<NT>(a, at, s_s, [](double u, double w) { return fmin(u, w); });
            if (m > r.m) r.s = at;
        }
        else
        {
            double s = 0.0;
#pragma unroll
            for (int k = 0; k < PER; ++k) s += term(a, powers, z[k], m);
            if (v != v0) s += r.s * term(a, powers, r.m, m);
            r.s = s;
        }
        r.m = m;
    }
    if constexpr (!GREEDY) r.s = of_column<NT>(a, r.s, s_s, [](double u, double w) { return u + w; });
    if (part == 0 && n < a.tokens)
    {
        const size_t at = ((size_t)blockIdx.y * a.tokens + n) * a.n_seg + seg;
        a.part_m[at] = r.m;
        a.part_s[at] = r.s;
    }
}

__device__ __forceinline__ double wave_sum64(double v)
{
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// The drafted token behind row n, -1 where it is none.
__device__ __forceinline__ int drafted(const VerifyArgs& a, unsigned n)
{
    size_t x;
    return row_index(a.fed[n + 1], a.vocab, x) ? (int)x : -1;
}

constexpr int kRowsAtOnce = kThreads / 32;   // rows that a workgroup decides on together: 16 lanes a model's row
struct DecideShared
{
    float m[2 * kRowsAtOnce];
    double s[2 * kRowsAtOnce];   // or the index of m
    int x[kRowsAtOnce];          // the drafted tokens behind the rows
    int first;
};
// A workgroup: what becomes of sequence b.
template <bool GREEDY> __device__ __forceinline__ Decision decide(const VerifyArgs& a, const Table& powers, unsigned b, DecideShared& sh)
{
    const int t = threadIdx.x, group = t >> 4, lane = t & 15, model = group & 1;
    const int lo = length_of(a.start[b], a.tokens), hi = length_of(a.start[b + 1], a.tokens), n = min(hi - lo, (int)a.most);
    Decision d{};
    d.row = -1;
    d.token = -1;
    d.mt = d.md = -__builtin_inff();
    for (int i0 = 0; i0 < n; i0 += kRowsAtOnce)
    {
        // A row a lane: its drafted token and what belongs to that, on their way while the sums are joined.
        const bool there = t < kRowsAtOnce && i0 + t < n, has_token = there && i0 + t < n - 1;
        int x = -1;
        float accept = 0.0f, zt = 0.0f, zd = 0.0f;
        if (has_token)
        {
            const size_t row = lo + i0 + t;
            x = drafted(a, row);
            if (!GREEDY && x >= 0)
            {
                accept = a.accept[row];
                zt = a.target[row * a.t_row + (size_t)x * a.t_col];
                if (a.draft) zd = a.draft[row * a.d_row + (size_t)x * a.d_col];
            }
        }
        const int i = i0 + (group >> 1);
        if (i < n && (model == 0 || (a.draft && i < n - 1)))
        {
            // The row's segments together.
            const size_t at = ((size_t)model * a.tokens + lo + i) * a.n_seg;
            float m = -__builtin_inff();
            for (unsigned k = lane; k < a.n_seg; k += 16) m = larger(m, a.part_m[at + k]);
            for (int o = 8; o > 0; o >>= 1) m = larger(m, __shfl_xor(m, o, 16));
            double s = GREEDY ? (double)a.vocab : 0.0;
            for (unsigned k = lane; k < a.n_seg; k += 16)
            {
                const float mk = a.part_m[at + k];
                const double sk = a.part_s[at + k];
                if constexpr (GREEDY) s = mk == m ? fmin(s, sk) : s;
                else s += sk * term(a, powers, mk, m);
            }
            for (int o = 8; o > 0; o >>= 1)
            {
                const double y = __shfl_xor(s, o, 16);
                s = GREEDY ? fmin(s, y) : s + y;
            }
            if (lane == 0)
            {
                sh.m[group] = m;
                sh.s[group] = s;
            }
        }
        if (t == 0) sh.first = n;
        __syncthreads();
        if (t < 64)
        {
            bool stands = false;
            if (has_token)
            {
                if constexpr (GREEDY) stands = (int)sh.s[2 * t] == x;
                else if (x >= 0)   // no token stands with 0 of p, as one that is none
                {
                    auto p_of = [&](float z, int k) { return sh.s[k] == 0.0 ? 0.0 : term(a, powers, z, sh.m[k]) * (1.0 / sh.s[k]); };
                    const double px = p_of(zt, 2 * t), qx = a.draft ? p_of(zd, 2 * t + 1) : 1.0;
                    stands = (double)accept * qx < px;
                }
            }
            if (there) sh.x[t] = x;
            const unsigned long long ends = __builtin_amdgcn_ballot_w64(there && !stands);
            if (t == 0 && ends) sh.first = i0 + __builtin_ctzll(ends);
        }
        __syncthreads();
        const int f = sh.first, k = 2 * (f - i0);
        if (f < n)   // the last row ends the search if none does before
        {
            d.row = lo + f;
            d.accepted = f;
            d.drafted = f < n - 1;
            if constexpr (GREEDY) d.token = (int)sh.s[k];
            else
            {
                d.token = sh.x[f - i0];
                d.mt = sh.m[k];
                d.pt = sh.s[k] == 0.0 ? 0.0 : 1.0 / sh.s[k];
                if (d.drafted && a.draft)
                {
                    d.md = sh.m[k + 1];
                    d.pd = sh.s[k + 1] == 0.0 ? 0.0 : 1.0 / sh.s[k + 1];
                }
            }
            break;
        }
        __syncthreads();
    }
    return d;
}

// max(p - q, 0) of logit v of the decision's row.
__device__ __forceinline__ double left_of(const VerifyArgs& a, const Table& powers, const Decision& d, unsigned v)
{
#pragma clang fp contract(off)   // p = q has to leave 0
    const double p = term(a, powers, a.target[(size_t)d.row * a.t_row + (size_t)v * a.t_col], d.mt) * d.pt;
    double q = (int)v == d.token ? 1.0 : 0.0;
    if (a.draft) q = term(a, powers, a.draft[(size_t)d.row * a.d_row + (size_t)v * a.d_col], d.md) * d.pd;
    return fmax(p - q, 0.0);
}

// Sums of what is left of p over kLeft tokens, blockIdx.x = sequence * n_left + piece. A call of 24 sequences of up to 5 drafted
// tokens of 32000 with pieces of 2048 tokens 45 us, of 1024 41, of 512 48; of one sequence 23.5, 21, 20.
constexpr unsigned kLeft = 4 * kThreads;
constexpr int kEach = 8;                       // neighbouring tokens of a thread that looks for one
constexpr unsigned kWhole = kEach * kThreads;   // a vocabulary of which that thread's workgroup holds all
__global__ __launch_bounds__(kThreads) void k_verify_left(VerifyArgs a)
{
    __shared__ DecideShared sh;
    __shared__ double s_s[kThreads / 64];
    __shared__ Table powers;
    const int t = threadIdx.x;
    load_powers(powers);
    __syncthreads();
    const unsigned b = a.by_left.div(blockIdx.x), piece = blockIdx.x - b * a.n_left;
    const Decision d = decide<false>(a, powers, b, sh);
    if (piece == 0 && t == 0) a.decision[b] = d;
    if (!d.drafted) return;
    const unsigned v0 = piece * a.left_seg, end = min(v0 + a.left_seg, a.vocab);
    double s = 0.0;
    for (unsigned v = v0 + t; v < end; v += kLeft)
    {
        double x[kLeft / kThreads];
#pragma unroll
        for (unsigned i = 0; i < kLeft / kThreads; ++i) x[i] = left_of(a, powers, d, min(v + i * kThreads, end - 1));
#pragma unroll
        for (unsigned i = 0; i < kLeft / kThreads; ++i) s += v + i * kThreads < end ? x[i] : 0.0;
    }
    s = wave_sum64(s);
    if ((t & 63) == 0) s_s[t >> 6] = s;
    __syncthreads();
    if (t == 0) a.left[(size_t)b * a.n_left + piece] = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
}

// Sums of all threads' values up to and with the thread's own.
__device__ __forceinline__ double scan(double x, double (&wave_s)[kThreads / 64], double& all)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    for (int o = 1; o < 64; o *= 2)
    {
        const double y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) wave_s[wave] = x;
    __syncthreads();
    double before = 0.0;
    all = 0.0;
    for (int w = 0; w < kThreads / 64; ++w)
    {
        if (w < wave) before += wave_s[w];
        all += wave_s[w];
    }
    return before + x;
}

// The smallest of all threads' `first`, the largest of their `last`.
struct Found
{
    unsigned first, last;
};
__device__ __forceinline__ Found found(unsigned first, unsigned last, unsigned (&first_w)[kThreads / 64], unsigned (&last_w)[kThreads / 64])
{
    for (int o = 32; o > 0; o >>= 1)
    {
        first = min(first, (unsigned)__shfl_xor((int)first, o, 64));
        last = max(last, (unsigned)__shfl_xor((int)last, o, 64));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
    {
        first_w[threadIdx.x >> 6] = first;
        last_w[threadIdx.x >> 6] = last;
    }
    __syncthreads();
    return {min(min(first_w[0], first_w[1]), min(first_w[2], first_w[3])), max(max(last_w[0], last_w[1]), max(last_w[2], last_w[3]))};
}

// The next token of sequence blockIdx.x. DECIDE: without the second launch, which has nothing to do for single rows, and for
// a vocabulary of kWhole no more than this one does on its way: its threads hold all of it, so that it is read once
// (4 drafted tokens of 1024: 22 us a call with three launches, 15 with two that read it twice, 13 so).
template <bool GREEDY, bool DECIDE> __global__ __launch_bounds__(kThreads) void k_verify_pick(VerifyArgs a)
{
    __shared__ DecideShared sh;
    __shared__ double wave_s[kThreads / 64], before_s;
    __shared__ unsigned first_w[kThreads / 64], last_w[kThreads / 64];
    __shared__ Table powers;
    const int t = threadIdx.x;
    if constexpr (!GREEDY)
    {
        load_powers(powers);
        __syncthreads();
    }
    const unsigned b = blockIdx.x;
    const Decision d = DECIDE ? decide<GREEDY>(a, powers, b, sh) : a.decision[b];
    if (t == 0) a.out_accepted[b] = (float)d.accepted;
    if (GREEDY || d.row < 0)
    {
        if (t == 0) a.out_token[b] = (float)d.token;
        return;
    }
    const size_t at = (size_t)d.row * a.n_seg;
    bool left = d.drafted;   // whether p is lessened by q
    // The weights of tokens from v on, and their sum.
    auto weights = [&](unsigned v, unsigned end, double (&x)[kEach]) -> double {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
        {
            const unsigned at = min(v + i, end - 1);
            x[i] = left ? left_of(a, powers, d, at) : term(a, powers, a.target[(size_t)d.row * a.t_row + (size_t)at * a.t_col], d.mt);
            if (v + i >= end) x[i] = 0.0;
            sum += x[i];
        }
        return sum;
    };
    // Of these the first whose cumulative sum, of `up` before the first, is above `want`, and the last with anything.
    auto search = [&](unsigned v, const double (&x)[kEach], double up, double want) -> Found {
        unsigned first = a.vocab, last = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
        {
            up += x[i];
            if (x[i] > 0.0)
            {
                last = v + i;
                if (up > want) first = min(first, v + i);
            }
        }
        return found(first, last, first_w, last_w);
    };
    const float w = a.pick[b];
    const double share = w >= 1.0f ? 1.0 - 0x1p-53 : w > 0.0f ? (double)w : 0.0;
    if (DECIDE && a.vocab <= kWhole)
    {
        double x[kEach], mine = weights(kEach * t, a.vocab, x), all, up = scan(mine, wave_s, all);
        if (left && !(all > 0.0))
        {
            left = false;
            mine = weights(kEach * t, a.vocab, x);
            up = scan(mine, wave_s, all);
        }
        const Found in = search(kEach * t, x, up - mine, share * all);
        if (t == 0) a.out_token[b] = (float)(in.first < a.vocab ? in.first : in.last);
        return;
    }
    auto of_segment = [&](unsigned i) -> double {
        if (i >= (left ? a.n_left : a.n_seg)) return 0.0;
        return left ? a.left[(size_t)b * a.n_left + i] : a.part_s[at + i] * term(a, powers, a.part_m[at + i], d.mt);
    };
    double whole = 0.0, own = 0.0, own_up = 0.0;
    for (int again = 0; again < 2; ++again)
    {
        whole = 0.0;
        for (unsigned i = 0; i < (left ? a.n_left : a.n_seg); i += kThreads)
        {
            double all;
            own = of_segment(i + t);
            own_up = scan(own, wave_s, all);
            whole += all;
        }
        if (whole > 0.0 || !left) break;
        left = false;
    }
    const double want = share * whole;
    // The first segment whose cumulative sum is above that, the last one with anything where rounding leaves none.
    const unsigned segs = left ? a.n_left : a.n_seg, size = left ? a.left_seg : a.seg;
    Found in{segs, 0};
    double sum = 0.0, base = 0.0;
    for (unsigned i = 0; i < segs && in.first == segs; i += kThreads)
    {
        double all = 0.0;
        const bool once = segs <= kThreads;   // all of them are in the threads already
        const double x = once ? own : of_segment(i + t), up = sum + (once ? own_up : scan(x, wave_s, all));
        const Found here = found(x > 0.0 && up > want ? i + t : segs, x > 0.0 ? i + t : 0, first_w, last_w);
        in.first = min(in.first, here.first);
        in.last = max(in.last, here.last);
        if (in.first == i + t) before_s = up - x;
        __syncthreads();
        base = before_s;
        sum += all;
    }
    const bool some = in.first < segs;
    const unsigned seg = some ? in.first : in.last;
    // The token, alike.
    const unsigned end = min((seg + 1) * size, a.vocab);
    in = {a.vocab, 0};
    sum = some ? base : -__builtin_inf();
    for (unsigned v0 = seg * size; v0 < end && in.first == a.vocab; v0 += kThreads * kEach)
    {
        double x[kEach], all;
        const double mine = weights(v0 + kEach * t, end, x);
        const Found here = search(v0 + kEach * t, x, sum + (scan(mine, wave_s, all) - mine), want);
        in.first = min(in.first, here.first);
        in.last = max(in.last, here.last);
        sum += all;
    }
    if (t == 0) a.out_token[b] = (float)(in.first < a.vocab ? in.first : in.last);
}

struct VerifyPlan
{
    unsigned seg, n_seg, left_seg, n_left;
    int log2_cols, per, threads;   // the first launch: columns and threads of a workgroup, logits that a thread takes at once
};
VerifyPlan verify_plan(size_t tokens, size_t vocab, bool token_major)
{
    VerifyPlan p{};
    if (!token_major)
        while (p.log2_cols < 5 && ((size_t)1 << p.log2_cols) < tokens) ++p.log2_cols;
    // 16 logits a thread, for their way together and for fewer segments, or 4 where 16 leave CUs without work. A call with 4 and
    // with 16, by columns: 5 rows of 1024 20 and 22 us, 4 rows of 50257 (no draft) 15 and 19, 5 of 50257 both 26, 40 of 50257 44 and
    // 31; by rows: 20 of 32000 22 both, 144 of 100003 82 and 62.
    p.per = tokens * vocab < ((size_t)1 << 19) ? 4 : 16;
    // Of several columns more threads, for as few segments: every sequence reads its rows' twice more.
    p.threads = p.log2_cols >= 2 ? 1024 : kThreads;
    size_t seg = (size_t)(p.threads >> p.log2_cols) * p.per;
    while ((vocab + seg - 1) / seg > kMostSegments) seg *= 2;
    p.seg = static_cast<unsigned>(seg);
    p.n_seg = static_cast<unsigned>((vocab + seg - 1) / seg);
    size_t left = kLeft;
    while ((vocab + left - 1) / left > kMostSegments) left *= 2;
    p.left_seg = static_cast<unsigned>(left);
    p.n_left = static_cast<unsigned>((vocab + left - 1) / left);
    return p;
}

struct VerifySpace
{
    size_t part_s, part_m, decision, left, all;   // bytes
};
VerifySpace verify_space(size_t tokens, size_t batch, const VerifyPlan& p)
{
    VerifySpace s{};
    s.part_m = 2 * tokens * p.n_seg * sizeof(double);
    s.decision = (s.part_m + 2 * tokens * p.n_seg * sizeof(float) + 15) / 16 * 16;
    s.left = s.decision + batch * sizeof(Decision);
    s.all = s.left + batch * p.n_left * sizeof(double);
    return s;
}
static_assert(sizeof(Decision) % 8 == 0);

bool verify_ok(size_t tokens, size_t batch, size_t most, size_t vocab)
{
    return tokens > 0 && tokens <= kMaxIndex && batch > 0 && batch <= kMaxIndex && vocab > 0 && vocab <= kMaxIndex && most > 0 &&
           most <= kMostRows;
}

} // namespace
} // namespace nnhip

using namespace nnhip;

extern "C" size_t nnhip_draft_verify_workspace_bytes(size_t tokens, size_t batch, size_t most, size_t vocab)
{
    if (!verify_ok(tokens, batch, most, vocab)) return 0;
    const size_t rows = verify_space(tokens, batch, verify_plan(tokens, vocab, true)).all;   // enough for either layout
    const size_t columns = verify_space(tokens, batch, verify_plan(tokens, vocab, false)).all;
    return rows > columns ? rows : columns;
}

extern "C" int nnhip_draft_verify(const float* target, size_t t_ld, const float* draft, size_t d_ld, int token_major,
                                  size_t vocab, size_t tokens, const float* fed, const float* start, size_t batch,
                                  size_t most, float temperature, const float* accept, const float* pick,
                                  float* out_accepted, float* out_token, void* workspace, size_t workspace_bytes,
                                  void* stream)
{
    if (batch == 0) return 0;
    const size_t least_ld = token_major ? vocab : tokens;
    if (!verify_ok(tokens, batch, most, vocab) || !target || !fed || !start || !out_accepted || !out_token || t_ld < least_ld ||
        t_ld > ((size_t)1 << 32) || (draft && (d_ld < least_ld || d_ld > ((size_t)1 << 32))) || !(temperature >= 0.0f) ||
        temperature > kMaxF || (temperature > 0.0f && (!accept || !pick)))
        return -1;
    const VerifyPlan plan = verify_plan(tokens, vocab, token_major != 0);
    const VerifySpace space = verify_space(tokens, batch, plan);
    if (!workspace || workspace_bytes < space.all || !aligned16(workspace)) return -1;
    const bool greedy = temperature == 0.0f;
    VerifyArgs a{};
    a.target = target;
    a.draft = greedy || most == 1 ? nullptr : draft;
    a.fed = fed;
    a.start = start;
    a.accept = accept;
    a.pick = pick;
    a.t_row = token_major ? t_ld : 1;
    a.t_col = token_major ? 1 : t_ld;
    a.d_row = token_major ? d_ld : 1;
    a.d_col = token_major ? 1 : d_ld;
    a.vocab = static_cast<unsigned>(vocab);
    a.tokens = static_cast<unsigned>(tokens);
    a.batch = static_cast<unsigned>(batch);
    a.most = static_cast<unsigned>(most);
    a.seg = plan.seg;
    a.n_seg = plan.n_seg;
    a.left_seg = plan.left_seg;
    a.n_left = plan.n_left;
    a.by_seg = FastDiv(plan.n_seg);
    a.by_left = FastDiv(plan.n_left);
    a.log2_cols = plan.log2_cols;
    a.scale = greedy ? 0.0 : 32.0 / (static_cast<double>(temperature) * 0.6931471805599453);
    auto* ws = static_cast<char*>(workspace);
    a.part_s = reinterpret_cast<double*>(ws);
    a.part_m = reinterpret_cast<float*>(ws + space.part_m);
    a.decision = reinterpret_cast<Decision*>(ws + space.decision);
    a.left = reinterpret_cast<double*>(ws + space.left);
    a.out_accepted = out_accepted;
    a.out_token = out_token;
    const size_t cols = (size_t)1 << a.log2_cols, blocks = (tokens + cols - 1) / cols * plan.n_seg;
    if (blocks * plan.threads / kThreads > kGridMost || batch * plan.n_left > kGridMost) return -1;
    auto s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(blocks), a.draft ? 2 : 1);
    const dim3 all(static_cast<unsigned>(batch));
    auto sums = [&](auto few, auto many, auto few_cols, auto many_cols) {
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(static_cast<unsigned>(plan.threads)), 0, s, a); };
        if (plan.threads == kThreads) plan.per == 4 ? go(few) : go(many);
        else plan.per == 4 ? go(few_cols) : go(many_cols);
    };
    if (greedy)
    {
        sums(k_verify_sums<true, 4, kThreads>, k_verify_sums<true, 16, kThreads>, k_verify_sums<true, 4, 1024>, k_verify_sums<true, 16, 1024>);
        if (int rc = launch_status()) return rc;
        hipLaunchKernelGGL((k_verify_pick<true, true>), all, dim3(kThreads), 0, s, a);
        return launch_status();
    }
    sums(k_verify_sums<false, 4, kThreads>, k_verify_sums<false, 16, kThreads>, k_verify_sums<false, 4, 1024>, k_verify_sums<false, 16, 1024>);
    if (int rc = launch_status()) return rc;
    if (most == 1 || vocab <= kWhole)
    {
        hipLaunchKernelGGL((k_verify_pick<false, true>), all, dim3(kThreads), 0, s, a);
        return launch_status();
    }
    hipLaunchKernelGGL(k_verify_left, dim3(static_cast<unsigned>(batch * plan.n_left)), dim3(kThreads), 0, s, a);
    if (int rc = launch_status()) return rc;
    hipLaunchKernelGGL((k_verify_pick<false, false>), all, dim3(kThreads), 0, s, a);
    return launch_status();
}
