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
// in float64: float32's would move the border between two tokens by 2^-24 of
// the whole, far more than most tokens' probability.
#include "kv_pages.hpp"

namespace nnhip
{
namespace
{

constexpr int kThreads = 256;
constexpr int kAtOnce = 16;          // logits that a thread holds
constexpr unsigned kMostSegments = 1024;
constexpr size_t kMostRows = 1024;   // of a sequence

// The decision on a sequence: the row whose distribution the next token is from, -1 without rows; whether it is a drafted
// token's; the largest logits and the sums of both models' row.
struct Decision
{
    int row, accepted, drafted, token;
    float mt, md;
    double st, sd;
};

struct VerifyArgs
{
    const float *target, *draft, *fed, *start, *accept, *pick;
    size_t t_row, t_col, d_row, d_col;   // floats from a row's logits to the next row's, and from one logit to the next
    unsigned vocab, tokens, batch, most, seg, n_seg;
    int log2_cols, rows_along;           // logits by columns: 2^log2_cols of them to a workgroup
    FastDiv by_seg;
    double inv;                          // 1 / temperature; 0: the largest logit
    float* part_m;                       // per (model, row, segment): largest logit; and sum, or the largest one's index
    double* part_s;
    Decision* decision;                  // per sequence
    double* left;                        // per (sequence, segment): sum of max(p - q, 0)
    float *out_accepted, *out_token;
};

// exp((z - m) / temperature) for m >= z; NaN counts as -inf, and +inf beside +inf as equal.
__device__ __forceinline__ double term(const VerifyArgs& a, float z, float m)
{
    if (!(z > -__builtin_inff())) return 0.0;
    return z == m ? 1.0 : exp(((double)z - (double)m) * a.inv);
}
__device__ __forceinline__ float larger(float m, float z) { return z > m ? z : m; }   // of NaN and m, m

struct Sum
{
    float m;
    double s;   // or the index of m
};
template <bool GREEDY> __device__ __forceinline__ Sum join(const VerifyArgs& a, Sum x, Sum y)
{
    Sum r;
    r.m = larger(x.m, y.m);
    if constexpr (GREEDY) r.s = x.m == y.m ? fmin(x.s, y.s) : x.m > y.m ? x.s : y.s;
    else r.s = x.s * term(a, x.m, r.m) + y.s * term(a, y.m, r.m);
    return r;
}

// What a thread's logits come to: get(k) gives logit k of n and its index.
template <bool GREEDY, class F> __device__ __forceinline__ Sum sum_of(const VerifyArgs& a, unsigned v0, unsigned step, unsigned end, F&& get)
{
    Sum r{-__builtin_inff(), GREEDY ? (double)v0 : 0.0};
    for (unsigned v = v0; v < end; v += kAtOnce * step)
    {
        float z[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) z[k] = v + k * step < end ? get(v + k * step) : -__builtin_inff();
        Sum c{-__builtin_inff(), GREEDY ? (double)v : 0.0};
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
        {
            if (GREEDY && z[k] > c.m) c.s = v + k * step;
            c.m = larger(c.m, z[k]);
        }
        if constexpr (!GREEDY)
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) c.s += term(a, z[k], c.m);
        r = v == v0 ? c : join<GREEDY>(a, r, c);
    }
    return r;
}

// One segment of a row (logits by rows) or of up to 64 rows' columns. blockIdx.y: the target's, the draft's.
template <bool GREEDY> __global__ __launch_bounds__(kThreads) void k_verify_sums(VerifyArgs a)
{
    __shared__ float m_s[kThreads];
    __shared__ double s_s[kThreads];
    const int t = threadIdx.x;
    const unsigned outer = a.by_seg.div(blockIdx.x), seg = blockIdx.x - outer * a.n_seg;
    const unsigned cols = 1u << a.log2_cols, parts = kThreads >> a.log2_cols;
    const unsigned part = t >> a.log2_cols, n = outer * cols + (t & (cols - 1));
    const float* p = blockIdx.y ? a.draft : a.target;
    const size_t row = blockIdx.y ? a.d_row : a.t_row, col = blockIdx.y ? a.d_col : a.t_col;
    const unsigned v0 = seg * a.seg, end = min(v0 + a.seg, a.vocab);
    Sum r{-__builtin_inff(), (double)v0};
    if (n < a.tokens)
    {
        const float* x = p + (size_t)n * row;
        r = sum_of<GREEDY>(a, v0 + part, parts, end, [&](unsigned v) { return x[(size_t)v * col]; });
    }
    m_s[t] = r.m;
    s_s[t] = r.s;
    for (unsigned half = parts / 2; half > 0; half /= 2)
    {
        __syncthreads();
        if (part < half)
        {
            const unsigned o = t + (half << a.log2_cols);
            r = join<GREEDY>(a, r, Sum{m_s[o], s_s[o]});
            m_s[t] = r.m;
            s_s[t] = r.s;
        }
    }
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
// A wave: a row's segments together.
__device__ __forceinline__ Sum row_sum(const VerifyArgs& a, int model, unsigned n)
{
    const unsigned lane = threadIdx.x & 63;
    const size_t at = ((size_t)model * a.tokens + n) * a.n_seg;
    Sum r{-__builtin_inff(), 0.0};
    for (unsigned i = lane; i < a.n_seg; i += 64) r.m = larger(r.m, a.part_m[at + i]);
    r.m = wave_max(r.m);
    for (unsigned i = lane; i < a.n_seg; i += 64) r.s += a.part_s[at + i] * term(a, a.part_m[at + i], r.m);
    r.s = wave_sum64(r.s);
    return r;
}
__device__ __forceinline__ unsigned row_best(const VerifyArgs& a, unsigned n)
{
    const unsigned lane = threadIdx.x & 63;
    const size_t at = (size_t)n * a.n_seg;
    float m = -__builtin_inff();
    for (unsigned i = lane; i < a.n_seg; i += 64) m = larger(m, a.part_m[at + i]);
    m = wave_max(m);
    double best = a.vocab;
    for (unsigned i = lane; i < a.n_seg; i += 64)
        if (a.part_m[at + i] == m) best = fmin(best, a.part_s[at + i]);
    for (int o = 32; o > 0; o >>= 1) best = fmin(best, __shfl_xor(best, o, 64));
    return (unsigned)best;
}

// The drafted token behind row n, -1 where it is none.
__device__ __forceinline__ int drafted(const VerifyArgs& a, unsigned n)
{
    size_t x;
    return row_index(a.fed[n + 1], a.vocab, x) ? (int)x : -1;
}

// A workgroup: what becomes of sequence b. shared: kMostRows places.
template <bool GREEDY> __device__ __forceinline__ Decision decide(const VerifyArgs& a, unsigned b, int& first_s, Decision& d_s)
{
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int lo = length_of(a.start[b], a.tokens), hi = length_of(a.start[b + 1], a.tokens);
    const int n = min(hi - lo, (int)a.most);
    if (t == 0) first_s = n - 1;
    __syncthreads();
    for (int i = wave; i < n - 1; i += kThreads / 64)
    {
        const unsigned row = lo + i;
        const int x = drafted(a, row);
        bool stands;
        if constexpr (GREEDY) stands = (int)row_best(a, row) == x;
        else
        {
            const Sum p = row_sum(a, 0, row);
            const double px = x < 0 || p.s == 0.0 ? 0.0 : term(a, a.target[(size_t)row * a.t_row + (size_t)x * a.t_col], p.m) / p.s;
            double qx = 1.0;
            if (a.draft)
            {
                const Sum q = row_sum(a, 1, row);
                qx = x < 0 || q.s == 0.0 ? 0.0 : term(a, a.draft[(size_t)row * a.d_row + (size_t)x * a.d_col], q.m) / q.s;
            }
            stands = (double)a.accept[row] * qx < px;
        }
        if (!stands)
        {
            if (lane == 0) atomicMin(&first_s, i);   // in LDS: the smallest, in whatever order
            break;
        }
    }
    __syncthreads();
    const int f = first_s;
    if (wave == 0)
    {
        Decision d{};
        d.row = n > 0 ? lo + f : -1;
        d.accepted = n > 0 ? f : 0;
        d.drafted = f < n - 1;
        d.token = d.drafted ? drafted(a, lo + f) : -1;
        d.mt = d.md = -__builtin_inff();
        if (n > 0)
        {
            if constexpr (GREEDY) d.token = (int)row_best(a, lo + f);
            else
            {
                const Sum p = row_sum(a, 0, lo + f);
                d.mt = p.m;
                d.st = p.s;
                if (d.drafted && a.draft)
                {
                    const Sum q = row_sum(a, 1, lo + f);
                    d.md = q.m;
                    d.sd = q.s;
                }
            }
        }
        if (lane == 0) d_s = d;
    }
    __syncthreads();
    return d_s;
}

// max(p - q, 0) of logit v of the decision's row.
__device__ __forceinline__ double left_of(const VerifyArgs& a, const Decision& d, unsigned v)
{
    const double p = d.st == 0.0 ? 0.0 : term(a, a.target[(size_t)d.row * a.t_row + (size_t)v * a.t_col], d.mt) / d.st;
    double q = 0.0;
    if (!a.draft) q = (int)v == d.token ? 1.0 : 0.0;
    else if (d.sd != 0.0) q = term(a, a.draft[(size_t)d.row * a.d_row + (size_t)v * a.d_col], d.md) / d.sd;
    return fmax(p - q, 0.0);
}

// Segment sums of what is left of p, blockIdx.x = sequence * n_seg + segment.
__global__ __launch_bounds__(kThreads) void k_verify_left(VerifyArgs a)
{
    __shared__ int first_s;
    __shared__ Decision d_s;
    __shared__ double s_s[kThreads / 64];
    const int t = threadIdx.x;
    const unsigned b = a.by_seg.div(blockIdx.x), seg = blockIdx.x - b * a.n_seg;
    const Decision d = decide<false>(a, b, first_s, d_s);
    if (seg == 0 && t == 0) a.decision[b] = d;
    if (!d.drafted) return;
    const unsigned end = min((seg + 1) * a.seg, a.vocab);
    double s = 0.0;
    for (unsigned v = seg * a.seg + t; v < end; v += kThreads) s += left_of(a, d, v);
    s = wave_sum64(s);
    if ((t & 63) == 0) s_s[t >> 6] = s;
    __syncthreads();
    if (t == 0) a.left[(size_t)b * a.n_seg + seg] = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
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

// The next token of sequence blockIdx.x.
template <bool GREEDY, bool DECIDE> __global__ __launch_bounds__(kThreads) void k_verify_pick(VerifyArgs a)
{
    __shared__ int first_s;
    __shared__ Decision d_s;
    __shared__ double wave_s[kThreads / 64], before_s;
    __shared__ unsigned at_s, last_s;
    const int t = threadIdx.x;
    const unsigned b = blockIdx.x;
    const Decision d = DECIDE ? decide<GREEDY>(a, b, first_s, d_s) : a.decision[b];
    if (t == 0) a.out_accepted[b] = (float)d.accepted;
    if (GREEDY || d.row < 0)
    {
        if (t == 0) a.out_token[b] = (float)d.token;
        return;
    }
    const size_t at = (size_t)d.row * a.n_seg;
    bool left = d.drafted;   // whether p is lessened by q
    auto of_segment = [&](unsigned i) -> double {
        if (i >= a.n_seg) return 0.0;
        return left ? a.left[(size_t)b * a.n_seg + i] : a.part_s[at + i] * term(a, a.part_m[at + i], d.mt);
    };
    double whole = 0.0;
    for (int again = 0; again < 2; ++again)
    {
        whole = 0.0;
        for (unsigned i = 0; i < a.n_seg; i += kThreads)
        {
            double all;
            scan(of_segment(i + t), wave_s, all);
            whole += all;
        }
        if (whole > 0.0 || !left) break;
        left = false;
    }
    const float w = a.pick[b];
    const double want = (w >= 1.0f ? 1.0 - 0x1p-53 : w > 0.0f ? (double)w : 0.0) * whole;
    // The first segment whose cumulative sum is above that, the last one with anything where rounding leaves none.
    if (t == 0) at_s = a.n_seg, last_s = 0, before_s = 0.0;
    __syncthreads();
    double sum = 0.0;
    for (unsigned i = 0; i < a.n_seg; i += kThreads)
    {
        double all;
        const double x = of_segment(i + t), up = sum + scan(x, wave_s, all);
        if (x > 0.0)
        {
            atomicMax(&last_s, i + t);
            if (up > want) atomicMin(&at_s, i + t);
        }
        __syncthreads();
        if (at_s == i + t) before_s = up - x;
        __syncthreads();
        if (at_s < a.n_seg) break;
        sum += all;
    }
    const bool found = at_s < a.n_seg;
    const unsigned seg = found ? at_s : last_s;
    const double base = before_s;
    __syncthreads();
    // The token, alike: 'want' lies past the last one with anything where no cumulative sum is above it.
    if (t == 0) at_s = a.vocab, last_s = 0;
    __syncthreads();
    const unsigned end = min((seg + 1) * a.seg, a.vocab);
    sum = found ? base : -__builtin_inf();
    for (unsigned v0 = seg * a.seg; v0 < end; v0 += kThreads)
    {
        double all;
        const unsigned v = v0 + t;
        double x = 0.0;
        if (v < end) x = left ? left_of(a, d, v) : term(a, a.target[(size_t)d.row * a.t_row + (size_t)v * a.t_col], d.mt);
        const double up = sum + scan(x, wave_s, all);
        if (x > 0.0)
        {
            atomicMax(&last_s, v);
            if (up > want) atomicMin(&at_s, v);
        }
        __syncthreads();
        if (at_s < a.vocab) break;
        sum += all;
    }
    if (t == 0) a.out_token[b] = (float)(at_s < a.vocab ? at_s : last_s);
}

struct VerifyPlan
{
    unsigned seg, n_seg;
};
VerifyPlan verify_plan(size_t tokens, size_t vocab)
{
    // Some 8 workgroups a CU for the first launch, of 512 logits at least to a row.
    size_t seg = 512;
    while (seg < 4096 && 2 * tokens * ((vocab + seg - 1) / seg) > 8 * (size_t)device_cus()) seg *= 2;
    while ((vocab + seg - 1) / seg > kMostSegments) seg *= 2;
    return {static_cast<unsigned>(seg), static_cast<unsigned>((vocab + seg - 1) / seg)};
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
    s.all = s.left + batch * p.n_seg * sizeof(double);
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
    return verify_ok(tokens, batch, most, vocab) ? verify_space(tokens, batch, verify_plan(tokens, vocab)).all : 0;
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
    const VerifyPlan plan = verify_plan(tokens, vocab);
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
    a.by_seg = FastDiv(plan.n_seg);
    if (!token_major)
        while (a.log2_cols < 5 && ((size_t)1 << a.log2_cols) < tokens) ++a.log2_cols;
    a.inv = greedy ? 0.0 : 1.0 / static_cast<double>(temperature);
    auto* ws = static_cast<char*>(workspace);
    a.part_s = reinterpret_cast<double*>(ws);
    a.part_m = reinterpret_cast<float*>(ws + space.part_m);
    a.decision = reinterpret_cast<Decision*>(ws + space.decision);
    a.left = reinterpret_cast<double*>(ws + space.left);
    a.out_accepted = out_accepted;
    a.out_token = out_token;
    const size_t cols = (size_t)1 << a.log2_cols, blocks = (tokens + cols - 1) / cols * plan.n_seg;
    if (blocks > kGridMost || batch * plan.n_seg > kGridMost) return -1;
    auto s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(blocks), a.draft ? 2 : 1);
    const dim3 all(static_cast<unsigned>(batch));
    if (greedy)
    {
        hipLaunchKernelGGL(k_verify_sums<true>, grid, dim3(kThreads), 0, s, a);
        if (int rc = launch_status()) return rc;
        hipLaunchKernelGGL((k_verify_pick<true, true>), all, dim3(kThreads), 0, s, a);
        return launch_status();
    }
    hipLaunchKernelGGL(k_verify_sums<false>, grid, dim3(kThreads), 0, s, a);
    if (int rc = launch_status()) return rc;
    if (most == 1)
    {
        hipLaunchKernelGGL((k_verify_pick<false, true>), all, dim3(kThreads), 0, s, a);
        return launch_status();
    }
    hipLaunchKernelGGL(k_verify_left, dim3(static_cast<unsigned>(batch * plan.n_seg)), dim3(kThreads), 0, s, a);
    if (int rc = launch_status()) return rc;
    hipLaunchKernelGGL((k_verify_pick<false, false>), all, dim3(kThreads), 0, s, a);
    return launch_status();
}
