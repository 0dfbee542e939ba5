// k_attn_paged.hip — one query per sequence and head against paged keys and
// values, the first positions that a group of sequences shares read once for
// the whole group:
//
//   s_j = alpha q . k_j - slope (len - 1 - j),  m = max_j s_j,
//   l = sum_j exp(s_j - m),  O = sum_j exp(s_j - m) v_j / l.
//
// The positions are cut into ranges: each group's shared ones into n_shared,
// each sequence's others into n_own. A workgroup takes one range for up to 16
// rows of each of its row waves (a row: one query head of one sequence that
// reads the key head) and keeps m, l and the unnormalised O of its range; a
// second kernel joins a row's ranges in order.
//
// A wave forms both products transposed on the float32 matrix cores, 16
// positions by 16 rows at a time:
//   S^T = K Q^T    lane l gives K[position l % 16] and gets S of the positions
//                  4 (l / 16) + r, r < 4, of row l % 16;
//   O^T = V^T P^T  the lane's four weights are then the operand of the four
//                  products as they are: product r sums over the positions
//                  4 (l / 16) + r, for which the lane gives V.
// So keys, values and weights go from memory to the matrix cores without LDS
// or exchange between lanes, and the row's factor exp(m_old - m_new) is the
// lane's own.
#include "kv_pages.hpp"

namespace nnhip
{
namespace
{

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 16;          // positions and rows of a product
constexpr int kPagedMaxDim = 128;

struct PagedArgs
{
    Pages c;
    const float* q;
    long q_t, q_f;
    const float *len, *shared, *slopes;
    float* O;
    long o_t, o_f;
    float *m, *l;
    float *part_ml, *part_o;   // per (row of the batch, range): m and l; O unnormalised
    unsigned q_heads, group, n_shared, n_own, shared_blocks, shared_row_blocks, own_row_blocks;
    int shared_rws, own_rws;
    float alpha;
};

// The positions that sequence b's group shares, as far as they go.
__device__ __forceinline__ int shared_of(const PagedArgs& a, unsigned b)
{
    return a.shared ? length_of(a.shared[b / a.group], (int)(a.c.width * a.c.page.d)) : 0;
}

template <int DP> struct Geometry
{
    // Value columns of a lane: VW neighbouring ones of every 16 VW.
    static constexpr int VW = DP % 64 == 0 ? 4 : 2;
    static constexpr int T = DP / (16 * VW);
    static constexpr int KS = DP / 16;   // groups of 16 key dims
};

// The tile of 16 positions from p0 on, for the lane: its key dims and its value columns of 4 positions.
template <int DP> struct Tile
{
    using G = Geometry<DP>;
    f32x4 k[G::KS];
    float v[4][G::T][G::VW];
    bool there[4];   // of the lane's four positions
};

template <int DP, bool VEC>
__device__ __forceinline__ void load_tile(const PagedArgs& a, unsigned b, unsigned h, int p0, int end, int lane,
                                          Tile<DP>& x)
{
    using G = Geometry<DP>;
    const int j = lane & 15, g = lane >> 4, dim = a.c.dim;
    const long row = p0 + j < end ? a.c.row_of(b, p0 + j) : -1;
    const float* kp = a.c.K + row * a.c.row + (long)h * dim;
#pragma unroll
    for (int i = 0; i < G::KS; ++i)
    {
        const int d = 16 * i + 4 * g;
        f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row >= 0)
        {
            if constexpr (VEC)
            {
                if (d < dim) z = *reinterpret_cast<const f32x4*>(kp + d);
            }
            else
            {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < dim) z[e] = kp[d + e];
            }
        }
        x.k[i] = z;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
    {
        const int lo = __shfl((int)row, 4 * g + r, 64), hi = __shfl((int)(row >> 32), 4 * g + r, 64);
        const long vr = ((long)hi << 32) | (unsigned)lo;
        x.there[r] = vr >= 0;
        const float* vp = a.c.V + vr * a.c.row + (long)h * dim;
#pragma unroll
        for (int t = 0; t < G::T; ++t)
        {
            const int d = 16 * G::VW * t + G::VW * j;
#pragma unroll
            for (int e = 0; e < G::VW; ++e) x.v[r][t][e] = 0.0f;
            if (vr < 0) continue;
            if constexpr (VEC)
            {
                typedef float vec __attribute__((ext_vector_type(G::VW)));
                if (d < dim)
                {
                    const vec z = *reinterpret_cast<const vec*>(vp + d);
#pragma unroll
                    for (int e = 0; e < G::VW; ++e) x.v[r][t][e] = z[e];
                }
            }
            else
            {
#pragma unroll
                for (int e = 0; e < G::VW; ++e)
                    if (d + e < dim) x.v[r][t][e] = vp[d + e];
            }
        }
    }
}

// rws of the 4 waves lie along the rows (16 rws rows a workgroup), the others take the range's positions in turn.
template <int DP, bool VEC> __global__ __launch_bounds__(256) void k_attn_paged(PagedArgs a)
{
    using G = Geometry<DP>;
    __shared__ float o_s[4][kTile][DP + 4];
    __shared__ float ml_s[4][kTile][2];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int j = lane & 15, g = lane >> 4;
    const unsigned per = a.q_heads / a.c.heads;   // query heads of a key head

    // Which range of which positions for which rows.
    unsigned i = blockIdx.x;
    const bool is_shared = i < a.shared_blocks;
    const int rws = is_shared ? a.shared_rws : a.own_rws, kws = 4 / rws, rw = wave % rws, kw = wave / rws;
    unsigned b0, nb, h, c, rb;   // sequences b0 .. b0 + nb - 1, key head, range, block of rows
    if (is_shared)
    {
        rb = i % a.shared_row_blocks;
        i /= a.shared_row_blocks;
        c = i % a.n_shared;
        i /= a.n_shared;
        h = i % a.c.heads;
        b0 = i / a.c.heads * a.group;
        nb = a.group;
    }
    else
    {
        i -= a.shared_blocks;
        rb = i % a.own_row_blocks;
        i /= a.own_row_blocks;
        c = i % a.n_own;
        i /= a.n_own;
        h = i % a.c.heads;
        b0 = i / a.c.heads;
        nb = 1;
    }
    const int most = (int)(a.c.width * a.c.page.d);
    const int common = shared_of(a, b0);
    int lo = 0, hi = common;
    if (!is_shared)
    {
        hi = length_of(a.len[b0], most);
        lo = hi >= common ? common : 0;
    }
    const int ranges = is_shared ? a.n_shared : a.n_own;
    const int step = kws * kTile, steps = (hi - lo + step - 1) / step;
    const int first = (int)((long)steps * c / ranges), last = (int)((long)steps * (c + 1) / ranges);
    const int begin = lo + first * step, end = min(hi, lo + last * step);

    // The lane's row.
    const unsigned row = (rb * rws + rw) * kTile + j;
    const bool live = row < nb * per;
    const unsigned b = live ? b0 + row / per : b0, qh = h * per + (live ? row % per : 0);
    const int len = live ? length_of(a.len[b], most) : 0;
    const bool counts = live && (!is_shared || len >= common);
    const float slope = a.slopes && live ? a.slopes[qh] : 0.0f;
    const int dim = a.c.dim;
    float m = kLowest, l = 0.0f;
    f32x4 o[G::T][G::VW];
#pragma unroll
    for (int x = 0; x < G::T; ++x)
#pragma unroll
        for (int y = 0; y < G::VW; ++y) o[x][y] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    if (begin < end)
    {
        f32x4 q[G::KS];
        const float* qp = a.q + (long)b * a.q_t + (long)qh * dim * a.q_f;
#pragma unroll
        for (int x = 0; x < G::KS; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                const int d = 16 * x + 4 * g + e;
                q[x][e] = live && d < dim ? qp[(long)d * a.q_f] : 0.0f;
            }
        Tile<DP> cur, next;
        int p0 = begin + kw * kTile;
        load_tile<DP, VEC>(a, b0, h, p0, end, lane, cur);
        for (; p0 < end; p0 += step)
        {
            load_tile<DP, VEC>(a, b0, h, p0 + step, end, lane, next);
            f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < G::KS; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.k[x][e], q[x][e], s, 0, 0, 0);
            float top = kLowest;
#pragma unroll
            for (int r = 0; r < 4; ++r)
            {
                float z = a.alpha * s[r];
                if (a.slopes) z -= slope * (float)(len - 1 - (p0 + 4 * g + r));
                s[r] = cur.there[r] && counts ? z : -__builtin_inff();
                top = fmax_std(top, s[r]);
            }
            top = fmax_std(top, __shfl_xor(top, 16, 64));
            top = fmax_std(top, __shfl_xor(top, 32, 64));
            const float mn = fmax_std(m, top);
            const float f = __builtin_amdgcn_exp2f((m - mn) * kLog2e);
            const float mb = mn == kLowest ? 0.0f : mn * kLog2e;
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r)
            {
                s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], kLog2e, -mb));
                sum += s[r];
            }
            l = l * f + sum;   // of the lane's positions
            m = mn;
#pragma unroll
            for (int x = 0; x < G::T; ++x)
#pragma unroll
                for (int y = 0; y < G::VW; ++y)
                {
                    o[x][y] *= f;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        o[x][y] = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.v[r][x][y], s[r], o[x][y], 0, 0, 0);
                }
            cur = next;
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
    }

    // The waves of the same rows are joined through LDS, in the order of their positions.
    if (g == 0)
    {
        ml_s[wave][j][0] = m;
        ml_s[wave][j][1] = l;
    }
#pragma unroll
    for (int x = 0; x < G::T; ++x)
#pragma unroll
        for (int y = 0; y < G::VW; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) o_s[wave][j][16 * G::VW * x + G::VW * (4 * g + r) + y] = o[x][y][r];
    __syncthreads();
    const unsigned n_parts = a.n_shared + a.n_own, slot = is_shared ? c : a.n_shared + c;
    const bool direct = n_parts == 1;
    for (int w = 0; w < rws; ++w)
        for (int e = t; e < kTile * DP; e += 256)
        {
            const int jr = e / DP, d = e % DP;
            const unsigned rr = (rb * rws + w) * kTile + jr;
            if (rr >= nb * per || d >= dim) continue;
            const unsigned bb = b0 + rr / per, hh = h * per + rr % per;
            float mm = kLowest, ll = 0.0f, oo = 0.0f;
            for (int k = w; k < 4; k += rws) mm = fmax_std(mm, ml_s[k][jr][0]);
            for (int k = w; k < 4; k += rws)
            {
                const float lk = ml_s[k][jr][1];
                if (lk == 0.0f) continue;
                const float f = __builtin_amdgcn_exp2f((ml_s[k][jr][0] - mm) * kLog2e);
                ll += lk * f;
                oo += o_s[k][jr][d] * f;
            }
            const size_t at = (size_t)bb * a.q_heads + hh;
            if (direct)
            {
                a.O[(long)bb * a.o_t + ((long)hh * dim + d) * a.o_f] = ll == 0.0f ? 0.0f : oo / ll;
                if (d == 0 && a.m) a.m[at] = mm;
                if (d == 0 && a.l) a.l[at] = ll;
            }
            else
            {
                const size_t p = at * n_parts + slot;
                a.part_o[p * dim + d] = oo;
                if (d == 0)
                {
                    a.part_ml[2 * p] = mm;
                    a.part_ml[2 * p + 1] = ll;
                }
            }
        }
}

// Joins the ranges of one row: blockIdx.x = sequence * q_heads + head.
__global__ __launch_bounds__(128) void k_attn_paged_join(PagedArgs a)
{
    const size_t at = blockIdx.x;
    const unsigned b = (unsigned)(at / a.q_heads), h = (unsigned)(at % a.q_heads), n = a.n_shared + a.n_own;
    const int d = threadIdx.x, dim = a.c.dim;
    const float* ml = a.part_ml + 2 * at * n;
    float m = kLowest, l = 0.0f, o = 0.0f;
    for (unsigned i = 0; i < n; ++i)
        if (ml[2 * i + 1] != 0.0f) m = fmax_std(m, ml[2 * i]);
    for (unsigned i = 0; i < n; ++i)
    {
        const float li = ml[2 * i + 1];
        if (li == 0.0f) continue;
        const float f = __builtin_amdgcn_exp2f((ml[2 * i] - m) * kLog2e);
        l += li * f;
        if (d < dim) o += a.part_o[(at * n + i) * dim + d] * f;
    }
    if (d < dim) a.O[(long)b * a.o_t + ((long)h * dim + d) * a.o_f] = l == 0.0f ? 0.0f : o / l;
    if (d == 0 && a.m) a.m[at] = m;
    if (d == 0 && a.l) a.l[at] = l;
}

struct PagedPlan
{
    unsigned n_shared, n_own, shared_row_blocks, own_row_blocks;
    int shared_rws, own_rws;
    size_t shared_blocks, own_blocks;
    size_t parts() const { return (size_t)n_shared + n_own; }
};

// How a call is cut, from its sizes alone: the lengths are on the device.
PagedPlan paged_plan(const nnhip_kv_pages& c, size_t q_heads, size_t group)
{
    PagedPlan p{};
    const size_t per = q_heads / c.heads, most = c.width * c.page, target = 4 * (size_t)device_cus();
    auto along_rows = [](size_t rows, int& rws, unsigned& blocks) {
        rws = rows > 32 ? 4 : rows > 16 ? 2 : 1;
        blocks = static_cast<unsigned>((rows + kTile * rws - 1) / (kTile * rws));
    };
    auto ranges = [&](size_t others) {
        const size_t want = (target + others - 1) / others, most_ranges = (most + 63) / 64;
        return static_cast<unsigned>(want < most_ranges ? want : most_ranges);
    };
    along_rows(per, p.own_rws, p.own_row_blocks);
    const size_t own = c.batch * c.heads * p.own_row_blocks;
    p.n_own = ranges(own);
    p.own_blocks = own * p.n_own;
    if (group > 1)
    {
        along_rows(group * per, p.shared_rws, p.shared_row_blocks);
        const size_t sh = c.batch / group * c.heads * p.shared_row_blocks;
        p.n_shared = ranges(sh);
        p.shared_blocks = sh * p.n_shared;
    }
    return p;
}

template <int DP, bool VEC> void paged_launch(const PagedArgs& a, const PagedPlan& p, hipStream_t s)
{
    hipLaunchKernelGGL((k_attn_paged<DP, VEC>), dim3(static_cast<unsigned>(p.shared_blocks + p.own_blocks)), dim3(256),
                       0, s, a);
}

bool paged_ok(const nnhip_kv_pages* c, size_t q_heads, size_t group)
{
    return pages_ok(c, kPagedMaxDim) && q_heads > 0 && q_heads % c->heads == 0 && q_heads <= kMaxIndex && group > 0 &&
           group <= c->batch && c->batch % group == 0;
}

} // namespace
} // namespace nnhip

using namespace nnhip;

extern "C" size_t nnhip_attn_paged_workspace_bytes(const nnhip_kv_pages* c, size_t q_heads, size_t group)
{
    if (!paged_ok(c, q_heads, group)) return 0;
    const PagedPlan p = paged_plan(*c, q_heads, group);
    return p.parts() == 1 ? 0 : c->batch * q_heads * p.parts() * (2 + c->dim) * sizeof(float);
}

extern "C" int nnhip_attn_paged(const nnhip_kv_pages* c, const float* q, long q_t, long q_f, size_t q_heads,
                                const float* len, const float* shared, size_t group, const float* slopes, float alpha,
                                float* O, long o_t, long o_f, float* m, float* l, void* workspace,
                                size_t workspace_bytes, void* stream)
{
    if (!paged_ok(c, q_heads, group) || !q || !len || !O || q_t < 0 || q_f < 0 || o_t < 0 || o_f < 0 ||
        c->batch * q_heads > 0x7fffffffu)
        return -1;
    const size_t need = nnhip_attn_paged_workspace_bytes(c, q_heads, group);
    if (need > 0 && (!workspace || workspace_bytes < need)) return -1;
    PagedPlan p = paged_plan(*c, q_heads, group);
    if (group == 1) shared = nullptr;   // a group of one has all positions to itself
    if (!shared)
    {
        p.n_shared = 0;
        p.shared_blocks = 0;
    }
    if (p.shared_blocks + p.own_blocks > 0x7fffffffu) return -1;
    auto* ws = static_cast<float*>(workspace);
    PagedArgs a{pages_of(*c), q, q_t, q_f, len, shared, slopes, O, o_t, o_f, m, l, ws, nullptr,
                static_cast<unsigned>(q_heads), static_cast<unsigned>(group), p.n_shared, p.n_own,
                static_cast<unsigned>(p.shared_blocks), p.shared_row_blocks, p.own_row_blocks, p.shared_rws, p.own_rws,
                alpha};
    if (p.parts() > 1) a.part_o = ws + 2 * c->batch * q_heads * p.parts();
    const size_t d = c->dim;
    const bool vec = d % 4 == 0 && c->row % 4 == 0 && aligned16(c->K) && aligned16(c->V);
    auto s = static_cast<hipStream_t>(stream);
    if (d <= 32) vec ? paged_launch<32, true>(a, p, s) : paged_launch<32, false>(a, p, s);
    else if (d <= 64) vec ? paged_launch<64, true>(a, p, s) : paged_launch<64, false>(a, p, s);
    else if (d <= 96) vec ? paged_launch<96, true>(a, p, s) : paged_launch<96, false>(a, p, s);
    else vec ? paged_launch<128, true>(a, p, s) : paged_launch<128, false>(a, p, s);
    if (int rc = launch_status()) return rc;
    if (p.parts() > 1)
    {
        hipLaunchKernelGGL(k_attn_paged_join, dim3(static_cast<unsigned>(c->batch * q_heads)), dim3(128), 0, s, a);
        return launch_status();
    }
    return 0;
}
