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
//
// Unshared sequences are bound by HBM: 24 of 2500 to 5000 positions, 8 heads of
// 80, take 102 us, 4.9 TB/s. Few positions are bound by the latency of two
// launches (4 beams of 321 positions: 7.1 us and 4). Shared ones that more than
// 32 rows read are bound by the products and the vector instructions around
// them, which is why these rows have a walk in bf16 parts.
#include "kv_pages.hpp"
#include "split_bf16.hpp"

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
    unsigned q_heads, group, n_shared, n_own, shared_blocks;
    // per: query heads of a key head; of the shared and the own parts: 8 row blocks, ranges
    FastDiv by_per, by_heads, by_shared_rows, by_own_rows, by_n_shared, by_n_own;
    int q_rows;   // queries lie a token a row, 16-byte aligned
    int shared_row_waves, own_row_waves, own_wide;   // own_wide: own parts in RT row tiles a wave too
    float alpha;
};

// The positions that sequence b's group shares, as far as they go.
__device__ __forceinline__ int shared_of(const PagedArgs& a, unsigned b)
{
    return a.shared ? length_of(a.shared[b / a.group], (int)(a.c.width * a.c.page.d)) : 0;
}

// The first sequence of the group from b0 on that is as long as the positions it shares: a shorter one's table need not
// name them. b0 + group where there is none.
__device__ __forceinline__ unsigned reader_of(const PagedArgs& a, unsigned b0, int common)
{
    const unsigned lane = threadIdx.x & 63;
    for (unsigned i = 0; i < a.group; i += 64)
    {
        const int len = length_of(a.len[b0 + min(i + lane, a.group - 1)], (int)(a.c.width * a.c.page.d));
        const unsigned long long long_enough = __builtin_amdgcn_ballot_w64(i + lane < a.group && len >= common);
        if (long_enough) return b0 + i + __builtin_ctzll(long_enough);
    }
    return b0 + a.group;
}

// KS: groups of 16 key dims. Value columns of a lane: VW neighbouring ones of every 16 VW; columns past dim are
// formed and dropped.
template <int KS> struct Geometry
{
    static constexpr int VW = KS % 4 == 0 || KS % 4 == 3 ? 4 : 2;
    static constexpr int T = (KS + VW - 1) / VW;
    static constexpr int DV = 16 * VW * T;
};

// How keys and values are loaded: whole groups of 16 dims in 16-byte pieces; 16-byte pieces whose last group is
// cut (dim % 16 != 0); or one float at a time (rows that are not 16-byte aligned).
enum { kWhole = 0, kCut = 1, kSingle = 2 };

// 16 positions, for the lane: its dims of one key, its value columns of four positions.
template <int KS> struct Tile
{
    using G = Geometry<KS>;
    f32x4 k[KS];
    float v[4][G::T][G::VW];
    int row[4];   // of the values' positions, -1: none
};

// Loads are issued whatever the positions are, from row 0 where there is none, so that no branch holds the next
// tile's loads back behind this one's: the weights of such positions are 0, and their values are cleared before
// use (0 times a NaN that lies there would be one).
template <int KS, int MODE>
__device__ __forceinline__ void load_keys(const PagedArgs& a, int row, unsigned h, int lane, Tile<KS>& x)
{
    const int g = lane >> 4, dim = a.c.dim;
    const float* kp = a.c.K + (size_t)max(row, 0) * a.c.row + (size_t)h * dim;
#pragma unroll
    for (int i = 0; i < KS; ++i)
    {
        const int d = 16 * i + 4 * g;
        if constexpr (MODE == kWhole) x.k[i] = *reinterpret_cast<const f32x4*>(kp + d);
        else if constexpr (MODE == kCut)
        {
            x.k[i] = *reinterpret_cast<const f32x4*>(kp + (d < dim ? d : 0));
        }
        else
        {
#pragma unroll
            for (int e = 0; e < 4; ++e) x.k[i][e] = kp[d + e < dim ? d + e : 0];
        }
    }
}
template <int KS, int MODE>
__device__ __forceinline__ void load_values(const PagedArgs& a, int row, unsigned h, int lane, Tile<KS>& x)
{
    using G = Geometry<KS>;
    const int j = lane & 15, g = lane >> 4, dim = a.c.dim;
#pragma unroll
    for (int r = 0; r < 4; ++r)
    {
        x.row[r] = __shfl(row, 4 * g + r, 64);
        const float* vp = a.c.V + (size_t)max(x.row[r], 0) * a.c.row + (size_t)h * dim;
#pragma unroll
        for (int t = 0; t < G::T; ++t)
        {
            const int d = 16 * G::VW * t + G::VW * j;
            if constexpr (MODE == kSingle)
            {
#pragma unroll
                for (int e = 0; e < G::VW; ++e) x.v[r][t][e] = vp[d + e < dim ? d + e : 0];
            }
            else
            {
                typedef float vec __attribute__((ext_vector_type(G::VW)));
                const vec z = *reinterpret_cast<const vec*>(vp + (d < dim ? d : 0));
#pragma unroll
                for (int e = 0; e < G::VW; ++e) x.v[r][t][e] = z[e];
            }
        }
    }
}

// Dims past the last one are 0 in keys and queries.
template <int KS, int MODE> __device__ __forceinline__ void cut(f32x4 (&x)[KS], int g, int dim)
{
    if constexpr (MODE != kWhole)
    {
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = 16 * i + 4 * g + e < dim ? x[i][e] : 0.0f;
    }
}

// A lane's row of each of a wave's row tiles: its query dims, the sequence's length, the bias' slope, whether the
// positions count for it; and the running softmax.
template <int KS> struct Row
{
    using G = Geometry<KS>;
    f32x4 q[KS];
    int len;
    float slope;
    bool counts;
    float m, l;   // l: of the lane's positions alone
    f32x4 o[G::T][G::VW];
};

template <int KS, int MODE, int RT>
__device__ __forceinline__ void use_keys(const PagedArgs& a, Tile<KS>& x, const Row<KS> (&rows)[RT], int g, f32x4 (&s)[RT])
{
    cut<KS, MODE>(x.k, g, a.c.dim);
#pragma unroll
    for (int i = 0; i < RT; ++i) s[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < RT; ++i)
                s[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[k][e], rows[i].q[k][e], s[i], 0, 0, 0);
}

template <int KS, int RT>
__device__ __forceinline__ void use_values(const PagedArgs& a, Tile<KS>& x, f32x4 (&s)[RT], Row<KS> (&rows)[RT], int p0,
                                           int g)
{
    using G = Geometry<KS>;
    const int least = min(min(x.row[0], x.row[1]), min(x.row[2], x.row[3]));
    if (__builtin_amdgcn_ballot_w64(least < 0))
    {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < G::T; ++t)
#pragma unroll
                for (int y = 0; y < G::VW; ++y) x.v[r][t][y] = x.row[r] < 0 ? 0.0f : x.v[r][t][y];
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        Row<KS>& w = rows[i];
        float top = kLowest;
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            float z = a.alpha * s[i][r];
            if (a.slopes) z -= w.slope * (float)(w.len - 1 - (p0 + 4 * g + r));
            s[i][r] = x.row[r] >= 0 && w.counts ? z : -__builtin_inff();
            top = fmax_std(top, s[i][r]);
        }
        top = fmax_std(top, __shfl_xor(top, 16, 64));
        top = fmax_std(top, __shfl_xor(top, 32, 64));
        const float mn = fmax_std(w.m, top);
        const float f = __builtin_amdgcn_exp2f((w.m - mn) * kLog2e);
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            // The difference first: of scores times log2(e) it would be off by their size, and past 2^30 exp2 of that
            // overflows.
            s[i][r] = __builtin_amdgcn_exp2f((s[i][r] - mn) * kLog2e);
            sum += s[i][r];
        }
        w.l = w.l * f + sum;
        w.m = mn;
        if (__builtin_amdgcn_ballot_w64(f != 1.0f))   // seldom past the first tiles
        {
#pragma unroll
            for (int t = 0; t < G::T; ++t)
#pragma unroll
                for (int y = 0; y < G::VW; ++y) w.o[t][y] *= f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < G::T; ++t)
#pragma unroll
                for (int y = 0; y < G::VW; ++y)
                    w.o[t][y] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[r][t][y], s[i][r], w.o[t][y], 0, 0, 0);
    }
}

// A workgroup's rows and positions.
struct Part
{
    unsigned b0, nb, h, rb, slot;   // sequences b0 .. b0 + nb - 1, key head, block of rows, range of all
    unsigned by;                    // the sequence whose table is read
    int begin, end, common, row_waves;
    bool is_shared;
};
template <int KS> struct PartShared
{
    float o[4][kTile][Geometry<KS>::DV + 4];
    float ml[4][kTile][2];
};

// The waves' results for 16 rows of each row wave (rows first + rv * apart on) are joined through LDS, in the order
// of their positions, and written: 16 threads a row, 4 neighbouring values at a time.
template <int KS, int MODE>
__device__ __forceinline__ void join_waves(const PagedArgs& a, const Part& part, PartShared<KS>& sh, float m, float l,
                                           const f32x4 (&o)[Geometry<KS>::T][Geometry<KS>::VW], unsigned first, int rws,
                                           unsigned apart, unsigned n_rows)
{
    using G = Geometry<KS>;
    constexpr int DP = G::DV;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, j = lane & 15, g = lane >> 4, dim = a.c.dim;
    const unsigned per = a.by_per.d, n_parts = a.n_shared + a.n_own;
    const bool direct = n_parts == 1;
    __syncthreads();
    if (g == 0)
    {
        sh.ml[wave][j][0] = m;
        sh.ml[wave][j][1] = l;
    }
#pragma unroll
    for (int x = 0; x < G::T; ++x)
#pragma unroll
        for (int y = 0; y < G::VW; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) sh.o[wave][j][16 * G::VW * x + G::VW * (4 * g + r) + y] = o[x][y][r];
    __syncthreads();
    const int jr = t >> 4;
    for (int rv = 0; rv < rws; ++rv)   // row waves
    {
        const unsigned row = first + rv * apart + jr;
        if (row >= n_rows) break;
        const unsigned bq = a.by_per.div(row), b = part.b0 + bq, qh = part.h * per + (row - bq * per);
        float mm = kLowest, ll = 0.0f, f[4];
        bool any[4];   // waves that had positions: a NaN among these stays one, whatever its factor is
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k % rws == rv) mm = fmax_std(mm, sh.ml[k][jr][0]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            const float lk = sh.ml[k][jr][1];
            any[k] = k % rws == rv && lk != 0.0f;
            f[k] = __builtin_amdgcn_exp2f((sh.ml[k][jr][0] - mm) * kLog2e);
            ll += any[k] ? lk * f[k] : 0.0f;
        }
        const size_t at = (size_t)b * a.q_heads + qh, p = at * n_parts + part.slot;
        const float inv = !direct ? 1.0f : ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
        for (int x = 0; x < (DP + 63) / 64; ++x)
        {
            const int d = 64 * x + 4 * (t & 15);
            if (d >= dim) continue;
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (any[k]) o += *reinterpret_cast<const f32x4*>(&sh.o[k][jr][d]) * f[k];
            o *= inv;
            if (!direct && MODE != kSingle) *reinterpret_cast<f32x4*>(a.part_o + p * dim + d) = o;
            else
            {
                float* to = direct ? a.O + (long)b * a.o_t + (long)qh * dim * a.o_f : a.part_o + p * dim;
                const long step_f = direct ? a.o_f : 1;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < dim) to[(d + e) * step_f] = o[e];
            }
        }
        if ((t & 15) == 0)
        {
            if (!direct)
            {
                a.part_ml[2 * p] = mm;
                a.part_ml[2 * p + 1] = ll;
            }
            else
            {
                if (a.m) a.m[at] = mm;
                if (a.l) a.l[at] = ll;
            }
        }
    }
}

// One range of positions. row_waves of the 4 waves lie along the rows, RT tiles each; the others take 16 positions
// each in turn.
template <int KS, int MODE, int RT>
__device__ __forceinline__ void walk(const PagedArgs& a, const Part& part, PartShared<KS>& sh)
{
    using G = Geometry<KS>;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, j = lane & 15, g = lane >> 4, dim = a.c.dim;
    const unsigned per = a.by_per.d, n_rows = part.nb * per;
    const int rws = part.row_waves, kws = 4 / rws, rw = wave % rws, kw = wave / rws, step = kws * kTile;
    const int most = (int)(a.c.width * a.c.page.d), begin = part.begin, end = part.end;
    Row<KS> rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        Row<KS>& w = rows[i];
        const unsigned row = ((part.rb * rws + rw) * RT + i) * kTile + j;
        const bool live = row < n_rows;
        const unsigned bq = live ? a.by_per.div(row) : 0, b = part.b0 + bq, qh = part.h * per + (live ? row - bq * per : 0);
        w.len = live ? length_of(a.len[b], most) : 0;
        w.counts = live && (!part.is_shared || w.len >= part.common);
        w.slope = a.slopes && live ? a.slopes[qh] : 0.0f;
        w.m = kLowest;
        w.l = 0.0f;
#pragma unroll
        for (int x = 0; x < G::T; ++x)
#pragma unroll
            for (int y = 0; y < G::VW; ++y) w.o[x][y] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (begin >= end) continue;
        const float* qp = a.q + (long)b * a.q_t + (long)qh * dim * a.q_f;   // rows that are not live are formed and dropped
        if (MODE != kSingle && a.q_rows)
        {
#pragma unroll
            for (int x = 0; x < KS; ++x)
            {
                const int d = 16 * x + 4 * g;
                w.q[x] = *reinterpret_cast<const f32x4*>(qp + (d < dim ? d : 0));
            }
        }
        else
        {
#pragma unroll
            for (int x = 0; x < KS; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    const int d = 16 * x + 4 * g + e;
                    w.q[x][e] = qp[(long)(d < dim ? d : 0) * a.q_f];
                }
        }
    }
    if (begin < end)
    {
#pragma unroll
        for (int i = 0; i < RT; ++i)
        {
            // The loads stay in one run: without this each would move into a branch of the selection that follows.
#pragma unroll
            for (int x = 0; x < KS; ++x) asm volatile("" : "+v"(rows[i].q[x]));
            cut<KS, MODE>(rows[i].q, g, dim);
        }
        // Table entries are loaded two tiles ahead of their use, keys and values one: the entries' loads are then
        // older than the keys' and values' that are still on their way when the addresses are formed.
        auto entry = [&](int p) { return a.c.entry_of(part.by, p + j); };
        auto row_at = [&](float e, int p) {
            const int r = a.c.row_in(e, p + j);
            return p + j < end ? r : -1;
        };
        const int p1 = begin + kw * kTile;
        const float first = entry(p1);
        float ahead = entry(p1 + step);
        f32x4 s[RT];
        if constexpr (RT == 1)
        {
            Tile<KS> x[2];
            const int r0 = row_at(first, p1);
            load_keys<KS, MODE>(a, r0, part.h, lane, x[0]);
            load_values<KS, MODE>(a, r0, part.h, lane, x[0]);
            for (int p = p1; p < end; p += 2 * step)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                {
                    const int at = p + half * step;
                    if (half && at >= end) break;
                    const float further = entry(at + 2 * step);
                    const int r = row_at(ahead, at + step);
                    load_keys<KS, MODE>(a, r, part.h, lane, x[1 - half]);
                    load_values<KS, MODE>(a, r, part.h, lane, x[1 - half]);
                    __builtin_amdgcn_sched_barrier(0);
                    use_keys<KS, MODE, RT>(a, x[half], rows, g, s);
                    use_values<KS, RT>(a, x[half], s, rows, at, g);
                    ahead = further;
                }
        }
        else
        {
            // The registers hold one tile: its keys' loads follow the products of the keys before, its values' those
            // of the values before. Each has the other products' time, some 2000 cycles, to arrive.
            Tile<KS> x;
            const int r0 = row_at(first, p1);
            load_keys<KS, MODE>(a, r0, part.h, lane, x);
            __builtin_amdgcn_sched_barrier(0);
            load_values<KS, MODE>(a, r0, part.h, lane, x);
            __builtin_amdgcn_sched_barrier(0);
            for (int p = p1; p < end; p += step)
            {
                use_keys<KS, MODE, RT>(a, x, rows, g, s);
                __builtin_amdgcn_sched_barrier(0);
                const float further = entry(p + 2 * step);
                const int r = row_at(ahead, p + step);
                load_keys<KS, MODE>(a, r, part.h, lane, x);
                __builtin_amdgcn_sched_barrier(0);
                use_values<KS, RT>(a, x, s, rows, p, g);
                __builtin_amdgcn_sched_barrier(0);
                load_values<KS, MODE>(a, r, part.h, lane, x);
                ahead = further;
            }
        }
    }

#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        Row<KS>& w = rows[i];
        w.l += __shfl_xor(w.l, 16, 64);
        w.l += __shfl_xor(w.l, 32, 64);
        join_waves<KS, MODE>(a, part, sh, w.m, w.l, w.o, (part.rb * rws * RT + i) * kTile, rws, RT * kTile, n_rows);
    }
}

// ── many rows: the products from bf16 parts ─────────────────────────────────
// Where more than 32 rows read the same positions the float32 matrix cores bound the walk above. This one forms
// both products from three bf16 parts of each operand (split_bf16.hpp), six products of 16 x 16 x 32 for each: a
// wave takes 32 positions for 64 rows, so that splitting keys and values, some 9 instructions a pair, is shared by 4
// row tiles. The queries' parts lie in LDS, laid out by lane. Positions and weights are ordered alike on both sides
// of the second product: its k index 8 (l / 16) + e stands for position 16 (e / 4) + 4 (l / 16) + e % 4, which are
// the ones that the lane's scores belong to.
//
// A row's weights are taken against a fixed score, the largest of the wave's first tile that has any (with a slope, what
// that would be at the range's end): sums in floats are as exact against any score that keeps them in range, and
// nothing is scaled on the way, which took 15 us of 140 for moves of the outputs between the matrix cores' registers
// and the others. At the end they are scaled to the largest score.
//
// Weights are split as they are and values times 2^48: 24 added to the exponents' arguments, for the parts' scale, would
// cost these 4 bits, and parts of a weight that counts beside a sum of 2^-60 are normal without it.
//
// Values that the parts do not hold (queries of 2^104, values and sums of 2^80 and above, infinities, NaN) and scores that
// grow by more than some 55 to 69 over a range give sums that are not finite, or above 2^100 (up to there the factor that
// scales them back is a normal float), and scores that fall short of the slope's by 40 small sums; the range is then
// walked again in float32. Keys are split as they are too: of those below 2^-109 parts below 2^-126 are lost, dim alpha
// 2^-22 of a score at most with the largest queries that the parts hold.
//
// 64 rows over 65000 positions of 8 heads of 128 (532 MB) take 120 us by themselves, 4.4 TB/s (92 with the loads alone); 512 rows over
// 6000 take 93 us. Two waves a SIMD of 32 rows each took 160 where one of 64 took 144 (every wave splits all its keys
// and values), and 170 where two waves split a tile in halves, exchanged through LDS.
constexpr int kSplitRows = 4;   // row tiles of a wave

template <int KS> struct SplitTile
{
    using G = Geometry<KS>;
    f32x4 k[2][KS];
    float v[2][4][G::T][G::VW];
    int row[2][4];   // of the values' positions, -1: none
};
template <int KS> struct SplitRow
{
    using G = Geometry<KS>;
    int len;
    float slope;
    bool counts;
    float m, top, l;   // the score that the weights are against, the largest; l: of the lane's positions
    f32x4 o[G::T][G::VW];
};

__device__ __forceinline__ f32x4 mfma16(const bf16x8& x, const bf16x8& y, const f32x4& c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
}
// Which parts (0 large, 2 small) the six products take, the small products first.
constexpr int kPartA[6] = {0, 2, 1, 0, 1, 0}, kPartB[6] = {2, 0, 1, 1, 0, 0};

// Whether every result is finite; false leaves the partial results for the walk that follows.
template <int KS> __device__ __forceinline__ bool walk_split(const PagedArgs& a, const Part& part, bf16x8* qparts, PartShared<KS>& sh)
{
    using G = Geometry<KS>;
    constexpr int RT = kSplitRows, steps = KS / 2;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, j = lane & 15, g = lane >> 4, dim = a.c.dim;
    const unsigned per = a.by_per.d, n_rows = part.nb * per;
    const int most = (int)(a.c.width * a.c.page.d), begin = part.begin, end = part.end, step = 4 * 2 * kTile;
    const SplitUnits units;
    SplitRow<KS> rows[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        SplitRow<KS>& w = rows[i];
        const unsigned row = (part.rb * RT + i) * kTile + j;
        const bool live = row < n_rows;
        const unsigned bq = live ? a.by_per.div(row) : 0, b = part.b0 + bq, qh = part.h * per + (live ? row - bq * per : 0);
        w.len = live ? length_of(a.len[b], most) : 0;
        w.counts = live && w.len >= part.common;
        w.slope = a.slopes && live ? a.slopes[qh] : 0.0f;
        w.m = w.top = kLowest;
        w.l = 0.0f;
#pragma unroll
        for (int x = 0; x < G::T; ++x)
#pragma unroll
            for (int y = 0; y < G::VW; ++y) w.o[x][y] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (i != wave) continue;   // a wave splits the queries of one row tile
        const float* qp = a.q + (long)b * a.q_t + (long)qh * dim * a.q_f;
        floatx8 z[steps];
        if (a.q_rows)
        {
#pragma unroll
            for (int x = 0; x < steps; ++x)
            {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(qp + 32 * x + 8 * g), hi = *reinterpret_cast<const f32x4*>(qp + 32 * x + 8 * g + 4);
                z[x] = floatx8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            }
        }
        else
        {
#pragma unroll
            for (int x = 0; x < steps; ++x)
#pragma unroll
                for (int e = 0; e < 8; ++e) z[x][e] = qp[(long)(32 * x + 8 * g + e) * a.q_f];
        }
#pragma unroll
        for (int x = 0; x < steps; ++x)
        {
            bf16x8 h, m, l;
            split3(units, z[x], h, m, l);
            qparts[((i * 3 + 0) * steps + x) * 64 + lane] = h;
            qparts[((i * 3 + 1) * steps + x) * 64 + lane] = m;
            qparts[((i * 3 + 2) * steps + x) * 64 + lane] = l;
        }
    }
    __syncthreads();

    auto entry = [&](int p) { return a.c.entry_of(part.by, p + j); };
    auto row_at = [&](float e, int p) {
        const int r = a.c.row_in(e, p + j);
        return p + j < end ? r : -1;
    };
    SplitTile<KS> x;
    auto load_k = [&](int (&r)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
        {
            const float* kp = a.c.K + (size_t)max(r[u], 0) * a.c.row + (size_t)part.h * dim;
#pragma unroll
            for (int i = 0; i < KS; ++i) x.k[u][i] = *reinterpret_cast<const f32x4*>(kp + 32 * (i / 2) + 8 * g + 4 * (i % 2));
        }
    };
    auto load_v = [&](int (&r)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                x.row[u][e] = __shfl(r[u], 4 * g + e, 64);
                const float* vp = a.c.V + (size_t)max(x.row[u][e], 0) * a.c.row + (size_t)part.h * dim;
#pragma unroll
                for (int i = 0; i < G::T; ++i)
                {
                    typedef float vec __attribute__((ext_vector_type(G::VW)));
                    const int d = 16 * G::VW * i + G::VW * j;
                    const vec z = *reinterpret_cast<const vec*>(vp + (d < dim ? d : 0));
#pragma unroll
                    for (int y = 0; y < G::VW; ++y) x.v[u][e][i][y] = z[y];
                }
            }
    };
    const int p1 = begin + wave * 2 * kTile;
    float first[2] = {entry(p1), entry(p1 + kTile)}, ahead[2] = {entry(p1 + step), entry(p1 + step + kTile)};
    int r[2] = {row_at(first[0], p1), row_at(first[1], p1 + kTile)};
    load_k(r);
    __builtin_amdgcn_sched_barrier(0);
    load_v(r);
    __builtin_amdgcn_sched_barrier(0);
    // -inf among the scores, which a sum too large for the parts may be too, shows in the smallest; NaN and +inf make
    // the row's l one that is not finite.
    float low = 0.0f;
    const float alpha = a.alpha * (1.0f / kSplitScale);
    for (int p = p1; p < end; p += step)
    {
        f32x4 s[2][RT];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < RT; ++i) s[u][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < steps; ++k)
        {
            bf16x8 kp[2][3], qp[RT][3];
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int c = 0; c < 3; ++c) qp[i][c] = qparts[((i * 3 + c) * steps + k) * 64 + lane];
#pragma unroll
            for (int u = 0; u < 2; ++u)
            {
                const f32x4 lo = x.k[u][2 * k], hi = x.k[u][2 * k + 1];
                split3_scaled(units, floatx8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, kp[u][0], kp[u][1], kp[u][2]);
            }
#pragma unroll
            for (int c = 0; c < 6; ++c)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < RT; ++i) s[u][i] = mfma16(kp[u][kPartA[c]], qp[i][kPartB[c]], s[u][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
        const float further[2] = {entry(p + 2 * step), entry(p + 2 * step + kTile)};
        r[0] = row_at(ahead[0], p + step);
        r[1] = row_at(ahead[1], p + step + kTile);
        load_k(r);
        __builtin_amdgcn_sched_barrier(0);

#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u][i] *= alpha;
        if (a.slopes)
        {
            asm volatile("");   // stays a branch
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int q = 0; q < 4; ++q) s[u][i][q] -= rows[i].slope * (float)(rows[i].len - 1 - (p + kTile * u + 4 * g + q));
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int q = 0; q < 4; ++q) low = fminf(low, s[u][i][q]);
        int least = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) least = min(least, x.row[u][e]);
        if (__builtin_amdgcn_ballot_w64(least < 0))
        {
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int q = 0; q < 4; ++q) s[u][i][q] = x.row[u][q] < 0 ? -__builtin_inff() : s[u][i][q];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < G::T; ++i)
#pragma unroll
                        for (int y = 0; y < G::VW; ++y) x.v[u][e][i][y] = x.row[u][e] < 0 ? 0.0f : x.v[u][e][i][y];
        }
        bf16x8 pp[RT][3];
#pragma unroll
        for (int i = 0; i < RT; ++i)
        {
            SplitRow<KS>& w = rows[i];
            float top = kLowest;
            floatx8 z;
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                z[e] = s[e / 4][i][e % 4];
                top = fmaxf(top, z[e]);
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            w.top = fmaxf(w.top, top);
            if (w.m == kLowest && top > kLowest)   // the first tile with a position
                w.m = top + (a.slopes ? fmax_std(w.slope, 0.0f) * (float)(end - 1 - p) : 0.0f);
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                z[e] = __builtin_amdgcn_exp2f((z[e] - w.m) * kLog2e);
                w.l += z[e];
            }
            split3_scaled(units, z, pp[i][0], pp[i][1], pp[i][2]);
        }
#pragma unroll
        for (int b = 0; b < G::T; ++b)
#pragma unroll
            for (int y = 0; y < G::VW; ++y)
            {
                bf16x8 vp[3];
                floatx8 z;
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = x.v[e / 4][e % 4][b][y] * (1.0f / kSplitUnscale);
                split3_scaled(units, z, vp[0], vp[1], vp[2]);
#pragma unroll
                for (int c = 0; c < 6; ++c)
#pragma unroll
                    for (int i = 0; i < RT; ++i) rows[i].o[b][y] = mfma16(vp[kPartA[c]], pp[i][kPartB[c]], rows[i].o[b][y]);
            }
        __builtin_amdgcn_sched_barrier(0);
        load_v(r);
        __builtin_amdgcn_sched_barrier(0);
        ahead[0] = further[0];
        ahead[1] = further[1];
    }

    // The waves are joined as in walk, once all results are known to be finite.
    bool bad = !(low >= -kMaxF);
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        SplitRow<KS>& w = rows[i];
        const float f = __builtin_amdgcn_exp2f((w.m - w.top) * kLog2e);
        w.l += __shfl_xor(w.l, 16, 64);
        w.l += __shfl_xor(w.l, 32, 64);
        bad |= w.counts && w.m != kLowest && !(w.l >= 0x1p-60f && w.l <= 0x1p100f);
        w.m = w.top;
        w.l *= f;
        float size = 0.0f;
#pragma unroll
        for (int b = 0; b < G::T; ++b)
#pragma unroll
            for (int y = 0; y < G::VW; ++y)
            {
                w.o[b][y] = w.o[b][y] * kSplitUnscale * f;   // one after the other: f times that may be below every float
#pragma unroll
                for (int e = 0; e < 4; ++e) size += fabsf(w.o[b][y][e]) * 0x1p-12f;   // NaN or infinite if one is
            }
        bad |= w.counts && !(size + w.l <= kMaxF);
        if (!w.counts) w.m = kLowest, w.l = 0.0f;   // whatever came of these rows
    }
    if (__syncthreads_or(bad)) return false;
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        SplitRow<KS>& w = rows[i];
        join_waves<KS, kWhole>(a, part, sh, w.m, w.l, w.o, (part.rb * RT + i) * kTile, 1, 0, n_rows);
    }
    return true;
}

// RT: a wave's row tiles of the shared parts (kSplitRows: in bf16 parts), and 2 of the own ones where a key head has
// more than 16 query heads.
template <int KS, int MODE, int RT> __global__ __launch_bounds__(256, MODE == kSingle || RT == kSplitRows ? 1 : 2) void k_attn_paged(PagedArgs a)
{
    constexpr size_t kQueries = RT == kSplitRows ? (size_t)kSplitRows * 3 * (KS / 2) * 64 * sizeof(bf16x8) : 0;
    constexpr size_t kShared = sizeof(PartShared<KS>) > kQueries ? sizeof(PartShared<KS>) : kQueries;
    __shared__ __attribute__((aligned(16))) char lds[kShared];
    PartShared<KS>& sh = *reinterpret_cast<PartShared<KS>*>(lds);
    Part part;
    unsigned i = blockIdx.x, c;
    part.is_shared = i < a.shared_blocks;
    if (!part.is_shared) i -= a.shared_blocks;
    const FastDiv by_rows = part.is_shared ? a.by_shared_rows : a.by_own_rows;
    const FastDiv by_ranges = part.is_shared ? a.by_n_shared : a.by_n_own;
    const unsigned ranges = by_ranges.d;
    // The blocks of rows that read the same keys and values run on one XCD (workgroups go to the 8 in turn), so
    // that its L2 holds them once; the pieces are padded to a multiple of 8.
    const unsigned eight = by_rows.div(i);
    part.rb = (i - eight * by_rows.d) / 8;
    i = eight * 8 + i % 8;
    unsigned next = by_ranges.div(i);
    c = i - next * ranges;
    i = a.by_heads.div(next);
    part.h = next - i * a.c.heads;
    part.nb = part.is_shared ? a.group : 1;
    if (i * part.nb >= a.c.batch) return;
    part.b0 = i * part.nb;
    part.slot = part.is_shared ? c : a.n_shared + c;
    part.row_waves = part.is_shared ? a.shared_row_waves : a.own_row_waves;
    const int len0 = length_of(a.len[part.b0], (int)(a.c.width * a.c.page.d));   // on its way with the shared length
    part.common = shared_of(a, part.b0);
    part.by = part.b0;
    int lo = 0, hi = part.common;
    if (!part.is_shared)
    {
        hi = len0;
        lo = hi >= part.common ? part.common : 0;
    }
    else if (__builtin_expect(len0 < part.common, 0))   // marked seldom, 64 rows over 65000 positions take 120 us instead of 122
    {
        part.by = __builtin_amdgcn_readfirstlane(reader_of(a, part.b0, part.common));
        if (part.by - part.b0 == a.group) hi = 0;   // for no one
    }
    constexpr int kStep = 4 * kTile;
    const int steps = (hi - lo + kStep - 1) / kStep;
    const int first = (int)((long)steps * c / ranges), last = (int)((long)steps * (c + 1) / ranges);
    part.begin = lo + first * kStep;
    part.end = min(hi, lo + last * kStep);
    if (part.begin >= part.end && a.n_shared + a.n_own > 1)
    {
        // Nothing here: the join leaves out ranges of l = 0, whatever their O is.
        const unsigned tiles = part.is_shared ? RT : a.own_wide ? 2 : 1, rows_here = kTile * part.row_waves * tiles;
        const unsigned n_rows = part.nb * a.by_per.d, row = part.rb * rows_here + threadIdx.x;
        if (threadIdx.x < rows_here && row < n_rows)
        {
            const unsigned q = a.by_per.div(row);
            const size_t at = (size_t)(part.b0 + q) * a.q_heads + part.h * a.by_per.d + (row - q * a.by_per.d);
            const size_t p = at * (a.n_shared + a.n_own) + part.slot;
            a.part_ml[2 * p] = kLowest;
            a.part_ml[2 * p + 1] = 0.0f;
        }
        return;
    }
    if constexpr (RT == kSplitRows)
        if (part.is_shared)
        {
            if (walk_split<KS>(a, part, reinterpret_cast<bf16x8*>(lds), sh)) return;
            part.row_waves = 2;   // the same rows
        }
    constexpr bool kAll = RT == kSplitRows;   // shared parts alone: the own ones have a launch of their own
    if (kAll || (RT == 2 && (part.is_shared || a.own_wide))) walk<KS, MODE, 2>(a, part, sh);
    else if constexpr (!kAll) walk<KS, MODE, 1>(a, part, sh);
}

// In place of the factor of a range of l = 0, whose O is anything. A factor that underflows to 0 is one: a value of its
// range that is not finite makes O one that is not, as within a range.
constexpr float kNoRange = -1.0f;

// Joins the ranges of one row in order: blockIdx.x = sequence * q_heads + head. The ranges' factors go to LDS,
// then 2 or 4 groups of threads sum every 2nd or 4th range.
__global__ __launch_bounds__(256) void k_attn_paged_join(PagedArgs a)
{
    constexpr int kChunk = 256;
    __shared__ float w_s[kChunk];
    __shared__ float red[2][4];
    __shared__ float o_s[256];
    const size_t at = blockIdx.x;
    const unsigned b = (unsigned)(at / a.q_heads), h = (unsigned)(at % a.q_heads), n = a.n_shared + a.n_own;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, dim = a.c.dim;
    const int cols = dim <= 64 ? 64 : 128, groups = 256 / cols, d = t % cols, g = t / cols;
    const float* ml = a.part_ml + 2 * at * n;
    const float* po = a.part_o + at * n * dim + (d < dim ? d : 0);
    float m = kLowest, l = 0.0f, o = 0.0f;
    for (unsigned i = t; i < n; i += 256)
        if (ml[2 * i + 1] != 0.0f) m = fmax_std(m, ml[2 * i]);
    m = wave_max(m);
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmax_std(fmax_std(red[0][0], red[0][1]), fmax_std(red[0][2], red[0][3]));
    for (unsigned c = 0; c < n; c += kChunk)
    {
        float w = kNoRange;
        if (c + t < n)
        {
            const float li = ml[2 * (c + t) + 1];
            if (li != 0.0f)
            {
                w = __builtin_amdgcn_exp2f((ml[2 * (c + t)] - m) * kLog2e);
                l += li * w;
            }
        }
        __syncthreads();
        w_s[t] = w;
        __syncthreads();
        const int nc = min((int)(n - c), kChunk);
#pragma unroll 8
        for (int i = g; i < nc; i += groups)
        {
            const float x = po[(size_t)(c + i) * dim], f = w_s[i];
            o += f == kNoRange ? 0.0f : x * f;
        }
    }
    l = wave_sum(l);
    if (lane == 0) red[1][wave] = l;
    o_s[t] = o;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    if (t < dim)
    {
        o = 0.0f;
        for (int i = 0; i < groups; ++i) o += o_s[i * cols + t];
        a.O[(long)b * a.o_t + ((long)h * dim + t) * a.o_f] = l == 0.0f ? 0.0f : o / l;
    }
    if (t == 0 && a.m) a.m[at] = m;
    if (t == 0 && a.l) a.l[at] = l;
}

// The same for up to kFewParts ranges: a wave a row, everything it needs on its way at once. 4096 rows of 5 ranges take
// 6 us where the kernel above takes 11, 48 rows of 12 ranges 3.4 and 4.5; more ranges than 16 would need more registers
// than leave a SIMD 8 waves.
constexpr unsigned kFewParts = 16;
__global__ __launch_bounds__(256) void k_attn_paged_join_few(PagedArgs a)
{
    const unsigned at = blockIdx.x * 4 + threadIdx.x / 64, n = a.n_shared + a.n_own;
    if (at >= a.c.batch * a.q_heads) return;
    const int lane = threadIdx.x & 63, dim = a.c.dim;
    const unsigned b = at / a.q_heads, h = at - b * a.q_heads;
    const float2 own = reinterpret_cast<const float2*>(a.part_ml)[(size_t)at * n + min((unsigned)lane, n - 1)];
    const float* po = a.part_o + (size_t)at * n * dim;
    float x[kFewParts][2];
#pragma unroll
    for (unsigned i = 0; i < kFewParts; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y) x[i][y] = po[(size_t)min(i, n - 1) * dim + min(lane + 64 * y, dim - 1)];
    const bool any = lane < (int)n && own.y != 0.0f;
    const float m = wave_max(any ? own.x : kLowest), w = any ? __builtin_amdgcn_exp2f((own.x - m) * kLog2e) : kNoRange;
    const float l = wave_sum(any ? own.y * w : 0.0f);
    float o[2] = {0.0f, 0.0f};
#pragma unroll
    for (unsigned i = 0; i < kFewParts; ++i)
    {
        const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
#pragma unroll
        for (int y = 0; y < 2; ++y) o[y] += f == kNoRange ? 0.0f : x[i][y] * f;
    }
#pragma unroll
    for (int y = 0; y < 2; ++y)
    {
        const int d = lane + 64 * y;
        if (d < dim) a.O[(long)b * a.o_t + ((long)h * dim + d) * a.o_f] = l == 0.0f ? 0.0f : o[y] / l;
    }
    if (lane == 0 && a.m) a.m[at] = m;
    if (lane == 0 && a.l) a.l[at] = l;
}

struct PagedPlan
{
    int row_tiles, shared_row_waves, own_row_waves, own_wide;
    unsigned n_shared, n_own, shared_row_blocks, own_row_blocks;
    size_t shared_blocks, own_blocks;
    size_t parts() const { return (size_t)n_shared + n_own; }
};

// How a call is cut, from its sizes alone: the lengths are on the device.
PagedPlan paged_plan(const nnhip_kv_pages& c, size_t q_heads, size_t group, int mode, bool alpha_ok = true)
{
    PagedPlan p{};
    const size_t per = q_heads / c.heads, most = c.width * c.page, cus = device_cus();
    const size_t rows = group > 1 ? group * per : per;   // that read the same positions
    // More than 32 rows: bf16 parts. In float32 and so, over 16000 positions of 4 key heads: 128 wide 32 rows 37 us and
    // 40, 36 rows 44 and 41, 128 rows 67 and 53; 64 wide 32 rows 21 and 28, 36 rows 26 and 28, 128 rows 43 and 38.
    const bool split = group > 1 && rows > 32 && mode == kWhole && c.dim % 32 == 0 && alpha_ok;
    p.row_tiles = split ? kSplitRows : rows > kTile ? 2 : 1;
    p.own_wide = per > kTile;
    auto along_rows = [](size_t n, int tiles, int& waves) {
        const size_t need = (n + kTile * tiles - 1) / (kTile * tiles);
        waves = need > 2 ? 4 : need > 1 ? 2 : 1;
        return static_cast<unsigned>((need + waves - 1) / waves);
    };
    // Workgroups a CU: the streams of unshared sequences run best with 6 (attend of 24 sequences of 2500 to 5000:
    // 120 us with 2, 109 with 4, 103 with 6, 108 with 8). Ranges of shared positions cost a partial result of every
    // row, and a workgroup in bf16 parts has a CU to itself: 2 and 1. Beside shared positions the sequences' own are
    // few: 1, and 2 in the launch of their own that they have beside bf16 parts. A range has at least 64 positions,
    // one step of a workgroup's waves, and shared ones 128 once they fill the CUs (12 heads of 4 groups over 1000
    // positions: 13.4 us with 64, 11.5 with 128; of one group over 300: 7.1 and 8.0).
    auto ranges = [&](size_t others, size_t per_cu, bool long_ones = false) {
        const size_t least = long_ones && others * ((most + 63) / 64) > cus ? 128 : 64;
        const size_t want = (per_cu * cus + others - 1) / others, most_ranges = (most + least - 1) / least;
        return static_cast<unsigned>(want < most_ranges ? want : most_ranges);
    };
    auto blocks = [](size_t pieces, unsigned row_blocks) { return (pieces + 7) / 8 * 8 * row_blocks; };
    p.own_row_blocks = along_rows(per, p.own_wide ? 2 : 1, p.own_row_waves);
    const size_t own = c.batch * c.heads;
    p.n_own = ranges(own * p.own_row_blocks, group == 1 ? 6 : split ? 2 : 1);
    p.own_blocks = blocks(own * p.n_own, p.own_row_blocks);
    if (group > 1)
    {
        p.shared_row_blocks = along_rows(rows, p.row_tiles, p.shared_row_waves);
        if (split) p.shared_row_waves = 1, p.shared_row_blocks = static_cast<unsigned>((rows + kTile * kSplitRows - 1) / (kTile * kSplitRows));
        const size_t sh = c.batch / group * c.heads;
        p.n_shared = ranges(sh * p.shared_row_blocks, split ? 1 : 2, !split);
        p.shared_blocks = blocks(sh * p.n_shared, p.shared_row_blocks);
    }
    return p;
}

template <int KS, int MODE> void paged_launch(const PagedArgs& a, const PagedPlan& p, hipStream_t s)
{
    auto go = [&](auto kernel, PagedArgs args, size_t shared_blocks, size_t own_blocks) {
        args.shared_blocks = static_cast<unsigned>(shared_blocks);
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(shared_blocks + own_blocks)), dim3(256), 0, s, args);
    };
    if constexpr (MODE == kWhole && KS % 2 == 0)
        if (p.row_tiles == kSplitRows)
        {
            // In one launch the own parts would run at the one wave a SIMD that the bf16 parts' registers leave.
            go(k_attn_paged<KS, MODE, kSplitRows>, a, p.shared_blocks, 0);
            if (p.own_wide) go(k_attn_paged<KS, MODE, 2>, a, 0, p.own_blocks);
            else go(k_attn_paged<KS, MODE, 1>, a, 0, p.own_blocks);
            return;
        }
    if (p.row_tiles == 1) go(k_attn_paged<KS, MODE, 1>, a, p.shared_blocks, p.own_blocks);
    else go(k_attn_paged<KS, MODE, 2>, a, p.shared_blocks, p.own_blocks);
}

// m and l of every row and range, in whole 16 bytes.
size_t ml_floats(const nnhip_kv_pages& c, size_t q_heads, const PagedPlan& p)
{
    return (2 * c.batch * q_heads * p.parts() + 3) / 4 * 4;
}

int paged_mode(const nnhip_kv_pages& c)
{
    const bool vec = c.dim % 4 == 0 && c.row % 4 == 0 && aligned16(c.K) && aligned16(c.V);
    return !vec ? kSingle : c.dim % 16 == 0 ? kWhole : kCut;
}

size_t paged_workspace(const nnhip_kv_pages& c, size_t q_heads, const PagedPlan& p)
{
    return p.parts() == 1 ? 0 : (ml_floats(c, q_heads, p) + c.batch * q_heads * p.parts() * c.dim) * sizeof(float);
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
    // Enough for either way of the products, and without sharing.
    size_t most = 0;
    for (const int mode : {static_cast<int>(kWhole), static_cast<int>(kSingle)})
        for (const size_t g : {group, (size_t)1})
        {
            const size_t n = paged_workspace(*c, q_heads, paged_plan(*c, q_heads, g, mode));
            most = n > most ? n : most;
        }
    return most;
}

extern "C" int nnhip_attn_paged(const nnhip_kv_pages* c, const float* q, long q_t, long q_f, size_t q_heads,
                                const float* len, const float* shared, size_t group, const float* slopes, float alpha,
                                float* O, long o_t, long o_f, float* m, float* l, void* workspace,
                                size_t workspace_bytes, void* stream)
{
    if (!paged_ok(c, q_heads, group) || !q || !len || !O || q_t < 0 || q_f < 0 || o_t < 0 || o_f < 0 ||
        c->batch * q_heads > 0x7fffffffu)
        return -1;
    if (group == 1) shared = nullptr;   // a group of one has all positions to itself
    const int mode = paged_mode(*c);
    const PagedPlan p = paged_plan(*c, q_heads, shared ? group : 1, mode, __builtin_fabsf(alpha) >= 0x1p-64f);
    const size_t need = paged_workspace(*c, q_heads, p);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return -1;
    if (p.shared_blocks + p.own_blocks > kGridMost || (p.parts() > kFewParts && c->batch * q_heads > kGridMost)) return -1;
    auto* ws = static_cast<float*>(workspace);
    PagedArgs a{};
    a.c = pages_of(*c);
    a.q = q;
    a.q_t = q_t;
    a.q_f = q_f;
    a.len = len;
    a.shared = shared;
    a.slopes = slopes;
    a.O = O;
    a.o_t = o_t;
    a.o_f = o_f;
    a.m = m;
    a.l = l;
    a.part_ml = ws;
    a.q_heads = static_cast<unsigned>(q_heads);
    a.group = static_cast<unsigned>(group);
    a.n_shared = p.n_shared;
    a.n_own = p.n_own;
    a.shared_blocks = static_cast<unsigned>(p.shared_blocks);
    a.by_per = FastDiv(static_cast<unsigned>(q_heads / c->heads));
    a.by_heads = FastDiv(a.c.heads);
    a.by_shared_rows = FastDiv(8 * (shared ? p.shared_row_blocks : 1));
    a.by_own_rows = FastDiv(8 * p.own_row_blocks);
    a.by_n_shared = FastDiv(shared ? p.n_shared : 1);
    a.by_n_own = FastDiv(p.n_own);
    a.shared_row_waves = p.shared_row_waves;
    a.own_row_waves = p.own_row_waves;
    a.own_wide = p.own_wide;
    a.q_rows = q_f == 1 && q_t % 4 == 0 && aligned16(q);
    a.alpha = alpha;
    if (p.parts() > 1) a.part_o = ws + ml_floats(*c, q_heads, p);
    const size_t d = c->dim;
    auto s = static_cast<hipStream_t>(stream);
    // Whole groups have a kernel each; the others take the next even number of groups.
    const int ks = static_cast<int>((d + 15) / 16);
    switch (mode == kWhole ? ks : 8 * mode + (ks + 1) / 2)
    {
    case 1: paged_launch<1, kWhole>(a, p, s); break;
    case 2: paged_launch<2, kWhole>(a, p, s); break;
    case 3: paged_launch<3, kWhole>(a, p, s); break;
    case 4: paged_launch<4, kWhole>(a, p, s); break;
    case 5: paged_launch<5, kWhole>(a, p, s); break;
    case 6: paged_launch<6, kWhole>(a, p, s); break;
    case 7: paged_launch<7, kWhole>(a, p, s); break;
    case 8: paged_launch<8, kWhole>(a, p, s); break;
    case 9: paged_launch<2, kCut>(a, p, s); break;
    case 10: paged_launch<4, kCut>(a, p, s); break;
    case 11: paged_launch<6, kCut>(a, p, s); break;
    case 12: paged_launch<8, kCut>(a, p, s); break;
    case 17: paged_launch<2, kSingle>(a, p, s); break;
    case 18: paged_launch<4, kSingle>(a, p, s); break;
    case 19: paged_launch<6, kSingle>(a, p, s); break;
    default: paged_launch<8, kSingle>(a, p, s); break;
    }
    if (int rc = launch_status()) return rc;
    if (p.parts() > 1 && p.parts() <= kFewParts)
    {
        const unsigned blocks = static_cast<unsigned>((c->batch * q_heads + 3) / 4);
        hipLaunchKernelGGL(k_attn_paged_join_few, dim3(blocks), dim3(256), 0, s, a);
        return launch_status();
    }
    if (p.parts() > 1)
    {
        hipLaunchKernelGGL(k_attn_paged_join, dim3(static_cast<unsigned>(c->batch * q_heads)), dim3(256), 0, s, a);
        return launch_status();
    }
    return 0;
}
