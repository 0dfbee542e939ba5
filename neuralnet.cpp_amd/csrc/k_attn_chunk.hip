// k_attn_chunk.hip — attention of each sequence's new tokens against its paged
// keys and values, in float32 or as bytes with a scale a row and head:
//
//   s_j = alpha q . k_j - slope (p - j),  j <= p, the token's position,
//   m = max_j s_j,  l = sum_j exp(s_j - m),  O = sum_j exp(s_j - m) v_j / l.
//
// A sequence's rows are its (token, query head) pairs that read one key head. A
// workgroup takes a block of them and one range of the positions that its last
// token sees; where there are several ranges a second kernel joins them in
// order.
#include "kv_pages.hpp"

#include <algorithm>

namespace nnhip
{
namespace
{

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 16;          // positions and rows of a product
constexpr int kChunkMaxDim = 128;

struct ChunkArgs
{
    Pages8 c;                        // a float32 cache: c.t.K, c.t.V
    const float *q, *start, *len, *slopes;
    long q_t, q_f;
    float* O;
    long o_t, o_f;
    float *m, *l;
    float *part_ml, *part_o;         // per (token, head, range): m and l; O unnormalised
    unsigned q_heads, tokens, most, ranges;
    FastDiv by_per, by_heads, by_row_blocks, by_ranges;   // by_row_blocks: 8 of them
    int q_rows;                      // queries lie a token a row, 16-byte aligned
    int row_waves;
    float alpha;
};

// The tokens of sequence b: the first and how many; and the positions that the first of them sees.
struct Chunk
{
    unsigned first;
    int n, seen;
};
__device__ __forceinline__ Chunk chunk_of(const ChunkArgs& a, unsigned b)
{
    const int s0 = length_of(a.start[b], a.tokens), s1 = length_of(a.start[b + 1], a.tokens);
    const int len = length_of(a.len[b], (int)(a.c.t.width * a.c.t.page.d));
    Chunk r;
    r.first = s0;
    r.n = max(s1 - s0, 0);
    r.seen = len - r.n + 1;   // below 1 where the sequence is shorter than its chunk
    r.n = min(r.n, (int)a.most);
    return r;
}

// The last of `n` ascending things for which f holds, -1 where it holds for none: a wave together, 64 at a time.
template <class F> __device__ __forceinline__ int last_of(unsigned n, F&& f)
{
    const unsigned lane = threadIdx.x & 63;
    unsigned lo = 0, size = n;
    for (;;)
    {
        const unsigned step = (size + 63) / 64, i = lo + lane * step;
        const unsigned long long holds = __builtin_amdgcn_ballot_w64(i < lo + size && f(i));
        if (!holds) return -1;   // in the first pass alone
        const unsigned k = 63 - __builtin_clzll(holds), at = lo + k * step;
        if (step == 1) return (int)at;
        size = min(step, lo + size - at);
        lo = at;
    }
}

// KS: groups of 16 key dims. Value columns of a lane: 4 neighbouring ones of every 64 (2 of every 32 up to 32 dims and for
// 96); columns past dim are formed and dropped.
template <int KS> struct Geometry
{
    static constexpr int VW = KS % 4 == 0 ? 4 : 2;
    static constexpr int T = (KS + VW - 1) / VW;
    static constexpr int DV = 16 * VW * T;
};

// 16 positions, for the lane: its dims of one key, its value columns of four positions.
template <int KS> struct Tile
{
    using G = Geometry<KS>;
    f32x4 k[KS];
    float v[4][G::T][G::VW];
    int row[4];   // of the values' positions, -1: none
};

// N neighbouring values of a row's head, from d on; dims past the last are read as others of the head.
template <int BITS, bool VEC, int N>
__device__ __forceinline__ void load(const ChunkArgs& a, bool keys, int row, unsigned h, int d, float (&x)[N])
{
    const int dim = a.c.t.dim;
    const size_t at = (size_t)max(row, 0) * a.c.t.row + (size_t)h * dim;
    if constexpr (BITS == 32)
    {
        const float* p = (keys ? a.c.t.K : a.c.t.V) + at;
        if constexpr (VEC)
        {
            typedef float vec __attribute__((ext_vector_type(N)));
            const vec z = *reinterpret_cast<const vec*>(p + (d < dim ? d : 0));
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = z[e];
        }
        else
        {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = p[d + e < dim ? d + e : 0];
        }
    }
    else
    {
        const signed char* p = (keys ? a.c.K : a.c.V) + at;
        const float scale = (keys ? a.c.K_scale : a.c.V_scale)[(size_t)max(row, 0) * a.c.t.heads + h];
        if constexpr (VEC)
        {
            typedef signed char vec __attribute__((ext_vector_type(N)));
            const vec z = *reinterpret_cast<const vec*>(p + (d < dim ? d : 0));
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = (float)z[e] * scale;
        }
        else
        {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = (float)p[d + e < dim ? d + e : 0] * scale;
        }
    }
}

// Loads are issued whatever the positions are, from row 0 where there is none, so that no branch holds the next
// tile's loads back behind this one's.
template <int BITS, int KS, bool VEC>
__device__ __forceinline__ void load_keys(const ChunkArgs& a, int row, unsigned h, int lane, Tile<KS>& x)
{
    const int g = lane >> 4;
#pragma unroll
    for (int i = 0; i < KS; ++i)
    {
        float z[4];
        load<BITS, VEC, 4>(a, true, row, h, 16 * i + 4 * g, z);
        x.k[i] = f32x4{z[0], z[1], z[2], z[3]};
    }
}
template <int BITS, int KS, bool VEC>
__device__ __forceinline__ void load_values(const ChunkArgs& a, int row, unsigned h, int lane, Tile<KS>& x)
{
    using G = Geometry<KS>;
    const int j = lane & 15, g = lane >> 4;
#pragma unroll
    for (int r = 0; r < 4; ++r)
    {
        x.row[r] = __shfl(row, 4 * g + r, 64);
#pragma unroll
        for (int t = 0; t < G::T; ++t) load<BITS, VEC, G::VW>(a, false, x.row[r], h, 16 * G::VW * t + G::VW * j, x.v[r][t]);
    }
}

// A lane's row of each of a wave's row tiles: its query dims, how many positions it sees (0: it is none), the bias' slope,
// and the running softmax.
template <int KS> struct Row
{
    using G = Geometry<KS>;
    f32x4 q[KS];
    int seen;
    float slope;
    float m, l;   // l: of the lane's positions alone
    f32x4 o[G::T][G::VW];
};

// Dims past the last one are 0 in keys and queries.
template <int KS> __device__ __forceinline__ void cut(f32x4 (&x)[KS], int g, int dim)
{
    if (16 * KS == dim) return;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = 16 * i + 4 * g + e < dim ? x[i][e] : 0.0f;
}

template <int KS, int RT>
__device__ __forceinline__ void use_keys(const ChunkArgs& a, Tile<KS>& x, const Row<KS> (&rows)[RT], int g, f32x4 (&s)[RT])
{
    cut<KS>(x.k, g, a.c.t.dim);
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

// `all`: positions that every row of the wave sees.
template <int KS, int RT>
__device__ __forceinline__ void use_values(const ChunkArgs& a, Tile<KS>& x, f32x4 (&s)[RT], Row<KS> (&rows)[RT], int p0, int g,
                                           int all)
{
    using G = Geometry<KS>;
    const int least = min(min(x.row[0], x.row[1]), min(x.row[2], x.row[3]));
    if (__builtin_amdgcn_ballot_w64(least < 0))
    {
        // 0 times a NaN that lies there would be one.
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < G::T; ++t)
#pragma unroll
                for (int y = 0; y < G::VW; ++y) x.v[r][t][y] = x.row[r] < 0 ? 0.0f : x.v[r][t][y];
    }
    // So would it be for the rows that do not see a position that others do: these are taken one at a time then.
    bool apart = false;
    if (p0 + kTile > all)
    {
        bool odd = false;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < G::T; ++t)
#pragma unroll
                for (int y = 0; y < G::VW; ++y) odd |= !(fabsf(x.v[r][t][y]) <= kMaxF);
        apart = __builtin_amdgcn_ballot_w64(odd) != 0;
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        Row<KS>& w = rows[i];
        float top = kLowest;
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            const int p = p0 + 4 * g + r;
            float z = a.alpha * s[i][r];
            if (a.slopes) z -= w.slope * (float)(w.seen - 1 - p);
            s[i][r] = x.row[r] >= 0 && p < w.seen ? z : -__builtin_inff();
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
        if (__builtin_expect(apart, 0))
        {
            const int j = threadIdx.x & 15;
            for (int jj = 0; jj < kTile; ++jj)
            {
                const int seen = __shfl(w.seen, jj, 64);
#pragma unroll
                for (int t = 0; t < G::T; ++t)
#pragma unroll
                    for (int y = 0; y < G::VW; ++y)
                    {
                        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            o = __builtin_amdgcn_mfma_f32_16x16x4f32(p0 + 4 * g + r < seen ? x.v[r][t][y] : 0.0f, s[i][r], o, 0, 0, 0);
                        if (j == jj) w.o[t][y] += o;
                    }
            }
            continue;
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
    unsigned b, h, first;   // sequence, key head, first row
    Chunk chunk;
    int n_rows;             // of the sequence
    unsigned slot;          // range
    int begin, end;
};
template <int KS> struct WalkShared
{
    float o[4][kTile][Geometry<KS>::DV + 4];
    float ml[4][kTile][2];
};

// Where a row's results go: m, l and values d .. d + 3 of O, unnormalised.
__device__ __forceinline__ void put(const ChunkArgs& a, const Part& part, int row, int d, f32x4 o, float m, float l, bool stats)
{
    const unsigned i = a.by_per.div(row), qh = part.h * a.by_per.d + (row - i * a.by_per.d);
    const size_t n = part.chunk.first + i, at = n * a.q_heads + qh;
    const int dim = a.c.t.dim;
    if (a.ranges == 1)
    {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float* to = a.O + (long)n * a.o_t + (long)qh * dim * a.o_f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < dim) to[(long)(d + e) * a.o_f] = l == 0.0f ? 0.0f : o[e] * inv;
        if (stats && a.m) a.m[at] = m;
        if (stats && a.l) a.l[at] = l;
        return;
    }
    const size_t p = at * a.ranges + part.slot;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d + e < dim) a.part_o[p * dim + d + e] = o[e];
    if (stats)
    {
        a.part_ml[2 * p] = m;
        a.part_ml[2 * p + 1] = l;
    }
}

// The waves' results for 16 rows of each row wave (rows first + rv * apart on) are joined through LDS, in the order
// of their positions, and written: 16 threads a row, 4 neighbouring values at a time.
template <int KS>
__device__ __forceinline__ void join_waves(const ChunkArgs& a, const Part& part, WalkShared<KS>& sh, float m, float l,
                                           const f32x4 (&o)[Geometry<KS>::T][Geometry<KS>::VW], int first, int rws, int apart)
{
    using G = Geometry<KS>;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, j = lane & 15, g = lane >> 4;
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
        const int row = first + rv * apart + jr;
        if (row >= part.n_rows) break;
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
#pragma unroll
        for (int x = 0; x < (G::DV + 63) / 64; ++x)
        {
            const int d = 64 * x + 4 * (t & 15);
            if (d >= G::DV) continue;
            f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (any[k]) z += *reinterpret_cast<const f32x4*>(&sh.o[k][jr][d]) * f[k];
            put(a, part, row, d, z, mm, ll, d == 0);
        }
    }
}

// One range of positions. row_waves of the 4 waves lie along the rows, RT tiles each; the others take 16 positions
// each in turn.
template <int BITS, int KS, bool VEC, int RT>
__device__ __forceinline__ void walk(const ChunkArgs& a, const Part& part, int rws, WalkShared<KS>& sh)
{
    using G = Geometry<KS>;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, j = lane & 15, g = lane >> 4, dim = a.c.t.dim;
    const int kws = 4 / rws, rw = wave % rws, kw = wave / rws, step = kws * kTile;
    const int begin = part.begin, end = part.end;
    Row<KS> rows[RT];
    int all = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        Row<KS>& w = rows[i];
        const int row = part.first + (rw * RT + i) * kTile + j;
        const bool live = row < part.n_rows;
        const unsigned n = live ? a.by_per.div(row) : 0, qh = part.h * a.by_per.d + (live ? row - n * a.by_per.d : 0);
        w.seen = live ? max(part.chunk.seen + (int)n, 0) : 0;
        if (live) all = min(all, w.seen);
        w.slope = a.slopes && live ? a.slopes[qh] : 0.0f;
        w.m = kLowest;
        w.l = 0.0f;
#pragma unroll
        for (int x = 0; x < G::T; ++x)
#pragma unroll
            for (int y = 0; y < G::VW; ++y) w.o[x][y] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (begin >= end) continue;
        const float* qp = a.q + (long)(part.chunk.first + n) * a.q_t + (long)qh * dim * a.q_f;   // rows that are none are formed and dropped
#pragma unroll
        for (int x = 0; x < KS; ++x)
        {
            const int d = 16 * x + 4 * g;
            if (VEC && a.q_rows) w.q[x] = *reinterpret_cast<const f32x4*>(qp + (d < dim ? d : 0));
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) w.q[x][e] = qp[(long)(d + e < dim ? d + e : 0) * a.q_f];
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
            cut<KS>(rows[i].q, g, dim);
        }
        for (int o = 1; o < 16; o *= 2) all = min(all, __shfl_xor(all, o, 64));
        all = __builtin_amdgcn_readfirstlane(all);
        // Table entries are loaded two tiles ahead of their use, keys and values one.
        auto entry = [&](int p) { return a.c.t.entry_of(part.b, p + j); };
        auto row_at = [&](float e, int p) {
            const int r = a.c.t.row_in(e, p + j);
            return p + j < end ? r : -1;
        };
        const int p1 = begin + kw * kTile;
        float ahead = entry(p1 + step);
        Tile<KS> x;
        const int r0 = row_at(entry(p1), p1);
        load_keys<BITS, KS, VEC>(a, r0, part.h, lane, x);
        load_values<BITS, KS, VEC>(a, r0, part.h, lane, x);
        for (int p = p1; p < end; p += step)
        {
            f32x4 s[RT];
            use_keys<KS, RT>(a, x, rows, g, s);
            const float further = entry(p + 2 * step);
            const int r = row_at(ahead, p + step);
            load_keys<BITS, KS, VEC>(a, r, part.h, lane, x);
            __builtin_amdgcn_sched_barrier(0);
            use_values<KS, RT>(a, x, s, rows, p, g, all);
            __builtin_amdgcn_sched_barrier(0);
            load_values<BITS, KS, VEC>(a, r, part.h, lane, x);
            ahead = further;
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        Row<KS>& w = rows[i];
        w.l += __shfl_xor(w.l, 16, 64);
        w.l += __shfl_xor(w.l, 32, 64);
        join_waves<KS>(a, part, sh, w.m, w.l, w.o, part.first + i * kTile, rws, RT * kTile);
    }
}

// The positions of range `slot` of `ranges` for rows up to `last`: whole steps of `step` positions; empty ones are marked
// for the join and give false.
template <int STEP> __device__ __forceinline__ bool cut_range(const ChunkArgs& a, Part& part, int rows_here)
{
    const int last = min((int)part.first + rows_here, part.n_rows) - 1;
    const int hi = max(part.chunk.seen + (int)a.by_per.div(last), 0);
    const int steps = (hi + STEP - 1) / STEP;
    part.begin = (int)((long)steps * part.slot / a.ranges) * STEP;
    part.end = min(hi, (int)((long)steps * (part.slot + 1) / a.ranges) * STEP);
    if (part.begin < part.end || a.ranges == 1) return true;
    for (int row = part.first + threadIdx.x; row <= last; row += blockDim.x)
    {
        const unsigned i = a.by_per.div(row);
        const size_t at = (size_t)(part.chunk.first + i) * a.q_heads + part.h * a.by_per.d + (row - i * a.by_per.d);
        a.part_ml[2 * (at * a.ranges + part.slot)] = kLowest;
        a.part_ml[2 * (at * a.ranges + part.slot) + 1] = 0.0f;
    }
    return false;
}

template <int BITS, int KS, bool VEC, int RT> __global__ __launch_bounds__(256, VEC ? 2 : 1) void k_attn_chunk(ChunkArgs a)
{
    __shared__ WalkShared<KS> sh;
    Part part;
    // The blocks of rows that read the same keys and values run on one XCD (workgroups go to the 8 in turn), so that its
    // L2 holds them once; the pieces are padded to a multiple of 8.
    unsigned i = blockIdx.x;
    const unsigned eight = a.by_row_blocks.div(i), block = (i - eight * a.by_row_blocks.d) / 8;
    i = eight * 8 + i % 8;
    unsigned next = a.by_ranges.div(i);
    part.slot = i - next * a.ranges;
    part.b = a.by_heads.div(next);
    part.h = next - part.b * a.c.t.heads;
    if (part.b >= a.c.t.batch) return;
    part.chunk = chunk_of(a, part.b);
    part.n_rows = part.chunk.n * a.by_per.d;
    const int rows_here = kTile * RT * a.row_waves;
    part.first = block * rows_here;
    if ((int)part.first >= part.n_rows || !cut_range<4 * kTile>(a, part, rows_here)) return;
    walk<BITS, KS, VEC, RT>(a, part, a.row_waves, sh);
}

// In place of the factor of a range of l = 0, whose O is anything. A factor that underflows to 0 is one: a value of its
// range that is not finite makes O one that is not, as within a range.
constexpr float kNoRange = -1.0f;

// Joins the ranges of a row in order: a wave a row.
__global__ __launch_bounds__(256) void k_attn_chunk_join(ChunkArgs a)
{
    const unsigned at = blockIdx.x * 4 + threadIdx.x / 64;
    const unsigned n = at / a.q_heads, h = at - n * a.q_heads;
    if (n >= a.tokens) return;
    const int lane = threadIdx.x & 63, dim = a.c.t.dim;
    const int b = last_of(a.c.t.batch, [&](unsigned i) { return length_of(a.start[i], a.tokens) <= (int)n; });
    if (b < 0) return;
    const Chunk c = chunk_of(a, b);
    if (n >= c.first + c.n) return;   // no sequence's
    const float* ml = a.part_ml + 2 * (size_t)at * a.ranges;
    const float* po = a.part_o + (size_t)at * a.ranges * dim;
    float m = kLowest, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (unsigned i = lane; i < a.ranges; i += 64)
        if (ml[2 * i + 1] != 0.0f) m = fmax_std(m, ml[2 * i]);
    m = wave_max(m);
    for (unsigned c0 = 0; c0 < a.ranges; c0 += 64)
    {
        float w = kNoRange;
        if (c0 + lane < a.ranges && ml[2 * (c0 + lane) + 1] != 0.0f)
        {
            w = __builtin_amdgcn_exp2f((ml[2 * (c0 + lane)] - m) * kLog2e);
            l += ml[2 * (c0 + lane) + 1] * w;
        }
        const int nc = min(a.ranges - c0, 64u);
        for (int i = 0; i < nc; ++i)
        {
            const float f = __shfl(w, i, 64);
#pragma unroll
            for (int y = 0; y < 2; ++y)
            {
                const float x = po[(size_t)(c0 + i) * dim + min(lane + 64 * y, dim - 1)];
                o[y] += f == kNoRange ? 0.0f : x * f;
            }
        }
    }
    l = wave_sum(l);
#pragma unroll
    for (int y = 0; y < 2; ++y)
    {
        const int d = lane + 64 * y;
        if (d < dim) a.O[(long)n * a.o_t + ((long)h * dim + d) * a.o_f] = l == 0.0f ? 0.0f : o[y] / l;
    }
    if (lane == 0 && a.m) a.m[at] = m;
    if (lane == 0 && a.l) a.l[at] = l;
}

// A call's sizes, whichever cache it is over.
struct ChunkCall
{
    Pages8 c;
    int bits;
    bool vec;          // rows can be read in pieces of 4 values
    size_t q_heads, tokens, most;
};

struct ChunkPlan
{
    int row_tiles, row_waves;
    unsigned row_blocks, ranges;
    size_t blocks;
};

// How a call is cut, from its sizes alone: the lengths are on the device.
ChunkPlan chunk_plan(const ChunkCall& c)
{
    ChunkPlan p{};
    const size_t per = c.q_heads / c.c.t.heads, rows = c.most * per, positions = (size_t)c.c.t.width * c.c.t.page.d, cus = device_cus();
    p.row_tiles = rows > kTile ? 2 : 1;
    const size_t need = (rows + kTile * p.row_tiles - 1) / (kTile * p.row_tiles);
    p.row_waves = need > 2 ? 4 : need > 1 ? 2 : 1;
    p.row_blocks = static_cast<unsigned>((need + p.row_waves - 1) / p.row_waves);
    const size_t others = c.c.t.heads * std::min<size_t>((size_t)c.c.t.batch * p.row_blocks, c.c.t.batch + c.tokens * per / (kTile * p.row_tiles * p.row_waves));
    const size_t want = (4 * cus + others - 1) / others, most_ranges = (positions + 63) / 64;
    p.ranges = static_cast<unsigned>(std::min<size_t>(std::min(want, most_ranges), 256));
    p.blocks = ((size_t)c.c.t.batch * c.c.t.heads * p.ranges + 7) / 8 * 8 * p.row_blocks;
    return p;
}

// m and l of every row and range, in whole 16 bytes.
size_t ml_floats(const ChunkCall& c, const ChunkPlan& p) { return (2 * c.tokens * c.q_heads * p.ranges + 3) / 4 * 4; }
size_t chunk_workspace(const ChunkCall& c, const ChunkPlan& p)
{
    return p.ranges == 1 ? 0 : (ml_floats(c, p) + c.tokens * c.q_heads * p.ranges * c.c.t.dim) * sizeof(float);
}

bool chunk_ok(const ChunkCall& c, size_t heads)
{
    return c.q_heads > 0 && c.q_heads % heads == 0 && c.q_heads <= kMaxIndex && c.tokens > 0 && c.tokens <= kMaxIndex && c.most > 0 &&
           c.most <= c.tokens && c.tokens * c.q_heads < (size_t)0x80000000u;
}
bool chunk_call(const nnhip_kv_pages* c, size_t q_heads, size_t tokens, size_t most, ChunkCall& out)
{
    if (!pages_ok(c, kChunkMaxDim)) return false;
    out = {Pages8{pages_of(*c), nullptr, nullptr, nullptr, nullptr}, 32, c->dim % 4 == 0 && c->row % 4 == 0 && aligned16(c->K) && aligned16(c->V),
           q_heads, tokens, most};
    return chunk_ok(out, c->heads);
}
bool chunk_call(const nnhip_kv8_pages* c, size_t q_heads, size_t tokens, size_t most, ChunkCall& out)
{
    if (!pages8_ok(c, kChunkMaxDim)) return false;
    out = {pages8_of(*c), 8, c->dim % 4 == 0 && c->row % 4 == 0 && ((reinterpret_cast<uintptr_t>(c->K) | reinterpret_cast<uintptr_t>(c->V)) & 3) == 0,
           q_heads, tokens, most};
    return chunk_ok(out, c->heads);
}

template <int BITS, int KS, bool VEC> void chunk_launch(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s)
{
    const dim3 grid(static_cast<unsigned>(p.blocks));
    if (p.row_tiles == 1) hipLaunchKernelGGL((k_attn_chunk<BITS, KS, VEC, 1>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_attn_chunk<BITS, KS, VEC, 2>), grid, dim3(256), 0, s, a);
}
template <int BITS, bool VEC> void chunk_launch(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s)
{
    switch ((a.c.t.dim + 31) / 32)
    {
    case 1: chunk_launch<BITS, 2, VEC>(a, p, s); break;
    case 2: chunk_launch<BITS, 4, VEC>(a, p, s); break;
    case 3: chunk_launch<BITS, 6, VEC>(a, p, s); break;
    default: chunk_launch<BITS, 8, VEC>(a, p, s); break;
    }
}

template <class C> size_t chunk_bytes(const C* c, size_t q_heads, size_t tokens, size_t most)
{
    ChunkCall call;
    return chunk_call(c, q_heads, tokens, most, call) ? chunk_workspace(call, chunk_plan(call)) : 0;
}

template <class C>
int attn_chunk(const C* c, const float* q, long q_t, long q_f, size_t q_heads, size_t tokens, const float* start, size_t most,
               const float* len, const float* slopes, float alpha, float* O, long o_t, long o_f, float* m, float* l, void* workspace,
               size_t workspace_bytes, void* stream)
{
    ChunkCall call;
    if (!chunk_call(c, q_heads, tokens, most, call) || !q || !start || !len || !O || q_t < 0 || q_f < 0 || o_t < 0 || o_f < 0) return -1;
    const ChunkPlan p = chunk_plan(call);
    const size_t need = chunk_workspace(call, p);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return -1;
    if (p.blocks > kGridMost || tokens * q_heads / 4 + 1 > kGridMost) return -1;
    auto* ws = static_cast<float*>(workspace);
    ChunkArgs a{};
    a.c = call.c;
    a.q = q;
    a.q_t = q_t;
    a.q_f = q_f;
    a.start = start;
    a.len = len;
    a.slopes = slopes;
    a.O = O;
    a.o_t = o_t;
    a.o_f = o_f;
    a.m = m;
    a.l = l;
    a.part_ml = ws;
    if (p.ranges > 1) a.part_o = ws + ml_floats(call, p);
    a.q_heads = static_cast<unsigned>(q_heads);
    a.tokens = static_cast<unsigned>(tokens);
    a.most = static_cast<unsigned>(most);
    a.ranges = p.ranges;
    a.by_per = FastDiv(static_cast<unsigned>(q_heads / c->heads));
    a.by_heads = FastDiv(call.c.t.heads);
    a.by_row_blocks = FastDiv(8 * p.row_blocks);
    a.by_ranges = FastDiv(p.ranges);
    a.q_rows = q_f == 1 && q_t % 4 == 0 && aligned16(q) && c->dim % 4 == 0;
    a.row_waves = p.row_waves;
    a.alpha = alpha;
    auto s = static_cast<hipStream_t>(stream);
    if (call.bits == 32) call.vec ? chunk_launch<32, true>(a, p, s) : chunk_launch<32, false>(a, p, s);
    else call.vec ? chunk_launch<8, true>(a, p, s) : chunk_launch<8, false>(a, p, s);
    if (int rc = launch_status()) return rc;
    if (p.ranges == 1) return 0;
    hipLaunchKernelGGL(k_attn_chunk_join, dim3(static_cast<unsigned>((tokens * q_heads + 3) / 4)), dim3(256), 0, s, a);
    return launch_status();
}

} // namespace
} // namespace nnhip

using namespace nnhip;

extern "C" size_t nnhip_attn_chunk_workspace_bytes(const nnhip_kv_pages* c, size_t q_heads, size_t tokens, size_t most)
{
    return chunk_bytes(c, q_heads, tokens, most);
}
extern "C" size_t nnhip_attn_chunk8_workspace_bytes(const nnhip_kv8_pages* c, size_t q_heads, size_t tokens, size_t most)
{
    return chunk_bytes(c, q_heads, tokens, most);
}
extern "C" int nnhip_attn_chunk(const nnhip_kv_pages* c, const float* q, long q_t, long q_f, size_t q_heads, size_t tokens,
                                const float* start, size_t most, const float* len, const float* slopes, float alpha, float* O, long o_t,
                                long o_f, float* m, float* l, void* workspace, size_t workspace_bytes, void* stream)
{
    return attn_chunk(c, q, q_t, q_f, q_heads, tokens, start, most, len, slopes, alpha, O, o_t, o_f, m, l, workspace, workspace_bytes, stream);
}
extern "C" int nnhip_attn_chunk8(const nnhip_kv8_pages* c, const float* q, long q_t, long q_f, size_t q_heads, size_t tokens,
                                 const float* start, size_t most, const float* len, const float* slopes, float alpha, float* O, long o_t,
                                 long o_f, float* m, float* l, void* workspace, size_t workspace_bytes, void* stream)
{
    return attn_chunk(c, q, q_t, q_f, q_heads, tokens, start, most, len, slopes, alpha, O, o_t, o_f, m, l, workspace, workspace_bytes, stream);
}
