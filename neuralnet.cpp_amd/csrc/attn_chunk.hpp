// attn_chunk.hpp — attention of chunks of new tokens: what its kernels share, and
// the float32 walk that every call can take.
#pragma once

#include "kv_pages.hpp"

namespace nnhip
{

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kTile = 16;          // positions and rows of a product
constexpr int kChunkMaxDim = 128;
constexpr int kNarrowRows = 32;   // of a sequence and key head that the kernels of few rows take at most

struct ChunkArgs
{
    Pages8 c;                        // a float32 cache: c.t.K, c.t.V
    const float *q, *start, *len, *slopes;
    long q_t, q_f;
    float* O;
    long o_t, o_f;
    float *m, *l;
    float *part_ml, *part_o;         // per (row, range): m and l; O unnormalised (result_of)
    float *wide_ml, *wide_o;         // in the joins: those of k_attn_chunk_wide's rows
    unsigned q_heads, tokens, most;
    unsigned ranges;                 // that the kernel cuts positions into
    int few_rows;                    // results are of kNarrowRows for each sequence and key head, not of every token and head
    unsigned result_step;            // from a token's results to the next one's
    int wide_from;                   // sequences of more rows are k_attn_chunk_wide's
    char* images;                    // its keys' and values' parts: `tiles` a piece, of the pieces (slot and key head)
    unsigned tiles, first_piece, pieces;   // that the launch is for
    int slots_by_batch;              // a slot a sequence
    FastDiv by_block_rows;           // its blocks of rows are numbered from first row / these on, plus, if block_seqs, the
    int block_seqs;                  // sequence's number
    FastDiv by_per, by_heads, by_q_heads, by_row_blocks, by_ranges;   // by_row_blocks: of k_attn_chunk_wide
    int q_rows;                      // queries lie a token a row, 16-byte aligned
    int vec;                         // the cache's rows can be read in pieces of 4 values
    int page4;                       // pages have a multiple of 4 rows
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
        const float scale = scale_or_nan((keys ? a.c.K_scale : a.c.V_scale)[(size_t)max(row, 0) * a.c.t.heads + h]);
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
    size_t results;         // the place of the first row's results of ranges
};
template <int KS> struct WalkShared
{
    float o[4][kTile][Geometry<KS>::DV + 4];
    float ml[4][kTile][2];
};

// The place of the results of a sequence's first row of a key head, and of token i's head qh of them.
__device__ __forceinline__ size_t results_of(const ChunkArgs& a, unsigned b, unsigned h, unsigned first)
{
    return a.few_rows ? ((size_t)b * a.c.t.heads + h) * kNarrowRows : (size_t)first * a.q_heads + h * a.by_per.d;
}
__device__ __forceinline__ size_t result_of(const ChunkArgs& a, size_t results, unsigned i, unsigned qh)
{
    return results + (size_t)i * a.result_step + qh;
}

// Where a row's results go: m, l and values d .. d + 3 of O, unnormalised. LOG2: m is a score times log2(e). The results of
// ranges that others form so (WIDE) are joined so: a score's product with log2(e) is rounded once, before the ranges part.
template <bool WIDE, bool LOG2>
__device__ __forceinline__ void put(const ChunkArgs& a, const Part& part, int row, int d, f32x4 o, float m, float l, bool stats)
{
    if (LOG2 && a.ranges == 1 && m != kLowest) m *= kLn2;
    if (WIDE && !LOG2 && a.ranges > 1 && m != kLowest) m *= kLog2e;
    const unsigned i = a.by_per.div(row), own = row - i * a.by_per.d, qh = part.h * a.by_per.d + own;
    const size_t n = part.chunk.first + i;
    const int dim = a.c.t.dim;
    if (a.ranges == 1)
    {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float* to = a.O + (long)n * a.o_t + (long)qh * dim * a.o_f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < dim) to[(long)(d + e) * a.o_f] = l == 0.0f ? 0.0f : o[e] * inv;
        if (stats && a.m) a.m[n * a.q_heads + qh] = m;
        if (stats && a.l) a.l[n * a.q_heads + qh] = l;
        return;
    }
    const size_t p = result_of(a, part.results, i, own) * a.ranges + part.slot;
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
template <int KS, bool WIDE>
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
            put<WIDE, false>(a, part, row, d, z, mm, ll, d == 0);
        }
    }
}

// One range of positions. row_waves of the 4 waves lie along the rows, RT tiles each; the others take 16 positions
// each in turn.
template <int BITS, int KS, bool VEC, int RT, bool WIDE>
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
        join_waves<KS, WIDE>(a, part, sh, w.m, w.l, w.o, part.first + i * kTile, rws, RT * kTile);
    }
}

// The positions of range `slot` of `ranges` for rows up to `last`: whole steps of `step` positions; empty ones are marked
// for the join and give false.
__device__ __forceinline__ bool cut_range(const ChunkArgs& a, Part& part, int rows_here, int step)
{
    const int last = min((int)part.first + rows_here, part.n_rows) - 1;
    const int hi = max(part.chunk.seen + (int)a.by_per.div(last), 0);
    const int steps = (hi + step - 1) / step;
    part.begin = (int)((long)steps * part.slot / a.ranges) * step;
    part.end = min(hi, (int)((long)steps * (part.slot + 1) / a.ranges) * step);
    if (part.begin < part.end || a.ranges == 1) return true;
    for (int row = part.first + threadIdx.x; row <= last; row += blockDim.x)
    {
        const unsigned i = a.by_per.div(row);
        const size_t p = result_of(a, part.results, i, row - i * a.by_per.d) * a.ranges + part.slot;
        a.part_ml[2 * p] = kLowest;
        a.part_ml[2 * p + 1] = 0.0f;
    }
    return false;
}

// A workgroup of the kernels of few rows: all rows of a sequence and key head, one range of positions in steps of `step`.
// False: nothing is left to do.
__device__ __forceinline__ bool narrow_part(const ChunkArgs& a, Part& part, int step)
{
    // The key heads of one range run on one XCD (workgroups go to the 8 in turn), one after another: neighbouring heads have
    // parts of the same lines, of a row's bytes up to 64 wide and of its scales. 48 sequences of 6000 positions, 8 heads of 64
    // bytes: 119 us with a piece's ranges side by side, 88 so.
    const unsigned y = blockIdx.x >> 3, group = a.by_heads.div(y), q = 8 * group + (blockIdx.x & 7);
    part.h = y - group * a.c.t.heads;
    part.b = a.by_ranges.div(q);
    part.slot = q - part.b * a.ranges;
    if (part.b >= a.c.t.batch) return false;
    part.chunk = chunk_of(a, part.b);
    part.n_rows = part.chunk.n * a.by_per.d;
    part.first = 0;
    part.results = results_of(a, part.b, part.h, part.chunk.first);
    return part.n_rows > 0 && part.n_rows <= a.wide_from && cut_range(a, part, part.n_rows, step);
}

// k_attn_chunk8 (bytes: what rows, heads and caches are aligned to, 4, 8 or 16), and k_attn_chunk_wide: their launches; rows
// of a workgroup.
void chunk8(const ChunkArgs& a, int bytes, unsigned blocks, hipStream_t s);
constexpr int kWideRows = 128;
size_t chunk_image_bytes(int bits, unsigned dim);
void chunk_parts(const ChunkArgs& a, int bits, unsigned pieces, unsigned blocks, hipStream_t s);
void chunk_wide(const ChunkArgs& a, int bits, unsigned blocks, hipStream_t s);

} // namespace nnhip
