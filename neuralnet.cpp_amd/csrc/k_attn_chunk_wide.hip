// k_attn_chunk_wide.hip — chunk attention of sequences with many rows: both
// products on the float16 matrix cores, from parts (f16_parts.hpp): three float16
// products for a float32 one, two over an 8-bit cache.
//
// k_attn_chunk_parts forms the parts of 32 positions of a key head at a time, once
// for all of its blocks of rows, in the order of the matrix cores' operands. It
// reads the cache and writes as much again (2048 tokens behind 6000, 8 heads of
// 128: 24 us), and takes the scaling, the rounding and the pages' table out of the
// loop below, of whose vector instructions they were two thirds: with parts formed
// by every block of 128 rows the call took 951 us, so 712, and 8 sequences of 192
// rows a key head behind 2000 positions 200 and 181.
//
// Scales are exact: a key's goes into its scores, a value's into its position's
// weights, relative to the largest such product that the row has met (a row's
// outputs are rescaled when that grows, and as it shrinks with a growing score).
// So what a row does not see, and what has next to no weight, takes no accuracy
// from the rest.
//
// A workgroup of k_attn_chunk_wide takes 128 rows, 32 to a wave, and 32 positions at
// a time, copied to LDS a tile ahead. Both products are formed transposed (S^T = K
// Q^T, O^T = V^T P^T), 32 x 32 x 16 at a time: lane l has the scores of row l % 32
// and of the positions 8 (r / 4) + 4 (l / 32) + r % 4, r < 16, and its weights are
// the second product's operand as they lie, if its k index 8 (l / 32) + e of step t
// stands for position 8 (2 t + e / 4) + 4 (l / 32) + e % 4.
//
// What bounds it, 2048 tokens behind 6000 of 32 heads: with 128 dims the matrix
// cores are busy for 53 % of the cycles and the vector instructions of the softmax
// and of the weights' parts (some 200 a tile and wave, 16 of them exponentials, at a
// quarter of the rate) for 41 %, and as the clock falls under both (1.8 GHz) two
// waves a SIMD hardly hide one behind the other. There no order of reads, products
// and priorities changed it by 2 %; four waves of 64 rows each, with half the reads
// from LDS, ran 1503 us. Heads of 32, 64 and 128 take 301, 426 and 732 us (and up to
// 10 % more on other cards); up to 64 it is the float32 walk below that takes the
// registers of a third wave (245 to 256, 163 to 167 without it). Over 8 bits, 16
// heads of 80, the matrix cores are busy for 33 % and the vector instructions, as
// many beside 22 products a tile instead of 48, for 49 %.
//
// Of a float32 cache, results that are not finite are formed again by the float32
// walk: infinities and NaN among keys, queries and values, also at positions
// that some of the rows do not see.
#include "attn_chunk.hpp"
#include "f16_parts.hpp"

#include <cstddef>
#include <type_traits>

namespace nnhip
{
namespace
{

constexpr int kPos = 32;      // positions of a tile

__device__ __forceinline__ floatx16 mfma32(const half8& x, const half8& y, const floatx16& c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
}

// A tile's parts, of one key head of up to 16 KS dims.
template <int BITS, int KS> struct alignas(16) Image
{
    static constexpr int P = BITS == 32 ? 2 : 1;   // parts
    static constexpr int NB = (KS + 1) / 2;        // blocks of 32 value dims
    // Operands by lane: [step or block of 32 dims and k step][part][lane's place]
    half8 k[KS][P][64];
    half8 v[NB][2][P][64];
    float k_scale[kPos];           // of the scores, times 2^-shift
    float v_scale[kPos];           // of the weights: the values' scales; BITS 32: a quarter of 2^(exponent of the position's values)
    int there[4];                  // [0]: which positions exist; [1]: the keys' shift (shift_of)
};

// What a thread of k_attn_chunk_parts holds of a tile. Keys: 8 dims of one position each; values: VD dims of the 8 positions of
// the wave's group.
template <int BITS, int KS> struct Raw
{
    static constexpr int CP = KS <= 2 ? 4 : KS <= 4 ? 8 : 16;                  // pieces of 8 dims of a row, rounded up to 2^n
    static constexpr int KI = kPos * CP / 256 > 0 ? kPos * CP / 256 : 1;       // pieces of a thread
    static constexpr int VD = KS > 4 ? 2 : 1;
    float k[KI][BITS == 32 ? 8 : 2], v[8][BITS == 32 ? VD : 1];
    float scale;                   // BITS 8: lane p < 32 position p's key scale, lane 32 + p its value scale
};

template <int BITS, int KS> struct Wide
{
    using R = Raw<BITS, KS>;
    using S = Image<BITS, KS>;
    static constexpr int P = S::P, NB = S::NB;

    const ChunkArgs& a;
    const Part& part;
    int t, lane, wave;

    // Whether this thread has piece i of the keys, of which position, and its first dim.
    __device__ __forceinline__ bool piece(int i, int& p, int& d) const
    {
        const int item = t + 256 * i;
        p = item / R::CP;
        d = 8 * (item % R::CP);
        return p < kPos && d < 16 * KS;
    }
    // Position e of the wave's group of values.
    __device__ __forceinline__ int value_pos(int e) const { return 8 * (2 * (wave >> 1) + e / 4) + 4 * (wave & 1) + e % 4; }

    // row: of position lane % 32, -1 where there is none. key_rows: those of the thread's pieces.
    __device__ __forceinline__ void key_rows(int row, int (&kr)[R::KI]) const
    {
#pragma unroll
        for (int i = 0; i < R::KI; ++i)
        {
            int p, d;
            piece(i, p, d);
            kr[i] = max(__shfl(row, p & 31, 64), 0);
        }
    }
    __device__ __forceinline__ void load(int row, const int (&kr)[R::KI], R& r) const
    {
        const int dim = a.c.t.dim;
        const bool vec = a.vec;
#pragma unroll
        for (int i = 0; i < R::KI; ++i)
        {
            int p, d;
            piece(i, p, d);
            const size_t at = (size_t)kr[i] * a.c.t.row + (size_t)part.h * dim;
            if constexpr (BITS == 32)
            {
                const float* from = a.c.t.K + at;
                if (vec)
                {
                    const f32x4 lo = *reinterpret_cast<const f32x4*>(from + (d < dim ? d : 0));
                    const f32x4 hi = *reinterpret_cast<const f32x4*>(from + (d + 4 < dim ? d + 4 : 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) r.k[i][e] = lo[e], r.k[i][4 + e] = hi[e];
                }
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) r.k[i][e] = from[d + e < dim ? d + e : 0];
            }
            else
            {
                const signed char* from = a.c.K + at;
                if (vec)
                {
                    r.k[i][0] = *reinterpret_cast<const float*>(from + (d < dim ? d : 0));
                    r.k[i][1] = *reinterpret_cast<const float*>(from + (d + 4 < dim ? d + 4 : 0));
                }
                else
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                    {
                        unsigned z = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) z |= (unsigned)(unsigned char)from[d + 4 * w + e < dim ? d + 4 * w + e : 0] << (8 * e);
                        r.k[i][w] = __builtin_bit_cast(float, z);
                    }
            }
        }
        const int d = R::VD * lane;
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            const int vr = max(__builtin_amdgcn_readlane(row, value_pos(e)), 0);
            const size_t at = (size_t)vr * a.c.t.row + (size_t)part.h * dim;
            if constexpr (BITS == 32)
            {
                const float* from = a.c.t.V + at;
                if (R::VD == 2 && vec)
                {
                    const floatx2 z = *reinterpret_cast<const floatx2*>(from + (d < dim ? d : 0));
                    r.v[e][0] = z[0];
                    r.v[e][R::VD - 1] = z[1];
                }
                else
#pragma unroll
                    for (int y = 0; y < R::VD; ++y) r.v[e][y] = from[d + y < dim ? d + y : 0];
            }
            else
            {
                const signed char* from = a.c.V + at;
                unsigned z;
                if (R::VD == 2 && vec) z = *reinterpret_cast<const unsigned short*>(from + (d < dim ? d : 0));
                else
                {
                    z = (unsigned char)from[d < dim ? d : 0];
                    if constexpr (R::VD == 2) z |= (unsigned)(unsigned char)from[d + 1 < dim ? d + 1 : 0] << 8;
                }
                r.v[e][0] = __builtin_bit_cast(float, z);
            }
        }
        if constexpr (BITS == 8)
        {
            const float* from = lane < 32 ? a.c.K_scale : a.c.V_scale;
            r.scale = from[(size_t)max(row, 0) * a.c.t.heads + part.h];
        }
    }

    // The tile's parts; there: which of its positions exist. Absent ones, and dims past the last, are 0.
    __device__ __forceinline__ void stage(const R& r, S& sh, unsigned there)
    {
        const int dim = a.c.t.dim;
        const bool whole = there == 0xffffffffu && dim == 32 * NB;
#pragma unroll
        for (int i = 0; i < R::KI; ++i)
        {
            int p, d;
            const bool mine = piece(i, p, d);
            const bool ok = there >> (p & 31) & 1;
            const int step = d / 16, h = d / 8 % 2, place = (p + 32 * h) ^ ((2 * step + h) & 7);
            if constexpr (BITS == 32)
            {
                floatx8 z;
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = r.k[i][e];
                if (!whole)
                {
                    asm volatile("");   // stays a branch
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[e] = ok && d + e < dim ? z[e] : 0.0f;
                }
                float top = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(z[e]));
                top = max_of<R::CP>(top);
                const int ke = top > 0.0f ? exponent_of(top) : kNone;
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = __builtin_ldexpf(z[e], 15 - ke);
                half8 hi, lo;
                split2(z, hi, lo);
                if (mine)
                {
                    sh.k[step][0][place] = hi;
                    sh.k[step][P - 1][place] = lo;
                    if (d == 0) sh.k_scale[p] = __builtin_ldexpf(1.0f, ke - 20);
                }
            }
            else
            {
                uintx4 z;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                {
                    unsigned x = __builtin_bit_cast(unsigned, r.k[i][w]);
                    x = ok ? x : 0u;
                    if (d + 4 * w + 4 > dim) x = d + 4 * w >= dim ? 0u : x & (0xffffffffu >> 8 * (d + 4 * w + 4 - dim));
                    z[2 * w] = halves_of(__builtin_amdgcn_perm(0u, x, 0x0c010c00u));
                    z[2 * w + 1] = halves_of(__builtin_amdgcn_perm(0u, x, 0x0c030c02u));
                }
                if (mine) sh.k[step][0][place] = __builtin_bit_cast(half8, z);
            }
        }
        {
            const int group = wave;   // k step group >> 1, half group & 1
            const int d0 = R::VD * lane;
            unsigned ok = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) ok |= (there >> value_pos(e) & 1u) << e;
            floatx8 z[R::VD];
            int ve[8] = {};
            if constexpr (BITS == 32)
            {
#pragma unroll
                for (int y = 0; y < R::VD; ++y)
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[y][e] = r.v[e][y];
                if (!whole)
                {
                    asm volatile("");
#pragma unroll
                    for (int y = 0; y < R::VD; ++y)
#pragma unroll
                        for (int e = 0; e < 8; ++e) z[y][e] = (ok >> e & 1) && d0 + y < dim ? z[y][e] : 0.0f;
                }
                float top[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    top[e] = fabsf(z[0][e]);
                    if constexpr (R::VD == 2) top[e] = fmaxf(top[e], fabsf(z[R::VD - 1][e]));
                }
                const float mine = max_of_8(top, lane);   // position lane % 8's
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), e));
                    ve[e] = x > 0.0f ? exponent_of(x) : kNone;
                }
                if (lane < 8) sh.v_scale[value_pos(lane)] = mine > 0.0f ? __builtin_ldexpf(0.25f, exponent_of(mine)) : 0.0f;
            }
#pragma unroll
            for (int y = 0; y < R::VD; ++y)
            {
                const int d = d0 + y;
                if (d >= 32 * NB) continue;
                const int slot = d % 32 + 32 * (group & 1), place = slot ^ (slot >> 3 & 7);
                half8(&to)[P][64] = sh.v[d / 32][group >> 1];
                if constexpr (BITS == 32)
                {
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[y][e] = __builtin_ldexpf(z[y][e], 15 - ve[e]);
                    half8 hi, lo;
                    split2(z[y], hi, lo);
                    to[0][place] = hi;
                    to[P - 1][place] = lo;
                }
                else
                {
                    uintx4 x;
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                    {
                        const unsigned lo = (ok >> e & 1) && d < dim ? __builtin_bit_cast(unsigned, r.v[e][0]) : 0u;
                        const unsigned hi = (ok >> (e + 1) & 1) && d < dim ? __builtin_bit_cast(unsigned, r.v[e + 1][0]) : 0u;
                        x[e / 2] = halves_of(__builtin_amdgcn_perm(hi, lo, y == 0 ? 0x0c040c00u : 0x0c050c01u));
                    }
                    to[0][place] = __builtin_bit_cast(half8, x);
                }
            }
        }
        if constexpr (BITS == 8)
            if (wave == 0)
            {
                const bool ok = there >> (lane & 31) & 1;
                const float s = ok ? scale_or_nan(r.scale) : 0.0f;
                if (lane < 32) sh.k_scale[lane] = s;
                else sh.v_scale[lane - 32] = s;
            }
    }
};

// The place of a sequence among those whose parts are formed: its own number, or, as these have more than kNarrowRows rows
// each, its first row's share of them.
__device__ __forceinline__ unsigned slot_of(const ChunkArgs& a, unsigned b)
{
    if (a.slots_by_batch) return b;
    return (unsigned)((size_t)length_of(a.start[b], a.tokens) * a.by_per.d / (kNarrowRows + 1));
}

// The parts of every tile, once for all blocks of rows, of the pieces (slot and key head) from a.first_piece on. blocks:
// workgroups of a piece.
template <int BITS, int KS> __global__ __launch_bounds__(256) void k_attn_chunk_parts(ChunkArgs a, FastDiv blocks)
{
    using W = Wide<BITS, KS>;
    using S = Image<BITS, KS>;
    __shared__ S sh;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31;
    Part part{};
    const unsigned piece = blocks.div(blockIdx.x), first = blockIdx.x - piece * blocks.d;
    const unsigned slot = a.by_heads.div(a.first_piece + piece);
    part.h = a.first_piece + piece - slot * a.c.t.heads;
    int b = slot;
    if (!a.slots_by_batch)
    {
        b = last_of(a.c.t.batch, [&](unsigned i) { return slot_of(a, i) <= slot; });
        if (b < 0 || slot_of(a, b) != slot) return;
    }
    part.b = b;
    part.chunk = chunk_of(a, part.b);
    if (part.chunk.n * (int)a.by_per.d <= a.wide_from) return;
    const int end = max(part.chunk.seen + part.chunk.n - 1, 0), tiles = (end + kPos - 1) / kPos;
    W w{a, part, t, lane, wave};
    S* to = reinterpret_cast<S*>(a.images) + (size_t)piece * a.tiles;
    for (int i = first; i < tiles; i += blocks.d)
    {
        const int p = kPos * i + j;
        int row = a.c.t.row_in(a.c.t.entry_of(part.b, p), p);
        if (p >= end) row = -1;
        int kr[W::R::KI];
        typename W::R raw;
        w.key_rows(row, kr);
        w.load(row, kr, raw);
        const unsigned there = (unsigned)__builtin_amdgcn_ballot_w64(row >= 0);
        w.stage(raw, sh, there);
        if (t < 4) sh.there[t] = there;
        __syncthreads();
        const float size = fabsf(sh.k_scale[j]);
        const int shift = shift_of(__builtin_amdgcn_ballot_w64(size > kFar),
                                   !__builtin_amdgcn_ballot_w64(size >= kNear) && __builtin_amdgcn_ballot_w64(size > 0.0f));
        const f32x4* from = reinterpret_cast<const f32x4*>(&sh);
        f32x4* out = reinterpret_cast<f32x4*>(to + i);
        constexpr int kScales = offsetof(S, k_scale) / 16, kThere = offsetof(S, there) / 16;
        for (int x = t; x < (int)(sizeof(S) / 16); x += 256)
        {
            f32x4 z = from[x];
            if (x == kThere) z[1] = __builtin_bit_cast(float, shift);
            if (shift != 0 && x >= kScales && x < kScales + kPos / 4)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = __builtin_ldexpf(z[e], -shift);
            out[x] = z;
        }
        __syncthreads();
    }
}

template <int BITS, int KS> __global__ __launch_bounds__(256, 2) void k_attn_chunk_wide(ChunkArgs a)
{
    using S = Image<BITS, KS>;
    constexpr int NB = S::NB, P = S::P;
    constexpr size_t kLds = BITS == 32 && sizeof(WalkShared<KS>) > 2 * sizeof(S) ? sizeof(WalkShared<KS>) : 2 * sizeof(S);
    __shared__ __attribute__((aligned(16))) char lds[kLds];
    S* const sh = reinterpret_cast<S*>(lds);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, g = lane >> 5;
    Part part;
    const S* images;
    // Workgroups go to the 8 XCDs in turn: each takes neighbouring pieces of work, the blocks of rows of one range of one key
    // head after another (they read the same keys and values), the rows that see most first.
    {
        const unsigned each = gridDim.x / 8, at = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
        const unsigned piece = a.by_row_blocks.div(at);
        const unsigned x = a.by_row_blocks.d - 1 - (at - piece * a.by_row_blocks.d);
        part.h = a.by_ranges.div(piece);
        part.slot = piece - part.h * a.ranges;
        if (part.h >= a.c.t.heads) return;
        // At least as many numbers as a sequence of more than kNarrowRows rows has blocks: first row / 128 + its own number,
        // or first row / (kNarrowRows + 1).
        auto base = [&](unsigned b) { return a.by_block_rows.div(length_of(a.start[b], a.tokens) * a.by_per.d) + (a.block_seqs ? b : 0); };
        const int b = last_of(a.c.t.batch, [&](unsigned i) { return base(i) <= x; });
        if (b < 0) return;
        part.b = b;
        part.chunk = chunk_of(a, part.b);
        part.n_rows = part.chunk.n * a.by_per.d;
        const unsigned block = x - base(b);
        const unsigned at_piece = slot_of(a, part.b) * a.c.t.heads + part.h - a.first_piece;
        if (part.n_rows <= a.wide_from || at_piece >= a.pieces || block >= (unsigned)(part.n_rows + kWideRows - 1) / kWideRows) return;
        images = reinterpret_cast<const S*>(a.images) + (size_t)at_piece * a.tiles;
        part.first = block * kWideRows;
        part.results = results_of(a, part.b, part.h, part.chunk.first);
        if (!cut_range(a, part, kWideRows, 64)) return;
    }
    const int dim = a.c.t.dim, begin = part.begin, end = part.end;
    const int row = part.first + 32 * wave + j;
    const bool live = row < part.n_rows;
    const unsigned n = live ? a.by_per.div(row) : 0, qh = part.h * a.by_per.d + (live ? row - n * a.by_per.d : 0);
    const int seen = live ? max(part.chunk.seen + (int)n, 0) : 0;
    int all = live ? seen : 0x7fffffff, most = seen;   // positions that every row, that any row of the wave sees
    for (int o = 1; o < 32; o *= 2)
    {
        all = min(all, __shfl_xor(all, o, 64));
        most = max(most, __shfl_xor(most, o, 64));
    }
    all = __builtin_amdgcn_readfirstlane(all);
    most = __builtin_amdgcn_readfirstlane(most);

    const int tiles = (end - begin + kPos - 1) / kPos;
    // A thread's 16-byte pieces of a tile's keys and then of its values, and of what is behind them.
    constexpr int kKeys = sizeof(S::k) / 16, kValues = sizeof(S::v) / 16, kTail = sizeof(S) / 16 - kKeys - kValues;
    constexpr int kPieces = (kValues + 255) / 256;
    static_assert(kValues >= kKeys && kKeys % 64 == 0 && kValues % 64 == 0 && kTail <= 64);
    const f32x4* image = reinterpret_cast<const f32x4*>(images + begin / kPos);
    f32x4 piece[kPieces], tail;
    auto fetch = [&](int i, int half) __attribute__((always_inline)) {
        // (a sequence whose length is 0 has no tile: the first one's place is read for it)
        const f32x4* from = image + (size_t)max(min(i, tiles - 1), 0) * (sizeof(S) / 16) + half * kKeys;
        const int count = half ? kValues : kKeys;
#pragma unroll
        for (int x = 0; x < kPieces; ++x)
            if (256 * x + 256 <= count || 256 * x + 64 * wave < count) piece[x] = from[256 * x + t];
        if (half == 1) tail = from[kValues + min(lane, kTail - 1)];
    };
    auto place = [&](S& to, int half) __attribute__((always_inline)) {
        f32x4* at = reinterpret_cast<f32x4*>(&to) + half * kKeys;
        const int count = half ? kValues : kKeys;
#pragma unroll
        for (int x = 0; x < kPieces; ++x)
            if (256 * x + 256 <= count || 256 * x + 64 * wave < count) at[256 * x + t] = piece[x];
        if (half == 1 && wave == 0 && lane < kTail) at[kValues + lane] = tail;
    };
    fetch(0, 0);

    // The queries' parts: row l % 32, dims 16 k + 8 (l / 32) + e.
    half8 qp[KS][2];
    int se;   // the scores' exponent
    {
        floatx8 z[KS];
        const float* qp0 = a.q + (long)(part.chunk.first + n) * a.q_t + (long)qh * dim * a.q_f;   // rows that are none are formed and dropped
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
        {
            const int d = 16 * k + 8 * g;
            if (a.q_rows)
            {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(qp0 + (d < dim ? d : 0));
                const f32x4 hi = *reinterpret_cast<const f32x4*>(qp0 + (d + 4 < dim ? d + 4 : 0));
#pragma unroll
                for (int e = 0; e < 4; ++e) z[k][e] = lo[e], z[k][4 + e] = hi[e];
            }
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) z[k][e] = qp0[(long)(d + e < dim ? d + e : 0) * a.q_f];
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                z[k][e] = d + e < dim ? z[k][e] : 0.0f;
                top = fmaxf(top, fabsf(z[k][e]));
            }
        }
        const float by = a.alpha * kLog2e, by_m = __builtin_amdgcn_frexp_mantf(by);
        top = across(top, larger_of);
        const int qe = exponent_of(by_m == 0.0f ? top : top * by_m);
        se = qe - (BITS == 32 ? 10 : 15) + __builtin_amdgcn_frexp_expf(by);   // a float32 key's scale has the other 5
#pragma unroll
        for (int k = 0; k < KS; ++k)
        {
#pragma unroll
            for (int x = 0; x < 8; ++x) z[k][x] = __builtin_ldexpf(z[k][x], 15 - qe) * by_m;
            split2(z[k], qp[k][0], qp[k][1]);
        }
    }

    place(sh[0], 0);
    fetch(0, 1);
    place(sh[0], 1);
    fetch(1, 0);
    __syncthreads();
    const float slope = a.slopes && live ? a.slopes[qh] * kLog2e : 0.0f;
    // Of the scores, which the softmax takes as products with it. Not 0, which would make a masked score's product NaN.
    const float scale = fmaxf(__builtin_ldexpf(1.0f, se), 0x1p-149f);
    const bool whole = a.slopes || __builtin_amdgcn_ballot_w64(!(scale <= kMaxF));   // scores that are formed themselves
    float m = kLowest, l = 0.0f;
    Held held;
    floatx16 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[b][r] = 0.0f;

    for (int i = 0; i < tiles; ++i)
    {
        const int p0 = begin + kPos * i;
        const S& in = sh[i & 1];
        const unsigned now = __builtin_amdgcn_readfirstlane(in.there[0]);
        S& out = sh[(i & 1) ^ 1];
        // The next tile's parts: its keys were loaded during the last tile's second product, its values are during this one's
        // softmax.
        auto turn = [&](int half) __attribute__((always_inline)) {
            place(out, half);   // behind the last tile, too: nothing reads it
            fetch(i + 1 + half, half ^ 1);
        };
        const bool work = p0 < most;   // some row of the wave sees some of it
        const int shift = __builtin_amdgcn_readfirstlane(in.there[1]);
        floatx16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
        if (work)
        {
            // Operands are read kDeep steps before their products.
            constexpr int kDeep = 2;
            half8 ks[kDeep + 1][P];
            auto keys = [&](int k) __attribute__((always_inline)) {
#pragma unroll
                for (int x = 0; x < P; ++x) ks[k % (kDeep + 1)][x] = in.k[k][x][lane ^ ((2 * k + g) & 7)];
            };
#pragma unroll
            for (int k = 0; k < kDeep; ++k) keys(k);
#pragma unroll
            for (int k = 0; k < KS; ++k)
            {
                if (k + kDeep < KS) keys(k + kDeep);
                __builtin_amdgcn_sched_barrier(0);
                const half8(&x)[P] = ks[k % (kDeep + 1)];
                if constexpr (BITS == 32) s = mfma32(x[P - 1], qp[k][0], s);
                s = mfma32(x[0], qp[k][1], s);
                s = mfma32(x[0], qp[k][0], s);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
            {
                const f32x4 f = *reinterpret_cast<const f32x4*>(&in.k_scale[8 * q + 4 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * q + e] *= f[e];
            }
        }
        turn(0);
        if (work)
        {
            float by = scale;   // of the scores as the softmax sees them
            if (whole || shift != 0)
            {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_ldexpf(s[r], se + shift) - slope * (float)(seen - 1 - (p0 + 8 * (r / 4) + 4 * g + r % 4));
                by = 1.0f;
            }
            f32x4 vs[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) vs[q] = *reinterpret_cast<const f32x4*>(&in.v_scale[8 * q + 4 * g]);
            if (now != 0xffffffffu || p0 + kPos > all)
            {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                {
                    const int p = 8 * (r / 4) + 4 * g + r % 4;
                    const bool sees = (now >> p & 1) && p0 + p < seen;
                    s[r] = sees ? s[r] : -__builtin_inff();
                    if constexpr (BITS == 8) vs[r / 4][r % 4] = sees ? vs[r / 4][r % 4] : 0.0f;   // 0 times a NaN would be one
                }
            }
            float high = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) high = fmaxf(high, s[r]);
            high *= by;
            if (__builtin_amdgcn_ballot_w64(high > m))   // seldom past the first tiles
            {
                const float mn = fmaxf(m, across(high, larger_of));
                const float up = mn - m, f = shrink(held, up);
                m = mn;
                l *= __builtin_amdgcn_exp2f(-up);
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= f;
            }
            // What rounding the largest score took away is added to the weights' exponents: of scores past 2^20 it may be
            // more than an exponent holds, and these are rounded first.
            float once = by;
            if (__builtin_amdgcn_ballot_w64(fabsf(m) > 0x1p20f && m != kLowest))
            {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= by;
                once = 1.0f;
            }
            float sum = 0.0f, size = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r)
            {
                s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], once, -m));
                sum += s[r];
                s[r] *= vs[r / 4][r % 4];
                size = fmaxf(size, fabsf(s[r]));
            }
            constexpr int kQuarter = BITS == 32 ? 2 : 0;   // weights are held with the scales' quarters
            if (__builtin_amdgcn_ballot_w64(exponent_of(size) + kQuarter > held.top()))   // seldom, too
            {
                const float f = raise(held, exponent_of(across(size, larger_of)) + kQuarter);
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= f;
            }
            l += sum;
            const float to = __builtin_ldexpf(BITS == 32 ? 4.0f : 1.0f, 15 - held.top());
            const int place1 = lane ^ (lane >> 3 & 7);
            half8 vh[NB], vl[NB];
            auto values = [&](int st, int x, half8(&to)[NB]) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) to[b] = in.v[b][st][x][place1];
                __builtin_amdgcn_sched_barrier(0);
            };
            auto product = [&](const half8(&x)[NB], const half8& y) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] = mfma32(x[b], y, o[b]);
                __builtin_amdgcn_sched_barrier(0);
            };
            values(0, 0, vh);
            if constexpr (BITS == 32) values(0, P - 1, vl);
            half8 pp[2][2];
#pragma unroll
            for (int st = 0; st < 2; ++st)
            {
                floatx8 z;
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = s[8 * st + e] * to;
                split2(z, pp[st][0], pp[st][1]);
            }
            product(vh, pp[0][1]);
            product(vh, pp[0][0]);
            values(1, 0, vh);
            if constexpr (BITS == 32)
            {
                product(vl, pp[0][0]);
                values(1, P - 1, vl);
            }
            product(vh, pp[1][1]);
            product(vh, pp[1][0]);
            if constexpr (BITS == 32) product(vl, pp[1][0]);
        }
        turn(1);
        __syncthreads();
    }

    l = across(l, [](float x, float y) { return x + y; });
    const int unscale = held.top() - (BITS == 32 ? 30 : 15);
    bool bad = false;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
        {
            o[b][r] = __builtin_ldexpf(o[b][r], unscale);
            bad |= !(fabsf(o[b][r]) <= kMaxF);
        }
    if constexpr (BITS == 32)
    {
        bad = live && (bad || !(l <= kMaxF));
        if (__syncthreads_or(bad))
        {
            walk<32, KS, false, 2, true>(a, part, 4, *reinterpret_cast<WalkShared<KS>*>(lds));
            return;
        }
    }
    if (!live) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            put<true, true>(a, part, row, 32 * b + 8 * q + 4 * g, f32x4{o[b][4 * q], o[b][4 * q + 1], o[b][4 * q + 2], o[b][4 * q + 3]}, m, l,
                b == 0 && q == 0 && g == 0);
}

} // namespace

namespace
{
// f of the number of 16-dim groups, as a constant: at least 2.
template <class F> void of_groups(unsigned dim, F&& f)
{
    switch ((dim + 15) / 16)
    {
    case 3: f(std::integral_constant<int, 3>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 5: f(std::integral_constant<int, 5>()); break;
    case 6: f(std::integral_constant<int, 6>()); break;
    case 7: f(std::integral_constant<int, 7>()); break;
    case 8: f(std::integral_constant<int, 8>()); break;
    default: f(std::integral_constant<int, 2>()); break;
    }
}
} // namespace

size_t chunk_image_bytes(int bits, unsigned dim)
{
    size_t bytes = 0;
    of_groups(dim, [&](auto n) { bytes = bits == 32 ? sizeof(Image<32, n()>) : sizeof(Image<8, n()>); });
    return bytes;
}

void chunk_parts(const ChunkArgs& a, int bits, unsigned pieces, unsigned blocks, hipStream_t s)
{
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(pieces * blocks), dim3(256), 0, s, a, FastDiv(blocks)); };
    of_groups(a.c.t.dim, [&](auto n) { bits == 32 ? go(k_attn_chunk_parts<32, n()>) : go(k_attn_chunk_parts<8, n()>); });
}

void chunk_wide(const ChunkArgs& a, int bits, unsigned blocks, hipStream_t s)
{
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, s, a); };
    of_groups(a.c.t.dim, [&](auto n) { bits == 32 ? go(k_attn_chunk_wide<32, n()>) : go(k_attn_chunk_wide<8, n()>); });
}

} // namespace nnhip
