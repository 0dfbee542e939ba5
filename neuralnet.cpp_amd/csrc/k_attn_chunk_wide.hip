// k_attn_chunk_wide.hip — chunk attention of sequences with many rows: both
// products on the float16 matrix cores, from parts (f16_parts.hpp): three float16 products for a float32 one, two over an 8-bit
// cache.
//
// The scales are exact: a key's goes into its scores, a value's into its
// position's weights, relative to the largest so far (the outputs are rescaled
// when that grows, as they are when a row's largest score does).
//
// A workgroup takes 128 rows, 32 to a wave, and 32 positions at a time. Its waves
// form the positions' parts together and leave them in LDS in the order of the
// matrix cores' operands. Both products are formed transposed (S^T = K Q^T, O^T =
// V^T P^T), 32 x 32 x 16 at a time: lane l has the scores of row l % 32 and of
// the positions 8 (r / 4) + 4 (l / 32) + r % 4, r < 16, and its weights are the
// second product's operand as they lie, if its k index 8 (l / 32) + e of step t
// stands for position 8 (2 t + e / 4) + 4 (l / 32) + e % 4.
//
// Of a float32 cache, results that are not finite are formed again by the float32
// walk: infinities and NaN among keys, queries and values, also at positions
// that some of the rows do not see.
#include "attn_chunk.hpp"
#include "f16_parts.hpp"

namespace nnhip
{
namespace
{

constexpr int kPos = 32;      // positions of a tile

__device__ __forceinline__ floatx16 mfma32(const half8& x, const half8& y, const floatx16& c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
}

template <int BITS, int KS> struct WideShared
{
    static constexpr int P = BITS == 32 ? 2 : 1;   // parts
    // Operands by lane: [buffer][step or block of 32 dims and k step][part][lane's place]
    half8 k[2][KS][P][64];
    half8 v[2][KS / 2][2][P][64];
    float k_scale[2][kPos];        // of the scores
    float v_scale[2][kPos];        // BITS 8: of the values
    int v_top[2][4];               // exponents of the values: of each group of 8 positions; BITS 8: all [0]
};

// What a thread holds of a tile on its way to LDS. Keys: 8 dims of one position each; values: VD dims of the 8 positions of
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
    using S = WideShared<BITS, KS>;
    static constexpr int P = S::P, NB = KS / 2;

    const ChunkArgs& a;
    const Part& part;
    S& sh;
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

    // The tile's parts into buffer b; there: which of its positions exist. Absent ones, and dims past the last, are 0.
    __device__ __forceinline__ void stage(const R& r, int b, unsigned there)
    {
        const int dim = a.c.t.dim;
        const bool whole = there == 0xffffffffu && dim == 16 * KS;
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
                    sh.k[b][step][0][place] = hi;
                    sh.k[b][step][P - 1][place] = lo;
                    if (d == 0) sh.k_scale[b][p] = __builtin_ldexpf(1.0f, ke - 20);
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
                if (mine) sh.k[b][step][0][place] = __builtin_bit_cast(half8, z);
            }
        }
        {
            const int group = wave;   // k step group >> 1, half group & 1
            const int d0 = R::VD * lane;
            unsigned ok = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) ok |= (there >> value_pos(e) & 1u) << e;
            floatx8 z[R::VD];
            float top = 0.0f;
            int ve = 0;
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
#pragma unroll
                for (int y = 0; y < R::VD; ++y)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(z[y][e]));
                top = max_of<64>(top);
                ve = top > 0.0f ? exponent_of(top) : kNone;
            }
#pragma unroll
            for (int y = 0; y < R::VD; ++y)
            {
                const int d = d0 + y;
                if (d >= 16 * KS) continue;
                const int slot = d % 32 + 32 * (group & 1), place = slot ^ (slot >> 3 & 7);
                half8(&to)[P][64] = sh.v[b][d / 32][group >> 1];
                if constexpr (BITS == 32)
                {
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[y][e] = __builtin_ldexpf(z[y][e], 15 - ve);
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
            if constexpr (BITS == 32)
                if (lane == 0) sh.v_top[b][group] = ve;
        }
        if constexpr (BITS == 8)
            if (wave == 0)
            {
                const bool ok = there >> (lane & 31) & 1;
                const float s = ok ? r.scale : 0.0f;
                const float top = max_of<32>(fabsf(s) <= kMaxF ? fabsf(s) : 0.0f);
                const int e = top > 0.0f ? exponent_of(top) : kNone;   // of the keys' scales, of the values'
                if (lane < 32) sh.k_scale[b][lane] = s * 0x1p-5f;
                else
                {
                    sh.v_scale[b][lane - 32] = s;
                    if (lane == 32) sh.v_top[b][0] = e;
                }
            }
    }
};

template <int BITS, int KS> __global__ __launch_bounds__(256, 2) void k_attn_chunk_wide(ChunkArgs a)
{
    using W = Wide<BITS, KS>;
    using S = WideShared<BITS, KS>;
    constexpr int NB = KS / 2, P = S::P;
    constexpr size_t kLds = BITS == 32 && sizeof(WalkShared<KS>) > sizeof(S) ? sizeof(WalkShared<KS>) : sizeof(S);
    __shared__ __attribute__((aligned(16))) char lds[kLds];
    S& sh = *reinterpret_cast<S*>(lds);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 31, g = lane >> 5;
    Part part;
    // Workgroups go to the 8 XCDs in turn: each takes neighbouring pieces of work, the blocks of rows of one range of one key
    // head after another (they read the same keys and values), the rows that see most first.
    {
        const unsigned each = gridDim.x / 8, at = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
        const unsigned piece = a.by_row_blocks.div(at);
        const unsigned x = a.by_row_blocks.d - 1 - (at - piece * a.by_row_blocks.d);
        part.h = a.by_ranges.div(piece);
        part.slot = piece - part.h * a.ranges;
        if (part.h >= a.c.t.heads) return;
        // Sequence b's blocks of rows are numbered from first row / 128 + b on: at least as many as it has.
        auto base = [&](unsigned b) { return (unsigned)((size_t)length_of(a.start[b], a.tokens) * a.by_per.d / kWideRows) + b; };
        const int b = last_of(a.c.t.batch, [&](unsigned i) { return base(i) <= x; });
        if (b < 0) return;
        part.b = b;
        part.chunk = chunk_of(a, part.b);
        part.n_rows = part.chunk.n * a.by_per.d;
        const unsigned block = x - base(b);
        if (part.n_rows <= a.wide_from || block >= (unsigned)(part.n_rows + kWideRows - 1) / kWideRows) return;
        part.first = block * kWideRows;
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

    W w{a, part, sh, t, lane, wave};
    typename W::R raw;
    auto entry = [&](int p) { return a.c.t.entry_of(part.b, p + j); };
    auto row_at = [&](float e, int p) {
        const int r = a.c.t.row_in(e, p + j);
        return p + j < end ? r : -1;
    };
    auto mask_of = [](int r) { return (unsigned)__builtin_amdgcn_ballot_w64(r >= 0); };
    float ahead = entry(begin + kPos);
    int at = row_at(entry(begin), begin), kr[W::R::KI];
    unsigned there = mask_of(at);   // of the tile in `raw`
    w.key_rows(at, kr);
    w.load(at, kr, raw);
    at = row_at(ahead, begin + kPos);
    w.key_rows(at, kr);
    ahead = entry(begin + 2 * kPos);

    // The queries' parts: row l % 32, dims 16 k + 8 (l / 32) + e.
    half8 qp[KS][2];
    int qe;
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
        qe = exponent_of(across(top, [](float x, float y) { return fmaxf(x, y); }));
#pragma unroll
        for (int k = 0; k < KS; ++k)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[k][e] = __builtin_ldexpf(z[k][e], 15 - qe);
            split2(z[k], qp[k][0], qp[k][1]);
        }
    }

    w.stage(raw, 0, there);
    const unsigned there0 = there;
    there = mask_of(at);
    w.load(at, kr, raw);
    at = row_at(ahead, begin + 2 * kPos);
    w.key_rows(at, kr);
    ahead = entry(begin + 3 * kPos);
    __syncthreads();
    unsigned now = there0;          // the positions of the tile whose parts are used
    const float slope = a.slopes && live ? a.slopes[qh] * kLog2e : 0.0f;
    const float scale = __builtin_ldexpf(a.alpha * kLog2e, qe - 10);   // scores times log2(e)
    float m = kLowest, l = 0.0f;
    int top = kNone;                // exponent that the values are held against
    floatx16 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[b][r] = 0.0f;

    const int tiles = (end - begin + kPos - 1) / kPos;
    for (int i = 0; i < tiles; ++i)
    {
        const int p0 = begin + kPos * i, buf = i & 1;
        unsigned next = 0;
        if (i + 1 < tiles)
        {
            next = there;
            w.stage(raw, buf ^ 1, there);
            there = mask_of(at);
            w.load(at, kr, raw);
            at = row_at(ahead, p0 + 3 * kPos);
            w.key_rows(at, kr);
            ahead = entry(p0 + 4 * kPos);
        }
        if (p0 < most)
        {
            floatx16 s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
            {
                const int place0 = lane ^ ((2 * k + g) & 7);
                const half8 hi = sh.k[buf][k][0][place0];
                if constexpr (BITS == 32)
                {
                    const half8 lo = sh.k[buf][k][P - 1][place0];
                    s = mfma32(lo, qp[k][0], s);
                }
                s = mfma32(hi, qp[k][1], s);
                s = mfma32(hi, qp[k][0], s);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
            {
                const f32x4 f = *reinterpret_cast<const f32x4*>(&sh.k_scale[buf][8 * q + 4 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * q + e] = s[4 * q + e] * f[e] * scale;
            }
            if (a.slopes)
            {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] -= slope * (float)(seen - 1 - (p0 + 8 * (r / 4) + 4 * g + r % 4));
            }
            if (now != 0xffffffffu || p0 + kPos > all)
            {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                {
                    const int p = 8 * (r / 4) + 4 * g + r % 4;
                    s[r] = (now >> p & 1) && p0 + p < seen ? s[r] : -__builtin_inff();
                }
            }
            float high = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) high = fmaxf(high, s[r]);
            high = across(high, [](float x, float y) { return fmaxf(x, y); });
            const float mn = fmaxf(m, high);
            float f = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r)
            {
                s[r] = __builtin_amdgcn_exp2f(s[r] - mn);
                sum += s[r];
            }
            l = l * f + sum;
            // The values' scales. Weights that are 0 stay so, whatever their position's scale is.
            int new_top = sh.v_top[buf][0];
            if constexpr (BITS == 32) new_top = max(max(new_top, sh.v_top[buf][1]), max(sh.v_top[buf][2], sh.v_top[buf][3]));
            new_top = max(top, __builtin_amdgcn_readfirstlane(new_top));
            if (new_top != top) f = __builtin_ldexpf(f, top - new_top);
            top = new_top;
            if (__builtin_amdgcn_ballot_w64(f != 1.0f))   // seldom past the first tiles
            {
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] *= f;
            }
            half8 pp[2][2];
#pragma unroll
            for (int st = 0; st < 2; ++st)
            {
                floatx8 z;
                if constexpr (BITS == 32)
                {
                    const float to = __builtin_ldexpf(1.0f, sh.v_top[buf][2 * st + g] - top + 15);
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[e] = s[8 * st + e] * to;
                }
                else
                {
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                    {
                        const f32x4 vs = *reinterpret_cast<const f32x4*>(&sh.v_scale[buf][8 * (2 * st + q) + 4 * g]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                        {
                            const float x = s[8 * st + 4 * q + e], y = x * __builtin_ldexpf(vs[e], 15 - top);
                            z[4 * q + e] = x == 0.0f ? 0.0f : y;
                        }
                    }
                }
                split2(z, pp[st][0], pp[st][1]);
            }
            const int place1 = lane ^ (lane >> 3 & 7);
#pragma unroll
            for (int st = 0; st < 2; ++st)
            {
                half8 hi[NB];
#pragma unroll
                for (int b = 0; b < NB; ++b) hi[b] = sh.v[buf][b][st][0][place1];
                if constexpr (BITS == 32)
                {
#pragma unroll
                    for (int b = 0; b < NB; ++b) o[b] = mfma32(sh.v[buf][b][st][P - 1][place1], pp[st][0], o[b]);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] = mfma32(hi[b], pp[st][1], o[b]);
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] = mfma32(hi[b], pp[st][0], o[b]);
            }
        }
        now = next;
        __syncthreads();
    }

    l = across(l, [](float x, float y) { return x + y; });
    const int unscale = top - (BITS == 32 ? 30 : 15);
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

void chunk_wide(const ChunkArgs& a, int bits, unsigned blocks, hipStream_t s)
{
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, s, a); };
    const int groups = (static_cast<int>(a.c.t.dim) + 31) / 32;
    if (bits == 32) groups == 1 ? go(k_attn_chunk_wide<32, 2>) : groups == 2 ? go(k_attn_chunk_wide<32, 4>) : groups == 3 ? go(k_attn_chunk_wide<32, 6>) : go(k_attn_chunk_wide<32, 8>);
    else groups == 1 ? go(k_attn_chunk_wide<8, 2>) : groups == 2 ? go(k_attn_chunk_wide<8, 4>) : groups == 3 ? go(k_attn_chunk_wide<8, 6>) : go(k_attn_chunk_wide<8, 8>);
}

} // namespace nnhip
