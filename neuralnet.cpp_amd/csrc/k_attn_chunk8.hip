// k_attn_chunk8.hip — chunk attention of sequences with few rows over an 8-bit
// cache (single tokens above all), bound by the cache's bytes.
//
// As in the float32 walk (attn_chunk.hpp) a wave forms both products transposed
// and a workgroup's four waves take 32 positions each in turn, but on the
// float16 matrix cores (16 x 16 x 32): bytes are float16 as they are, so that
// queries and weights in two parts (f16_parts.hpp) make float32's accuracy of
// two products, eight times faster than the float32 cores'. With their single
// products a key head's 16 positions would take 2048 cycles, which 5 TB/s of
// bytes do not leave.
//
// Lane l = 16 g + j has the scores of row j and of the positions 16 u + 4 g + r
// (u < 2, r < 4), which stand behind the k index 8 g + 4 u + r of the second
// product. Block b of the output's dims are those that leave the remainder b by
// VB, so that the lane's VB neighbouring bytes of a value row serve one block
// each.
//
// Rows are read 16, 8 or 4 bytes at a time, as heads begin (32 sequences of 3000
// positions, 12 heads: of 64 bytes 38 us, of 40 39, of 36 43; the float32 walk,
// which takes heads of odd widths byte by byte, took 183 us for 40).
#include "attn_chunk.hpp"
#include "f16_parts.hpp"

namespace nnhip
{
namespace
{

constexpr int kPos = 32;   // positions of a tile

__device__ __forceinline__ f32x4 mfma16(const half8& x, const half8& y, const f32x4& c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
}

// KS: groups of 16 dims, even. W: rows, heads and the caches themselves begin at multiples of W bytes, 16, 8 or 4, which is what
// a lane loads at a time. VB: value bytes of a lane and position, and blocks of dims; up to 16 VB dims.
template <int KS, int W> struct Bytes
{
    static constexpr int VB = KS <= 2 ? 2 : KS <= 4 ? 4 : 8, VW = (VB + 3) / 4, steps = KS / 2;
    // Keys are loaded 16 bytes at a time where whole pairs of steps let them: bytes 0 to 7 are the first step's.
    static constexpr bool WIDE = KS % 4 == 0 && W == 16;
    static __device__ __forceinline__ int dim_of(int step, int g) { return WIDE ? 64 * (step / 2) + 16 * g + 8 * (step % 2) : 32 * step + 8 * g; }
};

template <int KS, int W> struct Row8
{
    half8 q[KS / 2][2];
    int seen;
    Held held;                  // of weights times values' scales
    int e;                      // the scores' exponent
    float slope, m, l;          // slope and m: times log2(e)
    f32x4 o[Bytes<KS, W>::VB];
};

template <int KS, int W> struct Shared8
{
    using B = Bytes<KS, W>;
    union
    {
        float scales[4][2][kPos];   // by wave: the keys', the values'
        float o[4][kTile][16 * B::VB + 4];
    };
    float ml[4][kTile][2];
};

// One tile's bytes on their way.
template <int KS, int W> struct Tile8
{
    using B = Bytes<KS, W>;
    unsigned k[2][B::steps][2], v[8][B::VW];
    float scale;   // lane p < 32: position p's of the keys; lane 32 + p: of the values
};

template <int KS, int W> __device__ __forceinline__ void load_keys8(const ChunkArgs& a, int row, unsigned h, int lane, Tile8<KS, W>& x)
{
    using B = Bytes<KS, W>;
    const int j = lane & 15, g = lane >> 4, dim = a.c.t.dim;
#pragma unroll
    for (int u = 0; u < 2; ++u)
    {
        const signed char* from = a.c.K + (size_t)max(__shfl(row, 16 * u + j, 64), 0) * a.c.t.row + (size_t)h * dim;
#pragma unroll
        for (int s = 0; s < B::steps; s += B::WIDE ? 2 : 1)
        {
            const int d = B::dim_of(s, g);
            const signed char* at = from + (d < dim ? d : 0);
            if constexpr (B::WIDE)
            {
                const uintx4 z = *reinterpret_cast<const uintx4*>(at);
                x.k[u][s][0] = z[0];
                x.k[u][s][1] = z[1];
                x.k[u][s + 1][0] = z[2];
                x.k[u][s + 1][1] = z[3];
            }
            else if constexpr (W >= 8)
            {
                const uint2 z = *reinterpret_cast<const uint2*>(at);
                x.k[u][s][0] = z.x;
                x.k[u][s][1] = z.y;
            }
            else
            {
                x.k[u][s][0] = *reinterpret_cast<const unsigned*>(at);
                x.k[u][s][1] = *reinterpret_cast<const unsigned*>(from + (d + 4 < dim ? d + 4 : 0));
            }
        }
    }
    x.scale = (lane < 32 ? a.c.K_scale : a.c.V_scale)[(size_t)max(row, 0) * a.c.t.heads + h];
}
template <int KS, int W> __device__ __forceinline__ void load_values8(const ChunkArgs& a, int row, unsigned h, int lane, Tile8<KS, W>& x)
{
    using B = Bytes<KS, W>;
    const int j = lane & 15, g = lane >> 4, dim = a.c.t.dim, d = B::VB * j;
    auto load = [&](int e, size_t r) {
        const signed char* at = a.c.V + r * a.c.t.row + (size_t)h * dim + (d < dim ? d : 0);
        if constexpr (B::VB == 8 && W == 4)
        {
            x.v[e][0] = *reinterpret_cast<const unsigned*>(at);
            x.v[e][B::VW - 1] = *reinterpret_cast<const unsigned*>(at + (d + 4 < dim ? 4 : 0));
        }
        else if constexpr (B::VB == 8)
        {
            const uint2 z = *reinterpret_cast<const uint2*>(at);
            x.v[e][0] = z.x;
            x.v[e][B::VW - 1] = z.y;
        }
        else if constexpr (B::VB == 4) x.v[e][0] = *reinterpret_cast<const unsigned*>(at);
        else x.v[e][0] = *reinterpret_cast<const unsigned short*>(at);
    };
    if (a.page4)   // four neighbouring positions lie in neighbouring rows
    {
#pragma unroll
        for (int u = 0; u < 2; ++u)
        {
            const int r = __shfl(row, 16 * u + 4 * g, 64);
#pragma unroll
            for (int e = 0; e < 4; ++e) load(4 * u + e, r < 0 ? 0 : (size_t)r + e);
        }
    }
    else
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) load(e, max(__shfl(row, 16 * (e / 4) + 4 * g + e % 4, 64), 0));
    }
}

// 8 bytes as float16, in the order of the bytes.
__device__ __forceinline__ half8 halves8(unsigned lo, unsigned hi)
{
    uintx4 z;
    z[0] = halves_of(__builtin_amdgcn_perm(0u, lo, 0x0c010c00u));
    z[1] = halves_of(__builtin_amdgcn_perm(0u, lo, 0x0c030c02u));
    z[2] = halves_of(__builtin_amdgcn_perm(0u, hi, 0x0c010c00u));
    z[3] = halves_of(__builtin_amdgcn_perm(0u, hi, 0x0c030c02u));
    return __builtin_bit_cast(half8, z);
}

template <int KS, int W, int RT> __device__ __forceinline__ void walk8(const ChunkArgs& a, const Part& part, Shared8<KS, W>& sh)
{
    using B = Bytes<KS, W>;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), j = lane & 15, g = lane >> 4;
    const int dim = a.c.t.dim, begin = part.begin, end = part.end, step = 4 * kPos;
    Row8<KS, W> rows[RT];
    int all = 0x7fffffff;
    const float by = a.alpha * kLog2e, by_m = __builtin_amdgcn_frexp_mantf(by);
    const int p1 = begin + wave * kPos;
    // Lane p and lane 32 + p: the table's entry and the row of position p of a tile.
    auto entry = [&](int p) { return a.c.t.entry_of(part.b, p + (lane & 31)); };
    auto row_at = [&](float e, int p) {
        const int r = a.c.t.row_in(e, p + (lane & 31));
        return p + (lane & 31) < end ? r : -1;
    };
    Tile8<KS, W> x;
    float ahead = entry(p1 + step);
    int row = row_at(entry(p1), p1);
    unsigned there = (unsigned)__builtin_amdgcn_ballot_w64(row >= 0);
    load_keys8<KS, W>(a, row, part.h, lane, x);
    load_values8<KS, W>(a, row, part.h, lane, x);
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        Row8<KS, W>& w = rows[i];
        const int r = part.first + i * kTile + j;
        const bool live = r < part.n_rows;
        const unsigned n = live ? a.by_per.div(r) : 0, qh = part.h * a.by_per.d + (live ? r - n * a.by_per.d : 0);
        w.seen = live ? max(part.chunk.seen + (int)n, 0) : 0;
        all = min(all, live ? w.seen : 0x7fffffff);
        const float* from = a.q + (long)(part.chunk.first + n) * a.q_t + (long)qh * dim * a.q_f;   // rows that are none are formed and dropped
        floatx8 z[B::steps];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < B::steps; ++s)
        {
            const int d = B::dim_of(s, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[s][e] = from[(long)(d + e < dim ? d + e : 0) * a.q_f];
        }
#pragma unroll
        for (int s = 0; s < B::steps; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                z[s][e] = B::dim_of(s, g) + e < dim ? z[s][e] : 0.0f;   // dims past the last one
                top = fmaxf(top, fabsf(z[s][e]));
            }
        top = across4(top, larger_of);
        const int qe = exponent_of(by_m == 0.0f ? top : top * by_m);
#pragma unroll
        for (int s = 0; s < B::steps; ++s)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[s][e] = __builtin_ldexpf(z[s][e], 15 - qe) * by_m;
            split2(z[s], w.q[s][0], w.q[s][1]);
        }
        w.slope = a.slopes && live ? a.slopes[qh] * kLog2e : 0.0f;
        w.e = qe - 15 + __builtin_amdgcn_frexp_expf(by);
        w.held = Held();
        w.m = kLowest;
        w.l = 0.0f;
#pragma unroll
        for (int b = 0; b < B::VB; ++b) w.o[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int o = 1; o < 16; o *= 2) all = min(all, __shfl_xor(all, o, 64));
    all = __builtin_amdgcn_readfirstlane(all);
    for (int p = p1; p < end; p += step)
    {
        f32x4 s[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i) s[i][0] = s[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        // The scales, from a lane a position to a lane's positions, through LDS: the wave's own part of it.
        const float scale = there >> (lane & 31) & 1 ? scale_or_nan(x.scale) : 0.0f;
        const float size = fabsf(scale);
        const int shift = shift_of(__builtin_amdgcn_ballot_w64(lane < 32 && size > kFar), !__builtin_amdgcn_ballot_w64(lane < 32 && size >= kNear));
        (&sh.scales[wave][0][0])[lane] = lane < 32 ? __builtin_ldexpf(scale, -shift) : scale;
#pragma unroll
        for (int k = 0; k < B::steps; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u)
            {
                const half8 z = halves8(x.k[u][k][0], x.k[u][k][1]);
#pragma unroll
                for (int i = 0; i < RT; ++i) s[i][u] = mfma16(z, rows[i].q[k][1], s[i][u]);
#pragma unroll
                for (int i = 0; i < RT; ++i) s[i][u] = mfma16(z, rows[i].q[k][0], s[i][u]);
            }
        f32x4 ks[2], vs[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
        {
            ks[u] = *reinterpret_cast<const f32x4*>(&sh.scales[wave][0][16 * u + 4 * g]);
            vs[u] = *reinterpret_cast<const f32x4*>(&sh.scales[wave][1][16 * u + 4 * g]);
        }
        const float further = entry(p + 2 * step);
        row = row_at(ahead, p + step);
        const unsigned now = there;
        there = (unsigned)__builtin_amdgcn_ballot_w64(row >= 0);
        load_keys8<KS, W>(a, row, part.h, lane, x);
        __builtin_amdgcn_sched_barrier(0);

        const bool part_seen = now != 0xffffffffu || p + kPos > all, odd = a.slopes || part_seen;
        half8 pp[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i)
        {
            Row8<KS, W>& w = rows[i];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][u][e] = __builtin_ldexpf(s[i][u][e] * ks[u][e], w.e + shift);
            unsigned mine = 0;   // which of the lane's positions its row sees, where it does not see all
            if (odd)
            {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        const int q = 16 * u + 4 * g + e;
                        const float z = s[i][u][e] - w.slope * (float)(w.seen - 1 - (p + q));
                        const bool sees = (now >> q & 1) && p + q < w.seen;
                        s[i][u][e] = sees ? z : -__builtin_inff();
                        mine |= (sees ? 1u : 0u) << (4 * u + e);
                    }
            }
            float high = kLowest;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) high = fmaxf(high, s[i][u][e]);
            if (__builtin_amdgcn_ballot_w64(high > w.m))   // seldom past the first tiles
            {
                const float mn = fmaxf(w.m, across4(high, larger_of)), up = mn - w.m, f = shrink(w.held, up);
                w.m = mn;
                w.l *= __builtin_amdgcn_exp2f(-up);
#pragma unroll
                for (int b = 0; b < B::VB; ++b) w.o[b] *= f;
            }
            float sum = 0.0f, size = 0.0f;
            floatx8 z;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    const float y = __builtin_amdgcn_exp2f(s[i][u][e] - w.m);
                    sum += y;
                    z[4 * u + e] = y * vs[u][e];
                }
            if (part_seen)   // 0 times a NaN would be one
            {
                asm volatile("");   // stays a branch
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = mine >> e & 1 ? z[e] : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) size = fmaxf(size, fabsf(z[e]));
            if (__builtin_amdgcn_ballot_w64(exponent_of(size) > w.held.top()))   // seldom, too
            {
                const float f = raise(w.held, exponent_of(across4(size, larger_of)));
#pragma unroll
                for (int b = 0; b < B::VB; ++b) w.o[b] *= f;
            }
            w.l += sum;
            const float to = __builtin_ldexpf(1.0f, 15 - w.held.top());
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] *= to;
            split2(z, pp[i][0], pp[i][1]);
        }
#pragma unroll
        for (int b = 0; b < B::VB; ++b)
        {
            uintx4 z;
#pragma unroll
            for (int e = 0; e < 8; e += 2)
            {
                const unsigned pick = 0x0c040c00u + 0x00010001u * (b % 4);
                z[e / 2] = halves_of(__builtin_amdgcn_perm(x.v[e + 1][b / 4], x.v[e][b / 4], pick));
            }
            const half8 y = __builtin_bit_cast(half8, z);
#pragma unroll
            for (int i = 0; i < RT; ++i) rows[i].o[b] = mfma16(y, pp[i][1], rows[i].o[b]);
#pragma unroll
            for (int i = 0; i < RT; ++i) rows[i].o[b] = mfma16(y, pp[i][0], rows[i].o[b]);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_values8<KS, W>(a, row, part.h, lane, x);
        ahead = further;
    }

    // The waves joined in the order of their positions: 16 threads a row, 4 neighbouring values at a time.
#pragma unroll
    for (int i = 0; i < RT; ++i)
    {
        Row8<KS, W>& w = rows[i];
        w.l = across4(w.l, [](float x, float y) { return x + y; });
        __syncthreads();
        if (g == 0)
        {
            sh.ml[wave][j][0] = w.m;
            sh.ml[wave][j][1] = w.l;
        }
#pragma unroll
        for (int b = 0; b < B::VB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) sh.o[wave][j][B::VB * (4 * g + r) + b] = __builtin_ldexpf(w.o[b][r], w.held.top() - 15);
        __syncthreads();
        const int jr = t >> 4, r = part.first + i * kTile + jr;
        if (r >= part.n_rows) continue;
        float mm = kLowest, ll = 0.0f, f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) mm = fmaxf(mm, sh.ml[k][jr][0]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
        {
            f[k] = sh.ml[k][jr][1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(sh.ml[k][jr][0] - mm);
            ll += sh.ml[k][jr][1] * f[k];
        }
#pragma unroll
        for (int d0 = 0; d0 < 16 * B::VB; d0 += 64)
        {
            const int d = d0 + 4 * (t & 15);
            if (d >= 16 * B::VB) continue;
            f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (sh.ml[k][jr][1] != 0.0f) z += *reinterpret_cast<const f32x4*>(&sh.o[k][jr][d]) * f[k];
            put<true, true>(a, part, r, d, z, mm, ll, d == 0);
        }
    }
}

// RT 1: no sequence has more than 16 rows.
template <int KS, int W, int RT> __global__ __launch_bounds__(256, RT == 1 ? 3 : 2) void k_attn_chunk8(ChunkArgs a)
{
    __shared__ Shared8<KS, W> sh;
    Part part;
    if (!narrow_part(a, part, 4 * kPos)) return;
    if (RT == 1 || part.n_rows <= kTile) walk8<KS, W, 1>(a, part, sh);
    else walk8<KS, W, RT>(a, part, sh);
}

} // namespace

template <int W> void launch8(const ChunkArgs& a, unsigned blocks, hipStream_t s)
{
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, s, a); };
    constexpr int W8 = W < 8 ? W : 8;   // odd numbers of 32 dims are loaded 8 bytes at a time at most
    const int groups = (static_cast<int>(a.c.t.dim) + 31) / 32;
    if (a.wide_from <= kTile) groups == 1 ? go(k_attn_chunk8<2, W8, 1>) : groups == 2 ? go(k_attn_chunk8<4, W, 1>) : groups == 3 ? go(k_attn_chunk8<6, W8, 1>) : go(k_attn_chunk8<8, W, 1>);
    else groups == 1 ? go(k_attn_chunk8<2, W8, 2>) : groups == 2 ? go(k_attn_chunk8<4, W, 2>) : groups == 3 ? go(k_attn_chunk8<6, W8, 2>) : go(k_attn_chunk8<8, W, 2>);
}
void chunk8(const ChunkArgs& a, int bytes, unsigned blocks, hipStream_t s)
{
    if (bytes >= 16) launch8<16>(a, blocks, s);
    else if (bytes == 8) launch8<8>(a, blocks, s);
    else launch8<4>(a, blocks, s);
}

} // namespace nnhip
