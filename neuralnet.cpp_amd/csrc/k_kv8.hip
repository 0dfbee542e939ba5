// k_kv8.hip — 8-bit paged caches: new tokens' keys and values quantised as they
// are stored, rotated on the way, and what a cache holds read back.
//
// A head's row of a token has one scale, its largest size / 127 in float32; a
// byte is the value / scale to the nearest integer. The turned key is two
// exact products and one rounding in float64, and so are the quotients: a byte
// is then off by half a step at most, whatever float32 would have rounded, and
// the same on every engine.
#include "kv_pages.hpp"

namespace nnhip
{
namespace
{

constexpr int kTokens = 32;      // of a tile
constexpr int kWidest = 256;     // head

struct Store8Args
{
    Pages8 c;
    Features k, v, q, out;
    Tokens tokens;
    const float *cos, *sin;
    int half, log2_lanes;        // rope_dim / 2; lanes along a tile's tokens
    int words;                   // rows can be written 4 bytes at a time
    int log2_group;              // lanes of a head, where tokens are rows
    FastDiv by_slots;
};

// The scale of a head whose largest size is `top`: NaN where a value is not finite.
__device__ __forceinline__ float scale_of(double top)
{
    return top < __builtin_inf() ? (float)(top / 127.0) : __builtin_nanf("");
}
__device__ __forceinline__ int byte_of(double x, float scale)
{
    if (!(scale > 0.0f)) return 0;   // 0, NaN
    const double y = rint(x / (double)scale);
    return (int)fmin(fmax(y, -127.0), 127.0);   // past 127 where the scale is denormal and was rounded down
}
// The larger size, NaN if either is.
__device__ __forceinline__ double larger(double a, double b) { return a >= b || a != a ? a : b; }

// One tile of tokens of one head slot (blockIdx.y: keys, values, queries), in any layout. The tile is read in the order
// of its own layout into LDS; 8 to 64 threads then share a token's head.
__global__ __launch_bounds__(256) void k_kv8_append(Store8Args a)
{
    extern __shared__ float tile_s[];   // [token][dim + 1]
    __shared__ int row_s[kTokens];
    __shared__ unsigned pos_s[kTokens];
    const int t = threadIdx.x, dim = a.c.t.dim, ld = dim + 1;
    const unsigned n0 = blockIdx.x * kTokens, heads = a.c.t.heads, y = blockIdx.y;
    const int nt = min((unsigned)kTokens, a.tokens.n - n0);
    const int kind = y < heads ? 0 : y < 2 * heads ? 1 : 2;
    const unsigned h = kind == 0 ? y : kind == 1 ? y - heads : y - 2 * heads;
    const Features& x = kind == 0 ? a.k : kind == 1 ? a.v : a.q;
    const float* xp = x.p + (long)n0 * x.t + (long)h * dim * x.f;
    // Every (token, feature) of the tile, f(n, d).
    auto over = [&](bool along_features, auto&& f) {
        if (along_features)
            for (int n = t >> 6; n < nt; n += 4)
                for (int d = t & 63; d < dim; d += 64) f(n, d);
        else if (const int n = t & ((1 << a.log2_lanes) - 1); n < nt)
            for (int d = t >> a.log2_lanes; d < dim; d += 256 >> a.log2_lanes) f(n, d);
    };
    over(x.f == 1, [&](int n, int d) { tile_s[n * ld + d] = xp[(long)n * x.t + (long)d * x.f]; });
    if (t < nt) row_s[t] = a.tokens.row(a.c.t, n0 + t, pos_s[t]);
    __syncthreads();
    const int half = kind == 1 ? 0 : a.half;
    if (kind == 2)
    {
        over(a.out.f == 1, [&](int n, int d) {
            if (row_s[n] < 0) return;
            float v = tile_s[n * ld + d];
            if (d < 2 * half)
            {
                const int j = d < half ? d : d - half;
                const size_t at = (size_t)pos_s[n] * half + j;
                const float co = a.cos[at], si = a.sin[at];
                v = d < half ? v * co - tile_s[n * ld + d + half] * si : v * co + tile_s[n * ld + j] * si;
            }
            a.out.p[(long)(n0 + n) * a.out.t + ((long)h * dim + d) * a.out.f] = v;
        });
        return;
    }
    // As many threads to a token as its tile leaves: 8 of 32 tokens, 64 of up to 4.
    const int log2_tp = min(8 - a.log2_lanes, 6), tp = 1 << log2_tp, n = t >> log2_tp, e = t & (tp - 1), row = n < nt ? row_s[n] : -1;
    const float* xs = tile_s + n * ld;
    auto value = [&](int d) -> double {
        const double v = xs[d];
        if (d >= 2 * half) return v;
        const int j = d < half ? d : d - half;
        const size_t at = (size_t)pos_s[n] * half + j;
        const double co = a.cos[at], si = a.sin[at];
        return d < half ? v * co - xs[d + half] * si : v * co + xs[j] * si;
    };
    double z[4] = {0.0, 0.0, 0.0, 0.0}, top = 0.0;   // z: the last four values formed, all of the thread's where there are no more
    auto form = [&](int d0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = d0 + i < dim ? value(d0 + i) : 0.0;
    };
    if (row >= 0)
        for (int d0 = 4 * e; d0 < dim; d0 += 4 * tp)
        {
            form(d0);
#pragma unroll
            for (int i = 0; i < 4; ++i) top = larger(fabs(z[i]), top);
        }
    for (int o = 1; o < tp; o *= 2) top = larger(__shfl_xor(top, o, 64), top);
    if (row < 0) return;
    const float scale = scale_of(top);
    signed char* to = (kind == 0 ? a.c.K : a.c.V) + (long)row * a.c.t.row + (long)h * dim;
    for (int d0 = 4 * e; d0 < dim; d0 += 4 * tp)
    {
        if (dim > 4 * tp) form(d0);
        int b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = byte_of(z[i], scale);
        if (a.words)
            *reinterpret_cast<unsigned*>(to + d0) =
                (b[0] & 255u) | (b[1] & 255u) << 8 | (b[2] & 255u) << 16 | (unsigned)b[3] << 24;
        else
            for (int i = 0; i < 4 && d0 + i < dim; ++i) to[d0 + i] = (signed char)b[i];
    }
    if (e == 0) (kind == 0 ? a.c.K_scale : a.c.V_scale)[(size_t)row * heads + h] = scale;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// x / scale to the nearest integer, from a product with the reciprocal: of a quotient below 128 that is off by 2^-45 at most,
// so that only next to a border of two bytes the division is made.
__device__ __forceinline__ int byte_of(double x, float scale, double inverse)
{
    const double y = x * inverse, n = rint(y);
    if (__builtin_expect(fabs(fabs(y - n) - 0.5) < 0x1p-30 || !(fabs(n) <= 127.0), 0)) return byte_of(x, scale);
    return (int)n;
}
// The largest of N neighbouring lanes' numbers in all of them (rows of 16 lanes and below), none NaN.
template <int CTRL> __device__ __forceinline__ double max_dpp(double x)
{
    const auto b = __builtin_bit_cast(unsigned long long, x);
    const int lo = (int)(unsigned)b, hi = (int)(unsigned)(b >> 32);
    const unsigned l2 = __builtin_amdgcn_update_dpp(lo, lo, CTRL, 15, 15, false), h2 = __builtin_amdgcn_update_dpp(hi, hi, CTRL, 15, 15, false);
    return fmax(x, __builtin_bit_cast(double, (unsigned long long)h2 << 32 | l2));
}
__device__ __forceinline__ double max_of_lanes(double x, int log2_n)
{
    if (log2_n > 0) x = max_dpp<0xb1>(x);    // lanes 1, 0, 3, 2 of each 4
    if (log2_n > 1) x = max_dpp<0x4e>(x);    // 2, 3, 0, 1
    if (log2_n > 2) x = max_dpp<0x141>(x);   // each 8 mirrored
    if (log2_n > 3) x = max_dpp<0x140>(x);   // each 16 mirrored
    if (log2_n > 4) x = fmax(x, __shfl_xor(x, 16, 64));
    return x;
}

// Tokens a row each on every side, 16-byte aligned: a thread takes 4 neighbouring values of a head and the 4 that they turn
// with (j and j + rope_dim / 2), or two neighbouring fours of what is not turned; 2^log2_group neighbouring lanes a head.
// Bound by HBM: 4999 tokens of 8 + 8 + 32 heads of 128 (210 MB) take 38 us,
// 5.5 TB/s; through the tiles of the kernel above 80.
__global__ __launch_bounds__(256) void k_kv8_append_rows(Store8Args a)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const unsigned at = (unsigned)(i >> a.log2_group), piece = (unsigned)i & ((1u << a.log2_group) - 1);   // at: token and head slot
    const unsigned n = a.by_slots.div(at), slot = at - n * a.by_slots.d, heads = a.c.t.heads;
    if (n >= a.tokens.n) return;   // whole groups
    const int kind = slot < heads ? 0 : slot < 2 * heads ? 1 : 2, dim = a.c.t.dim;
    const unsigned h = kind == 0 ? slot : kind == 1 ? slot - heads : slot - 2 * heads;
    const int half = kind == 1 ? 0 : a.half, turned = half / 4;
    const bool turn = (int)piece < turned;
    const int d0 = turn ? 4 * piece : 2 * half + 8 * (piece - turned), d1 = turn ? d0 + half : d0 + 4;
    const Features& x = kind == 0 ? a.k : kind == 1 ? a.v : a.q;
    const float* xp = x.p + (long)n * x.t + (long)h * dim;
    f32x4 x0 = {0.0f, 0.0f, 0.0f, 0.0f}, x1 = x0;
    if (d0 < dim) x0 = *reinterpret_cast<const f32x4*>(xp + d0);
    if (d1 < dim) x1 = *reinterpret_cast<const f32x4*>(xp + d1);
    unsigned pos;
    const int row = a.tokens.row(a.c.t, n, pos);
    if (row < 0) return;
    f32x4 co = {1.0f, 1.0f, 1.0f, 1.0f}, si = {0.0f, 0.0f, 0.0f, 0.0f};
    if (turn)
    {
        co = *reinterpret_cast<const f32x4*>(a.cos + (size_t)pos * half + d0);
        si = *reinterpret_cast<const f32x4*>(a.sin + (size_t)pos * half + d0);
    }
    if (kind == 2)
    {
        if (turn)
        {
            const f32x4 y0 = x0 * co - x1 * si;
            x1 = x1 * co + x0 * si;
            x0 = y0;
        }
        float* o = a.out.p + (long)n * a.out.t + (long)h * dim;
        if (d0 < dim) *reinterpret_cast<f32x4*>(o + d0) = x0;
        if (d1 < dim) *reinterpret_cast<f32x4*>(o + d1) = x1;
        return;
    }
    double y[8], top = 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        y[e] = x0[e];
        y[4 + e] = x1[e];
        if (turn)
        {
            const double u = y[e], v = y[4 + e], c = co[e], s = si[e];
            y[e] = u * c - v * s;
            y[4 + e] = v * c + u * s;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmax(top, fabs(y[e]) < __builtin_inf() ? fabs(y[e]) : __builtin_inf());   // NaN too
    top = max_of_lanes(top, a.log2_group);
    const float scale = scale_of(top);
    const double inverse = 1.0 / (double)scale;
    signed char* to = (kind == 0 ? a.c.K : a.c.V) + (long)row * a.c.t.row + (long)h * dim;
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        w[e / 4] |= (scale > 0.0f ? (unsigned)byte_of(y[e], scale, inverse) & 255u : 0u) << 8 * (e % 4);
    if (d0 < dim) *reinterpret_cast<unsigned*>(to + d0) = w[0];
    if (d1 < dim) *reinterpret_cast<unsigned*>(to + d1) = w[1];
    if (piece == 0) (kind == 0 ? a.c.K_scale : a.c.V_scale)[(size_t)row * heads + h] = scale;
}

struct Read8Args
{
    Pages8 c;
    Features k, v;
    Tokens tokens;
    int log2_lanes;
    FastDiv by_pieces, by_groups;   // where tokens are rows: fours of a head, kHeads heads of keys and values
};

// The same tiles the other way: bytes in the order of the cache, floats in the order of the output.
__global__ __launch_bounds__(256) void k_kv8_read(Read8Args a)
{
    extern __shared__ float tile_s[];   // [token][dim + 1]
    __shared__ int row_s[kTokens];
    const int t = threadIdx.x, dim = a.c.t.dim, ld = dim + 1;
    const unsigned n0 = blockIdx.x * kTokens, heads = a.c.t.heads, y = blockIdx.y;
    const int nt = min((unsigned)kTokens, a.tokens.n - n0);
    const bool keys = y < heads;
    const unsigned h = keys ? y : y - heads;
    const Features& x = keys ? a.k : a.v;
    if (!x.p) return;
    if (t < nt)
    {
        unsigned pos;
        row_s[t] = a.tokens.row(a.c.t, n0 + t, pos);
    }
    __syncthreads();
    for (int n = t >> 6; n < nt; n += 4)
    {
        const int row = row_s[n];
        if (row < 0) continue;
        const signed char* from = (keys ? a.c.K : a.c.V) + (long)row * a.c.t.row + (long)h * dim;
        const float scale = (keys ? a.c.K_scale : a.c.V_scale)[(size_t)row * heads + h];
        for (int d = t & 63; d < dim; d += 64) tile_s[n * ld + d] = (float)from[d] * scale;
    }
    __syncthreads();
    float* xp = x.p + (long)n0 * x.t + (long)h * dim * x.f;
    if (x.f == 1)
    {
        for (int n = t >> 6; n < nt; n += 4)
            if (row_s[n] >= 0)
                for (int d = t & 63; d < dim; d += 64) xp[(long)n * x.t + d] = tile_s[n * ld + d];
    }
    else if (const int n = t & ((1 << a.log2_lanes) - 1); n < nt && row_s[n] >= 0)
        for (int d = t >> a.log2_lanes; d < dim; d += 256 >> a.log2_lanes) xp[(long)n * x.t + (long)d * x.f] = tile_s[n * ld + d];
}

// Tokens a row each, 16-byte aligned: a thread takes 4 neighbouring values of kHeads heads of a token, whose row it looks up
// once. 9 sequences of 2500 to 5000 positions, 8 heads of 128 (308 MB): 64 us, 4.8 TB/s;
// through the tiles of the kernel above 117.
constexpr int kHeads = 4;
__global__ __launch_bounds__(256) void k_kv8_read_rows(Read8Args a)
{
    const unsigned i = blockIdx.x * 256 + threadIdx.x, at = a.by_pieces.div(i), d = 4 * (i - at * a.by_pieces.d);
    const unsigned n = a.by_groups.div(at), slot0 = kHeads * (at - n * a.by_groups.d), heads = a.c.t.heads, dim = a.c.t.dim;
    if (n >= a.tokens.n) return;
    unsigned pos;
    const int row = a.tokens.row(a.c.t, n, pos);
    if (row < 0) return;
    unsigned x[kHeads];
    float scale[kHeads];
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
    {
        const unsigned slot = min(slot0 + k, 2 * heads - 1), h = slot < heads ? slot : slot - heads;
        x[k] = *reinterpret_cast<const unsigned*>((slot < heads ? a.c.K : a.c.V) + (long)row * a.c.t.row + (long)h * dim + d);
        scale[k] = (slot < heads ? a.c.K_scale : a.c.V_scale)[(size_t)row * heads + h];
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
    {
        const unsigned slot = slot0 + k, h = slot < heads ? slot : slot - heads;
        const Features& to = slot < heads ? a.k : a.v;
        if (slot >= 2 * heads || !to.p) continue;
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (float)(signed char)(x[k] >> 8 * e) * scale[k];
        *reinterpret_cast<f32x4*>(to.p + (long)n * to.t + (long)h * dim + d) = y;
    }
}

int lanes_along_tokens(size_t tokens)
{
    int n = 0;
    while (n < 5 && ((size_t)1 << n) < tokens) ++n;
    static_assert(kTokens == 1 << 5);
    return n;
}

} // namespace
} // namespace nnhip

using namespace nnhip;

extern "C" int nnhip_kv8_append(const nnhip_kv8_pages* c, const float* k, long k_t, long k_f, const float* v, long v_t,
                                long v_f, const float* q, long q_t, long q_f, float* q_out, long o_t, long o_f,
                                size_t q_heads, size_t tokens, const float* seq, const float* pos, const float* cos,
                                const float* sin, size_t rope_rows, size_t rope_dim, void* stream)
{
    if (!pages8_ok(c, kWidest)) return -1;
    if (tokens == 0) return 0;
    if (c->K == c->V || c->K_scale == c->V_scale || static_cast<void*>(c->K) == c->K_scale || static_cast<void*>(c->V) == c->V_scale ||
        static_cast<void*>(c->K) == c->V_scale || static_cast<void*>(c->V) == c->K_scale || !k || !v || !pos ||
        (q == nullptr) != (q_out == nullptr) || tokens > kMaxIndex || k_t < 0 || k_f < 0 || v_t < 0 || v_f < 0 || q_t < 0 ||
        q_f < 0 || o_t < 0 || o_f < 0 || (q && (q_heads == 0 || q_heads > kMaxIndex)) || (cos == nullptr) != (sin == nullptr) ||
        rope_dim % 2 != 0 || rope_dim > c->dim || (cos ? rope_rows == 0 || rope_rows > kMaxIndex || rope_dim == 0 : rope_dim != 0))
        return -1;
    const size_t y = 2 * c->heads + (q ? q_heads : 0);
    if (y > 65535) return -1;
    Store8Args a{};
    a.c = pages8_of(*c);
    a.k = {const_cast<float*>(k), k_t, k_f};
    a.v = {const_cast<float*>(v), v_t, v_f};
    a.q = {const_cast<float*>(q), q_t, q_f};
    a.out = {q_out, o_t, o_f};
    a.tokens = {seq, pos, static_cast<unsigned>(tokens), cos ? static_cast<unsigned>(rope_rows) : 0};
    a.cos = cos;
    a.sin = sin;
    a.half = static_cast<int>(rope_dim / 2);
    a.log2_lanes = lanes_along_tokens(tokens);
    auto aligned4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
    a.words = c->dim % 4 == 0 && c->row % 4 == 0 && aligned4(c->K) && aligned4(c->V);
    auto s = static_cast<hipStream_t>(stream);
    auto rows_of_4 = [](const float* p, long t, long f) { return !p || (f == 1 && t % 4 == 0 && aligned16(p)); };
    const size_t turned = rope_dim / 8, rest = c->dim - rope_dim, all_v = (c->dim + 7) / 8;
    const size_t pieces = turned + (rest + 7) / 8 > all_v ? turned + (rest + 7) / 8 : all_v;
    while (((size_t)1 << a.log2_group) < pieces) ++a.log2_group;
    const size_t threads = tokens * y << a.log2_group;
    // Heads of tokens are divided by their slots: those of the last workgroup's threads, too, are below 2^31 (FastDiv).
    if (tokens * y + 255 < 0x80000000u && a.words && rope_dim % 8 == 0 && rows_of_4(k, k_t, k_f) && rows_of_4(v, v_t, v_f) && rows_of_4(q, q_t, q_f) &&
        rows_of_4(q_out, o_t, o_f) && (!cos || (aligned16(cos) && aligned16(sin))) && threads / 256 < kGridMost && a.log2_group <= 5)
    {
        a.by_slots = FastDiv(static_cast<unsigned>(y));
        hipLaunchKernelGGL(k_kv8_append_rows, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, s, a);
        return launch_status();
    }
    const dim3 grid(static_cast<unsigned>((tokens + kTokens - 1) / kTokens), static_cast<unsigned>(y));
    hipLaunchKernelGGL(k_kv8_append, grid, dim3(256), kTokens * (c->dim + 1) * sizeof(float), s, a);
    return launch_status();
}

extern "C" int nnhip_kv8_read(const nnhip_kv8_pages* c, float* k, long k_t, long k_f, float* v, long v_t, long v_f,
                              size_t tokens, const float* seq, const float* pos, void* stream)
{
    if (!pages8_ok(c, kWidest)) return -1;
    if (tokens == 0 || (!k && !v)) return 0;
    if (!pos || tokens > kMaxIndex || k_t < 0 || k_f < 0 || v_t < 0 || v_f < 0 || 2 * c->heads > 65535) return -1;
    Read8Args a{};
    a.c = pages8_of(*c);
    a.k = {k, k_t, k_f};
    a.v = {v, v_t, v_f};
    a.tokens = {seq, pos, static_cast<unsigned>(tokens), 0};
    a.log2_lanes = lanes_along_tokens(tokens);
    auto rows_of_4 = [](const float* p, long t, long f) { return !p || (f == 1 && t % 4 == 0 && aligned16(p)); };
    const size_t groups = (2 * c->heads + kHeads - 1) / kHeads, threads = tokens * groups * (c->dim / 4);
    if (c->dim % 4 == 0 && c->row % 4 == 0 && ((reinterpret_cast<uintptr_t>(c->K) | reinterpret_cast<uintptr_t>(c->V)) & 3) == 0 &&
        rows_of_4(k, k_t, k_f) && rows_of_4(v, v_t, v_f) && threads + 256 < 0x80000000u)
    {
        a.by_pieces = FastDiv(static_cast<unsigned>(c->dim / 4));
        a.by_groups = FastDiv(static_cast<unsigned>(groups));
        hipLaunchKernelGGL(k_kv8_read_rows, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream), a);
        return launch_status();
    }
    const dim3 grid(static_cast<unsigned>((tokens + kTokens - 1) / kTokens), static_cast<unsigned>(2 * c->heads));
    hipLaunchKernelGGL(k_kv8_read, grid, dim3(256), kTokens * (c->dim + 1) * sizeof(float), static_cast<hipStream_t>(stream), a);
    return launch_status();
}
