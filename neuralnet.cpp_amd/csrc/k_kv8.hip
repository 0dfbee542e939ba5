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
// of its own layout into LDS; 8 threads then share a token's head.
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
    const int n = t >> 3, e = t & 7, row = n < nt ? row_s[n] : -1;
    const float* xs = tile_s + n * ld;
    auto value = [&](int d) -> double {
        const double v = xs[d];
        if (d >= 2 * half) return v;
        const int j = d < half ? d : d - half;
        const size_t at = (size_t)pos_s[n] * half + j;
        const double co = a.cos[at], si = a.sin[at];
        return d < half ? v * co - xs[d + half] * si : v * co + xs[j] * si;
    };
    double top = 0.0;
    if (row >= 0)
        for (int d0 = 4 * e; d0 < dim; d0 += 32)
            for (int d = d0; d < min(d0 + 4, dim); ++d) top = larger(fabs(value(d)), top);
    for (int o = 1; o < 8; o *= 2) top = larger(__shfl_xor(top, o, 64), top);
    if (row < 0) return;
    const float scale = scale_of(top);
    signed char* to = (kind == 0 ? a.c.K : a.c.V) + (long)row * a.c.t.row + (long)h * dim;
    for (int d0 = 4 * e; d0 < dim; d0 += 32)
    {
        int b[4];
        for (int i = 0; i < 4; ++i) b[i] = d0 + i < dim ? byte_of(value(d0 + i), scale) : 0;
        if (a.words)
            *reinterpret_cast<unsigned*>(to + d0) =
                (b[0] & 255u) | (b[1] & 255u) << 8 | (b[2] & 255u) << 16 | (unsigned)b[3] << 24;
        else
            for (int i = 0; i < 4 && d0 + i < dim; ++i) to[d0 + i] = (signed char)b[i];
    }
    if (e == 0) (kind == 0 ? a.c.K_scale : a.c.V_scale)[(size_t)row * heads + h] = scale;
}

struct Read8Args
{
    Pages8 c;
    Features k, v;
    Tokens tokens;
    int log2_lanes;
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
    const dim3 grid(static_cast<unsigned>((tokens + kTokens - 1) / kTokens), static_cast<unsigned>(y));
    hipLaunchKernelGGL(k_kv8_append, grid, dim3(256), kTokens * (c->dim + 1) * sizeof(float), static_cast<hipStream_t>(stream), a);
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
    const dim3 grid(static_cast<unsigned>((tokens + kTokens - 1) / kTokens), static_cast<unsigned>(2 * c->heads));
    hipLaunchKernelGGL(k_kv8_read, grid, dim3(256), kTokens * (c->dim + 1) * sizeof(float), static_cast<hipStream_t>(stream), a);
    return launch_status();
}
