// f16_parts.hpp — float32 products on the float16 matrix cores, from two parts of
// each factor, and what the kernels that form them share.
//
// A float32 x is scaled by a power of two so that the largest of its row lies in
// [2^14, 2^15) and held as two float16, each the round to nearest of what is
// left: h = f16(x), l = f16(x - h). A float16 has 11 significant bits, so that
// x - h - l is at most 2^-24 |x| (2^-25 where l is denormal: 2^-39 of the row's
// largest). A product is then ah bh + (ah bl + al bh) + [al bl], where the
// bracket, at most 2^-24 |ab|, is left out: three float16 products, exact in the
// matrix core's float32 sum, for a float32 one. Bytes are float16 as they are:
// two products.
#pragma once

#include <hip/hip_runtime.h>

namespace nnhip
{

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

constexpr int kNone = -200;   // exponent of nothing but zeros: below every float's
constexpr int kLeastTop = -108;   // values below 2^kLeastTop are held against that: 2^(17 - kLeastTop) is a float

// Two parts of eight floats that are scaled already. What rounding leaves of a pair, x - f16(x), is exact: the pair's dot
// product with (-1, 0) or (0, -1) added to x, one instruction each.
__device__ __forceinline__ void split2(const floatx8& x, half8& h, half8& l)
{
    unsigned c0 = 0x0000bc00u, c1 = 0xbc000000u;
    asm("" : "+s"(c0));
    asm("" : "+s"(c1));
    const half2_t e0 = __builtin_bit_cast(half2_t, c0), e1 = __builtin_bit_cast(half2_t, c1);
    uintx4 hv, lv;
#pragma unroll
    for (int p = 0; p < 4; ++p)
    {
        const half2_t a = __builtin_convertvector((floatx2){x[2 * p], x[2 * p + 1]}, half2_t);
        const floatx2 left = {__builtin_amdgcn_fdot2(a, e0, x[2 * p], false), __builtin_amdgcn_fdot2(a, e1, x[2 * p + 1], false)};
        hv[p] = __builtin_bit_cast(unsigned, a);
        lv[p] = __builtin_bit_cast(unsigned, __builtin_convertvector(left, half2_t));
    }
    h = __builtin_bit_cast(half8, hv);
    l = __builtin_bit_cast(half8, lv);
}
// Two float16 from two bytes that lie in bits 0-7 and 16-23 (the others 0): 1024 + (byte + 128) is 0x6400 | (byte ^ 0x80).
__device__ __forceinline__ unsigned halves_of(unsigned two)
{
    const half2_t z = __builtin_bit_cast(half2_t, two ^ 0x64806480u) - (half2_t){(_Float16)1152, (_Float16)1152};
    return __builtin_bit_cast(unsigned, z);
}
// e with |x| < 2^e, and 2^(e - 1) <= |x| but for denormals. What is not finite has 129.
__device__ __forceinline__ int exponent_of(float x) { return (int)max(__builtin_bit_cast(unsigned, x) >> 23 & 255u, 1u) - 126; }

// The largest of N neighbouring lanes' numbers, none negative, in all of them: without LDS, which the shuffles take.
template <int CTRL> __device__ __forceinline__ float swap_dpp(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 15, 15, true));
}
template <int CTRL> __device__ __forceinline__ float max_dpp(float x) { return fmaxf(x, swap_dpp<CTRL>(x)); }
template <int N> __device__ __forceinline__ float max_of(float x)
{
    x = max_dpp<0xb1>(x);                           // lanes 1, 0, 3, 2 of each 4
    x = max_dpp<0x4e>(x);                           // 2, 3, 0, 1
    if constexpr (N >= 8) x = max_dpp<0x141>(x);    // each 8 mirrored
    if constexpr (N >= 16) x = max_dpp<0x140>(x);   // each 16 mirrored
    if constexpr (N >= 32)
    {
        const int a = __builtin_bit_cast(int, x);   // 4 rows of 16 lanes, as whole numbers in the order of the floats
        const int lo = max(__builtin_amdgcn_readlane(a, 0), __builtin_amdgcn_readlane(a, 16));
        const int hi = max(__builtin_amdgcn_readlane(a, 32), __builtin_amdgcn_readlane(a, 48));
        if constexpr (N == 64) x = __builtin_bit_cast(float, max(lo, hi));
        else x = __builtin_bit_cast(float, (threadIdx.x & 32) ? hi : lo);
    }
    return x;
}
// Both halves of the wave: f of the lane's value and that of lane l ^ 32.
template <class F> __device__ __forceinline__ float across(float x, F&& f)
{
    unsigned a = __builtin_bit_cast(unsigned, x), b = a;
    asm("" : "+v"(b));   // of one value twice the compiler takes both results to be the same
    const auto z = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    const unsigned lo = z[0], hi = z[1];
    return f(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
// The wave's four rows of 16 lanes: f of the values of lanes l, l ^ 16, l ^ 32 and l ^ 48.
template <class F> __device__ __forceinline__ float across4(float x, F&& f)
{
    unsigned a = __builtin_bit_cast(unsigned, x), b = a;
    asm("" : "+v"(b));
    const auto z = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    const unsigned lo = z[0], hi = z[1];
    return across(f(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)), f);
}
__device__ __forceinline__ float larger_of(float a, float b) { return fmaxf(a, b); }

// Scores. alpha log2(e) is by_m 2^by_e: the query's parts take by_m, and a score, times log2(e), is s f 2^e with s the sum of
// the parts' products, f the key's scale and e the row's exponent. A tile's scales are multiplied by 2^-shift_of them and e is
// raised by it, so that neither s f leaves float32's range where the score does not, nor f has bits below that range: of
// scales above 2^80, of which s f might pass 2^128, it is 64, of nothing but scales below 2^-75 -64, else 0.
constexpr float kFar = 0x1p80f, kNear = 0x1p-75f;
__device__ __forceinline__ int shift_of(unsigned long long far, bool all_near) { return far ? 64 : all_near ? -64 : 0; }

// What weights times values are held against: 2^top, above the largest of these products that the row has met, which shrink
// with a growing score. size: that exponent before it is rounded up, so that no small step is lost.
struct Held
{
    float size = kLeastTop;
    __device__ __forceinline__ int top() const { return (int)ceilf(size); }
};
// Scores grow by `up` bits: what the outputs are multiplied by. The sum of the weights is by 2^-up.
__device__ __forceinline__ float shrink(Held& h, float up)
{
    const int was = h.top();
    h.size = fmaxf(h.size - up, kLeastTop);
    return __builtin_amdgcn_exp2f((float)(was - h.top()) - up);
}
// Products below 2^e have come: what the outputs are multiplied by.
__device__ __forceinline__ float raise(Held& h, int e)
{
    const int was = h.top();
    h.size = fmaxf(h.size, (float)e);
    return __builtin_ldexpf(1.0f, was - h.top());
}
// The largest over the wave of each of 8 numbers a lane, none negative: lane l has the number l % 8's.
__device__ __forceinline__ float max_of_8(const float (&x)[8], int lane)
{
    float a[4], b[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = fmaxf(lane & 4 ? x[4 + i] : x[i], swap_dpp<0x141>(lane & 4 ? x[i] : x[4 + i]));
#pragma unroll
    for (int i = 0; i < 2; ++i) b[i] = fmaxf(lane & 2 ? a[2 + i] : a[i], swap_dpp<0x4e>(lane & 2 ? a[i] : a[2 + i]));
    float r = fmaxf(lane & 1 ? b[1] : b[0], swap_dpp<0xb1>(lane & 1 ? b[0] : b[1]));
    r = max_dpp<0x128>(r);   // each 16 turned by 8
    return across4(r, larger_of);
}

} // namespace nnhip
