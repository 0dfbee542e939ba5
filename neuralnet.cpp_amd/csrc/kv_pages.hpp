// kv_pages.hpp — paged key/value caches (nnhip_kv_pages) as the kernels see them.
#pragma once

#include "common.hpp"
#include "nnhip_kernels.h"

namespace nnhip
{

constexpr size_t kMaxIndex = (size_t)1 << 24;   // integers that a float holds

// n / d for n < 2^31 and d < 2^31 by one multiplication: with s = ceil(log2 d) and mul = ceil(2^(31+s) / d),
// n mul = (n / d) 2^(31+s) + n e / d, e < d <= 2^s, and n e < 2^(31+s) keeps the floor.
struct FastDiv
{
    unsigned mul, shift, d;
    FastDiv() = default;
    explicit FastDiv(unsigned div) : d(div)
    {
        unsigned s = 0;
        while (s < 31 && (1ull << s) < div) ++s;
        shift = 31 + s;
        mul = static_cast<unsigned>(((1ull << shift) + div - 1) / div);
    }
    __device__ __forceinline__ unsigned div(unsigned n) const
    {
        return static_cast<unsigned>(((unsigned long long)n * mul) >> shift);
    }
};

struct Pages
{
    float* K;
    float* V;
    const float* table;
    unsigned batch, width, pages, heads, dim;
    long row;
    FastDiv page;

    // The table's entry for position pos of sequence b (the last one past the table's end), and the row that it
    // names, -1 where there is none. Neither branches: the kernels load entries ahead of their use, and a branch
    // would make the wait for one a wait for every load behind it.
    __device__ __forceinline__ float entry_of(unsigned b, unsigned pos) const
    {
        return table[(size_t)b * width + min(page.div(pos), width - 1)];
    }
    __device__ __forceinline__ int row_in(float entry, unsigned pos) const
    {
        const unsigned i = page.div(pos), p = (unsigned)(int)entry;
        const bool ok = i < width && entry > -1.0f && entry < (float)pages;   // pages <= 2^24 is exact
        return ok ? (int)(p * page.d + (pos - i * page.d)) : -1;
    }
    __device__ __forceinline__ int row_of(unsigned b, unsigned pos) const { return row_in(entry_of(b, pos), pos); }
};

// A length held as a float: negative and NaN are 0, at most `most`.
__device__ __forceinline__ int length_of(float f, int most)
{
    if (!(f >= 1.0f)) return 0;
    return f >= (float)most ? most : (int)f;
}

constexpr size_t kGridMost = 0xffffff;   // workgroups of 256: a launch has fewer than 2^32 threads along an axis

// The sizes that every entry point asks for: the kernels count pages, rows and a row's values in 32 bits.
inline bool pages_ok(const nnhip_kv_pages* c, size_t max_dim)
{
    return c && c->K && c->V && c->table && c->batch > 0 && c->width > 0 && c->pages > 0 && c->page > 0 &&
           c->heads > 0 && c->dim > 0 && c->dim <= max_dim && c->batch <= kMaxIndex && c->pages <= kMaxIndex &&
           c->page <= kMaxIndex && c->pages * c->page < (size_t)0x80000000u && c->width <= kMaxIndex && c->width * c->page <= kMaxIndex &&
           c->heads <= kMaxIndex && c->heads * c->dim < (size_t)0x80000000u && c->row >= c->heads * c->dim && c->row <= ((size_t)1 << 32);
}

inline Pages pages_of(const nnhip_kv_pages& c)
{
    return Pages{c.K,
                 c.V,
                 c.table,
                 static_cast<unsigned>(c.batch),
                 static_cast<unsigned>(c.width),
                 static_cast<unsigned>(c.pages),
                 static_cast<unsigned>(c.heads),
                 static_cast<unsigned>(c.dim),
                 static_cast<long>(c.row),
                 FastDiv(static_cast<unsigned>(c.page))};
}

// An 8-bit cache (nnhip_kv8_pages): the table's part as Pages has it (its K and V are not set), a byte a value in rows
// t.row apart, and a scale a row and head.
struct Pages8
{
    Pages t;
    signed char *K, *V;
    float *K_scale, *V_scale;
};

// A scale as attention takes it: one that is not finite is NaN, so that no byte of 0 and no weight of 0 hides it.
__device__ __forceinline__ float scale_or_nan(float s) { return fabsf(s) <= kMaxF ? s : __builtin_nanf(""); }

inline bool pages8_ok(const nnhip_kv8_pages* c, size_t max_dim)
{
    if (!c || !c->K || !c->V || !c->K_scale || !c->V_scale) return false;
    auto* some = c->K_scale;   // stands for the caches in the checks of the sizes
    const nnhip_kv_pages t{some, some, c->table, c->batch, c->width, c->pages, c->page, c->heads, c->dim, c->row};
    return pages_ok(&t, max_dim);
}

inline Pages8 pages8_of(const nnhip_kv8_pages& c)
{
    const nnhip_kv_pages t{nullptr, nullptr, c.table, c.batch, c.width, c.pages, c.page, c.heads, c.dim, c.row};
    return Pages8{pages_of(t), c.K, c.V, c.K_scale, c.V_scale};
}

// The tokens of a call that name positions of sequences. rope_rows: rows of the rotation's tables, 0 without one.
struct Tokens
{
    const float *seq, *pos;
    unsigned n, rope_rows;

    // Where token i goes: its row, or -1 for padding, and its position.
    __device__ __forceinline__ int row(const Pages& c, unsigned i, unsigned& at) const
    {
        size_t p = 0, b = i;
        const bool seq_ok = seq ? row_index(seq[i], c.batch, b) : i < c.batch;
        const bool ok = row_index(pos[i], kMaxIndex, p) && seq_ok && (!rope_rows || p < rope_rows);
        at = (unsigned)p;
        return ok ? c.row_of((unsigned)b, at) : -1;
    }
};

// Features of tokens: floats from a token and from a feature to the next.
struct Features
{
    float* p;
    long t, f;
};

} // namespace nnhip
