// k_kv_pages.hip — paged caches: new tokens' keys and values stored, rotated on
// the way, and the caches after a beam search's selection.
#include "kv_pages.hpp"

namespace nnhip
{
namespace
{

constexpr int kAppendTokens = 32;   // tokens of a tile
constexpr int kAppendDim = 256;     // widest head

struct HeadsView
{
    const float* p;
    long t, f;   // floats from a token and from a feature to the next
};

struct AppendArgs
{
    Pages c;
    HeadsView k, v, q;
    float* out;
    long o_t, o_f;
    const float *seq, *pos, *cos, *sin;
    unsigned tokens, tile, rope_rows;
    int half;   // rope_dim / 2
};

// One tile of tokens of one head: k heads, then v heads, then q heads along blockIdx.y. The tile is read in the
// order of its own layout into LDS and written in the order of the destination's, so either layout of either
// side gives whole lines.
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs a)
{
    extern __shared__ float tile_s[];   // [token][dim + 1]
    __shared__ int row_s[kAppendTokens];
    __shared__ unsigned pos_s[kAppendTokens];
    const int t = threadIdx.x, dim = a.c.dim, ld = dim + 1;
    const unsigned n0 = blockIdx.x * a.tile, heads = a.c.heads;
    const int nt = min(a.tile, a.tokens - n0);
    const unsigned y = blockIdx.y;
    const int kind = y < heads ? 0 : y < 2 * heads ? 1 : 2;
    const unsigned h = kind == 0 ? y : kind == 1 ? y - heads : y - 2 * heads;
    const HeadsView x = kind == 0 ? a.k : kind == 1 ? a.v : a.q;
    const float* xp = x.p + (long)n0 * x.t + (long)h * dim * x.f;
    if (t < nt)
    {
        const unsigned n = n0 + t;
        size_t p = 0, b = n;
        int row = -1;
        const bool seq_ok = a.seq ? row_index(a.seq[n], a.c.batch, b) : n < a.c.batch;
        if (seq_ok && row_index(a.pos[n], kMaxIndex, p) && (!a.cos || p < a.rope_rows)) row = a.c.row_of(b, p);
        row_s[t] = row;
        pos_s[t] = (unsigned)p;
    }
    const int count = nt * dim;
    for (int i = t; i < count; i += 256)
    {
        const int n = x.f == 1 ? i / dim : i % nt, d = x.f == 1 ? i % dim : i / nt;
        tile_s[n * ld + d] = xp[(long)n * x.t + (long)d * x.f];
    }
    __syncthreads();
    const int half = kind == 1 ? 0 : a.half;
    const bool by_token = kind != 2 || a.o_f == 1;
    for (int i = t; i < count; i += 256)
    {
        const int n = by_token ? i / dim : i % nt, d = by_token ? i % dim : i / nt;
        const int row = row_s[n];
        if (row < 0) continue;
        float v = tile_s[n * ld + d];
        if (d < 2 * half)
        {
            const int j = d < half ? d : d - half;
            const size_t at = (size_t)pos_s[n] * half + j;
            const float co = a.cos[at], si = a.sin[at];
            v = d < half ? v * co - tile_s[n * ld + d + half] * si : v * co + tile_s[n * ld + j] * si;
        }
        if (kind == 2)
            a.out[(long)(n0 + n) * a.o_t + ((long)h * dim + d) * a.o_f] = v;
        else
            (kind == 0 ? a.c.K : a.c.V)[(long)row * a.c.row + (long)h * dim + d] = v;
    }
}

constexpr int kReorderLayers = 32;   // caches of a launch
constexpr int kReorderRows = 4;      // rows that a workgroup copies

struct ReorderArgs
{
    Pages c;
    const float *parent, *len, *fresh;
    float *table_out, *len_out;
    unsigned out_batch, table_blocks, copy_rows, n_mem;   // copy_rows: row groups of a page
    float* mem[2 * kReorderLayers];
};

// What the new sequence b continues: its parent's row of the table, length, full pages and rows of the last.
struct Continued
{
    bool ok;
    size_t parent;
    unsigned n, full, tail;
};
__device__ __forceinline__ Continued continued(const ReorderArgs& a, unsigned b)
{
    Continued r{false, 0, 0, 0, 0};
    r.ok = row_index(a.parent[b], a.c.batch, r.parent);
    if (!r.ok) return r;
    r.n = length_of(a.len[r.parent], (int)(a.c.width * a.c.page.d));
    r.full = a.c.page.div(r.n);
    r.tail = r.n - r.full * a.c.page.d;
    return r;
}

__global__ __launch_bounds__(256) void k_kv_reorder(ReorderArgs a)
{
    const int t = threadIdx.x;
    if (blockIdx.x < a.table_blocks)
    {
        const size_t i = (size_t)blockIdx.x * 256 + t;
        if (i >= (size_t)a.out_batch * a.c.width) return;
        const unsigned b = (unsigned)(i / a.c.width), e = (unsigned)(i % a.c.width);
        const Continued r = continued(a, b);
        if (e == 0) a.len_out[b] = (float)r.n;
        float v = -1.0f;
        size_t p;
        if (r.ok && (e < r.full || (e == r.full && !a.fresh && r.tail))) v = a.c.table[r.parent * a.c.width + e];
        else if (r.ok && e == r.full && a.fresh && row_index(a.fresh[b], a.c.pages, p)) v = (float)p;
        a.table_out[i] = v;
        return;
    }
    // Rows [r0, r0 + kReorderRows) of the page in progress of new sequence b, in one cache.
    unsigned i = blockIdx.x - a.table_blocks;
    const unsigned r0 = (i % a.copy_rows) * kReorderRows;
    i /= a.copy_rows;
    const unsigned mi = i % a.n_mem, b = i / a.n_mem;
    const Continued r = continued(a, b);
    if (!r.ok || r0 >= r.tail || r.full >= a.c.width) return;
    size_t dst, src;
    if (!row_index(a.fresh[b], a.c.pages, dst) || !row_index(a.c.table[r.parent * a.c.width + r.full], a.c.pages, src) ||
        src == dst)
        return;
    float* m = a.mem[mi];
    const unsigned rows = min(r.tail - r0, (unsigned)kReorderRows), len = a.c.heads * a.c.dim;
    const float* s = m + ((long)src * a.c.page.d + r0) * a.c.row;
    float* d = m + ((long)dst * a.c.page.d + r0) * a.c.row;
    for (unsigned k = 0; k < rows; ++k)
        for (unsigned j = t; j < len; j += 256) d[(long)k * a.c.row + j] = s[(long)k * a.c.row + j];
}

bool overlap(const float* a, size_t na, const float* b, size_t nb)
{
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb * sizeof(float) && y < x + na * sizeof(float);
}

} // namespace
} // namespace nnhip

using namespace nnhip;

extern "C" int nnhip_kv_append(const nnhip_kv_pages* c, const float* k, long k_t, long k_f, const float* v, long v_t,
                               long v_f, const float* q, long q_t, long q_f, float* q_out, long o_t, long o_f,
                               size_t q_heads, size_t tokens, const float* seq, const float* pos, const float* cos,
                               const float* sin, size_t rope_rows, size_t rope_dim, void* stream)
{
    if (!pages_ok(c, kAppendDim)) return -1;
    if (tokens == 0) return 0;
    if (!k || !v || !pos || (q == nullptr) != (q_out == nullptr) || tokens > kMaxIndex || k_t < 0 || k_f < 0 ||
        v_t < 0 || v_f < 0 || q_t < 0 || q_f < 0 || o_t < 0 || o_f < 0 || (q && (q_heads == 0 || q_heads > kMaxIndex)) ||
        (cos == nullptr) != (sin == nullptr) || rope_dim % 2 != 0 || rope_dim > c->dim ||
        (cos ? rope_rows == 0 || rope_rows > kMaxIndex || rope_dim == 0 : rope_dim != 0))
        return -1;
    const size_t y = 2 * c->heads + (q ? q_heads : 0);
    if (y > 65535) return -1;
    AppendArgs a{pages_of(*c), {k, k_t, k_f}, {v, v_t, v_f}, {q, q_t, q_f}, q_out, o_t, o_f, seq, pos, cos, sin,
                 static_cast<unsigned>(tokens), kAppendTokens, static_cast<unsigned>(rope_rows),
                 static_cast<int>(rope_dim / 2)};
    const dim3 grid(static_cast<unsigned>((tokens + a.tile - 1) / a.tile), static_cast<unsigned>(y));
    hipLaunchKernelGGL(k_kv_append, grid, dim3(256), a.tile * (c->dim + 1) * sizeof(float),
                       static_cast<hipStream_t>(stream), a);
    return launch_status();
}

extern "C" int nnhip_kv_reorder(const nnhip_kv_pages* layers, size_t n_layers, const float* parent, const float* len,
                                const float* fresh, size_t out_batch, float* table_out, float* len_out, void* stream)
{
    if (n_layers == 0 || !layers) return -1;
    for (size_t i = 0; i < n_layers; ++i)
    {
        if (!pages_ok(&layers[i], kMaxIndex)) return -1;
        const nnhip_kv_pages &x = layers[i], &y = layers[0];
        if (x.table != y.table || x.batch != y.batch || x.width != y.width || x.pages != y.pages || x.page != y.page ||
            x.heads != y.heads || x.dim != y.dim || x.row != y.row)
            return -1;
    }
    const nnhip_kv_pages& c = layers[0];
    if (out_batch == 0) return 0;
    if (!parent || !len || !table_out || !len_out || out_batch > kMaxIndex ||
        overlap(c.table, c.batch * c.width, table_out, out_batch * c.width))
        return -1;
    ReorderArgs a{};
    a.c = pages_of(c);
    a.parent = parent;
    a.len = len;
    a.fresh = fresh;
    a.table_out = table_out;
    a.len_out = len_out;
    a.out_batch = static_cast<unsigned>(out_batch);
    const bool copy = fresh && c.page > 1;
    a.copy_rows = copy ? static_cast<unsigned>((c.page - 1 + kReorderRows - 1) / kReorderRows) : 0;
    for (size_t at = 0; at < n_layers; at += kReorderLayers)
    {
        const size_t n = n_layers - at < kReorderLayers ? n_layers - at : kReorderLayers;
        for (size_t i = 0; i < n; ++i)
        {
            a.mem[2 * i] = layers[at + i].K;
            a.mem[2 * i + 1] = layers[at + i].V;
        }
        a.n_mem = static_cast<unsigned>(2 * n);
        const size_t tables = at == 0 ? (out_batch * c.width + 255) / 256 : 0;
        const size_t blocks = tables + (size_t)a.copy_rows * a.n_mem * out_batch;
        if (blocks == 0) break;
        if (blocks > 0x7fffffffu) return -1;
        a.table_blocks = static_cast<unsigned>(tables);
        hipLaunchKernelGGL(k_kv_reorder, dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
        if (int rc = launch_status()) return rc;
    }
    return 0;
}
