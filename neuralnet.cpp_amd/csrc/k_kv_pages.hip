// k_kv_pages.hip — paged caches: new tokens' keys and values stored, rotated on
// the way, and the caches after a beam search's selection.
#include "kv_pages.hpp"

namespace nnhip
{
namespace
{

constexpr int kAppendTokens = 32;   // tokens of a tile
constexpr int kAppendDim = 256;     // widest head

typedef float f32x4 __attribute__((ext_vector_type(4)));

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
    unsigned tokens, rope_rows, head_slots;   // head_slots: k heads, v heads, q heads
    int half, log2_lanes;                     // rope_dim / 2; lanes along a tile's tokens
    unsigned pieces;                          // rows of 4 values that a thread takes two of, of a head
    FastDiv by_pieces, by_slots;
};

// Where token n goes: its row, or -1 for padding, and its position.
__device__ __forceinline__ int append_row(const AppendArgs& a, unsigned n, unsigned& pos)
{
    size_t p = 0, b = n;
    const bool seq_ok = a.seq ? row_index(a.seq[n], a.c.batch, b) : n < a.c.batch;
    const bool ok = row_index(a.pos[n], kMaxIndex, p) && seq_ok && (!a.cos || p < a.rope_rows);
    pos = (unsigned)p;
    return ok ? a.c.row_of((unsigned)b, pos) : -1;
}

// Tokens a row each on every side, 16-byte aligned: a thread takes 4 neighbouring values of a head and the 4 that
// they turn with (j and j + rope_dim / 2), or two neighbouring fours of what is not turned. Both are on their way
// before the position is known. Bound by HBM: 5003 tokens of 8 + 8 + 32 heads of 128 (243 MB) take 42 us, 5.8 TB/s;
// through the tile of the kernel below they took 118.
__global__ __launch_bounds__(256) void k_kv_append_rows(AppendArgs a)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const unsigned at = a.by_pieces.div((unsigned)i), piece = (unsigned)i - at * a.pieces;   // at: token and head slot
    const unsigned n = a.by_slots.div(at), slot = at - n * a.head_slots, heads = a.c.heads;
    if (n >= a.tokens) return;
    const int kind = slot < heads ? 0 : slot < 2 * heads ? 1 : 2, dim = a.c.dim;
    const unsigned h = kind == 0 ? slot : kind == 1 ? slot - heads : slot - 2 * heads;
    const int half = kind == 1 ? 0 : a.half, turned = half / 4;
    const bool turn = (int)piece < turned;
    const int d0 = turn ? 4 * piece : 2 * half + 8 * (piece - turned), d1 = turn ? d0 + half : d0 + 4;
    if (d0 >= dim) return;
    const HeadsView& x = kind == 0 ? a.k : kind == 1 ? a.v : a.q;
    const float* xp = x.p + (long)n * x.t + (long)h * dim;
    f32x4 x0 = *reinterpret_cast<const f32x4*>(xp + d0), x1 = x0;
    if (d1 < dim) x1 = *reinterpret_cast<const f32x4*>(xp + d1);
    unsigned pos;
    const int row = append_row(a, n, pos);
    if (row < 0) return;
    if (turn)
    {
        const f32x4 co = *reinterpret_cast<const f32x4*>(a.cos + (size_t)pos * half + d0);
        const f32x4 si = *reinterpret_cast<const f32x4*>(a.sin + (size_t)pos * half + d0);
        const f32x4 y0 = x0 * co - x1 * si;
        x1 = x1 * co + x0 * si;
        x0 = y0;
    }
    float* o = kind == 2 ? a.out + (long)n * a.o_t : (kind == 0 ? a.c.K : a.c.V) + (long)row * a.c.row;
    o += (long)h * dim;
    *reinterpret_cast<f32x4*>(o + d0) = x0;
    if (d1 < dim) *reinterpret_cast<f32x4*>(o + d1) = x1;
}

// Any layout: one tile of tokens of one head slot (blockIdx.y). The tile is read in the order of its own layout
// into LDS and written in the order of the destination's, so either layout of either side gives whole lines:
// 64 lanes along a token's features, or as many along the tokens as there are, 32 at most. One token each of 4
// sequences (12 heads of 64) takes 4 us: the position, the page and the row wait for one another.
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs a)
{
    extern __shared__ float tile_s[];   // [token][dim + 1]
    __shared__ int row_s[kAppendTokens];
    __shared__ unsigned pos_s[kAppendTokens];
    const int t = threadIdx.x, dim = a.c.dim, ld = dim + 1;
    const unsigned n0 = blockIdx.x * kAppendTokens, heads = a.c.heads;
    const int nt = min((unsigned)kAppendTokens, a.tokens - n0);
    const unsigned y = blockIdx.y;
    const int kind = y < heads ? 0 : y < 2 * heads ? 1 : 2;
    const unsigned h = kind == 0 ? y : kind == 1 ? y - heads : y - 2 * heads;
    const HeadsView& x = kind == 0 ? a.k : kind == 1 ? a.v : a.q;
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
    if (t < nt) row_s[t] = append_row(a, n0 + t, pos_s[t]);
    __syncthreads();
    const int half = kind == 1 ? 0 : a.half;
    over(kind != 2 || a.o_f == 1, [&](int n, int d) {
        const int row = row_s[n];
        if (row < 0) return;
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
    });
}

constexpr int kReorderLayers = 32;   // caches of a launch
constexpr int kReorderRows = 4;      // rows that a workgroup copies

struct ReorderArgs
{
    Pages c;
    const float *parent, *len, *fresh;
    float *table_out, *len_out;
    unsigned out_batch, table_blocks, splits, n_mem;   // splits: workgroups that a page's rows are cut into
    int vec;                                              // rows are copied 4 floats at a time
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

// Tables, lengths and pages in one launch, whose time is that of the parent, its length, its page and its rows waiting
// for one another: 8 layers of 48 beams, pages of 32 rows of 8 heads of 128, take 5.1 us (13 MB: 2.4 us of HBM);
// 15.6 us with a workgroup a page that copied row by row.
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
    // The page in progress of new sequence b, in one cache: kReorderRows rows at a time, in turn with the others
    // of the page's workgroups.
    unsigned i = blockIdx.x - a.table_blocks;
    const unsigned split = i % a.splits;
    i /= a.splits;
    const unsigned mi = i % a.n_mem, b = i / a.n_mem;
    const float fresh = a.fresh[b];
    const Continued r = continued(a, b);
    if (!r.ok || r.full >= a.c.width) return;
    size_t dst, src;
    if (!row_index(fresh, a.c.pages, dst) || !row_index(a.c.table[r.parent * a.c.width + r.full], a.c.pages, src) ||
        src == dst)
        return;
    float* m = a.mem[mi];
    const unsigned len = a.c.heads * a.c.dim;
    for (unsigned r0 = split * kReorderRows; r0 < r.tail; r0 += a.splits * kReorderRows)
    {
        const unsigned rows = min(r.tail - r0, (unsigned)kReorderRows);
        const float* s = m + ((long)src * a.c.page.d + r0) * a.c.row;
        float* d = m + ((long)dst * a.c.page.d + r0) * a.c.row;
        if (!a.vec)
        {
            for (unsigned k = 0; k < rows; ++k)
                for (unsigned j = t; j < len; j += 256) d[(long)k * a.c.row + j] = s[(long)k * a.c.row + j];
            continue;
        }
        for (unsigned j = t; j < len / 4; j += 256)
        {
            f32x4 x[kReorderRows];
#pragma unroll
            for (unsigned k = 0; k < kReorderRows; ++k)
                x[k] = *reinterpret_cast<const f32x4*>(s + (long)min(k, rows - 1) * a.c.row + 4 * j);
#pragma unroll
            for (unsigned k = 0; k < kReorderRows; ++k)
                if (k < rows) *reinterpret_cast<f32x4*>(d + (long)k * a.c.row + 4 * j) = x[k];
        }
    }
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
    if (c->K == c->V || !k || !v || !pos || (q == nullptr) != (q_out == nullptr) || tokens > kMaxIndex || k_t < 0 || k_f < 0 ||
        v_t < 0 || v_f < 0 || q_t < 0 || q_f < 0 || o_t < 0 || o_f < 0 || (q && (q_heads == 0 || q_heads > kMaxIndex)) ||
        (cos == nullptr) != (sin == nullptr) || rope_dim % 2 != 0 || rope_dim > c->dim ||
        (cos ? rope_rows == 0 || rope_rows > kMaxIndex || rope_dim == 0 : rope_dim != 0))
        return -1;
    const size_t y = 2 * c->heads + (q ? q_heads : 0);
    if (y > 65535) return -1;
    AppendArgs a{};
    a.c = pages_of(*c);
    a.k = {k, k_t, k_f};
    a.v = {v, v_t, v_f};
    a.q = {q, q_t, q_f};
    a.out = q_out;
    a.o_t = o_t;
    a.o_f = o_f;
    a.seq = seq;
    a.pos = pos;
    a.cos = cos;
    a.sin = sin;
    a.tokens = static_cast<unsigned>(tokens);
    a.rope_rows = static_cast<unsigned>(rope_rows);
    a.head_slots = static_cast<unsigned>(y);
    a.half = static_cast<int>(rope_dim / 2);
    auto rows_of_4 = [](const float* p, long t, long f) { return !p || (f == 1 && t % 4 == 0 && aligned16(p)); };
    const size_t turned = rope_dim / 8, rest = c->dim - rope_dim, all_v = (c->dim + 7) / 8;
    a.pieces = static_cast<unsigned>(turned + (rest + 7) / 8 > all_v ? turned + (rest + 7) / 8 : all_v);
    const size_t threads = tokens * y * a.pieces;
    auto s = static_cast<hipStream_t>(stream);
    if (c->dim % 4 == 0 && rope_dim % 8 == 0 && c->row % 4 == 0 && aligned16(c->K) && aligned16(c->V) &&
        rows_of_4(k, k_t, k_f) && rows_of_4(v, v_t, v_f) && rows_of_4(q, q_t, q_f) && rows_of_4(q_out, o_t, o_f) &&
        (!cos || (aligned16(cos) && aligned16(sin))) && threads + 256 < 0x80000000u)
    {
        a.by_pieces = FastDiv(a.pieces);
        a.by_slots = FastDiv(a.head_slots);
        hipLaunchKernelGGL(k_kv_append_rows, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, s, a);
        return launch_status();
    }
    while (a.log2_lanes < 5 && ((size_t)1 << a.log2_lanes) < tokens) ++a.log2_lanes;
    static_assert(kAppendTokens == 1 << 5);
    const dim3 grid(static_cast<unsigned>((tokens + kAppendTokens - 1) / kAppendTokens), static_cast<unsigned>(y));
    hipLaunchKernelGGL(k_kv_append, grid, dim3(256), kAppendTokens * (c->dim + 1) * sizeof(float), s, a);
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
    if (!parent || !len || !table_out || !len_out || out_batch > kMaxIndex) return -1;
    // The workgroups of the tables read what the others' outputs would have overwritten, in any order.
    auto over_outputs = [&](const float* x, size_t n) {
        return x && (overlap(x, n, table_out, out_batch * c.width) || overlap(x, n, len_out, out_batch));
    };
    if (over_outputs(c.table, c.batch * c.width) || over_outputs(len, c.batch) || over_outputs(parent, out_batch) ||
        over_outputs(fresh, out_batch) || overlap(table_out, out_batch * c.width, len_out, out_batch))
        return -1;
    const size_t extent = (c.pages * c.page - 1) * c.row + c.heads * c.dim;   // of a cache: nothing behind its last row's heads
    for (size_t i = 0; i < n_layers; ++i)
        if (over_outputs(layers[i].K, extent) || over_outputs(layers[i].V, extent)) return -1;
    ReorderArgs a{};
    a.c = pages_of(c);
    a.parent = parent;
    a.len = len;
    a.fresh = fresh;
    a.table_out = table_out;
    a.len_out = len_out;
    a.out_batch = static_cast<unsigned>(out_batch);
    const bool copy = fresh && c.page > 1;
    for (size_t at = 0; at < n_layers; at += kReorderLayers)
    {
        const size_t n = n_layers - at < kReorderLayers ? n_layers - at : kReorderLayers;
        for (size_t i = 0; i < n; ++i)
        {
            a.mem[2 * i] = layers[at + i].K;
            a.mem[2 * i + 1] = layers[at + i].V;
        }
        a.n_mem = static_cast<unsigned>(2 * n);
        a.vec = c.heads * c.dim % 4 == 0 && c.row % 4 == 0;
        for (size_t i = 0; i < 2 * n; ++i) a.vec = a.vec && aligned16(a.mem[i]);
        const size_t tables = at == 0 ? (out_batch * c.width + 255) / 256 : 0;
        // Some 4 workgroups a CU: the lengths are on the device, and one that finds nothing to copy still waits for
        // the parent, its length and its page, one after another.
        const size_t pages = copy ? a.n_mem * out_batch : 0, most = (c.page - 1 + kReorderRows - 1) / kReorderRows;
        const size_t want = pages ? 4 * (size_t)device_cus() / pages : 0;
        a.splits = static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
        const size_t blocks = tables + a.splits * pages;
        if (blocks == 0) break;
        if (blocks > kGridMost) return -1;   // of the first launch, if of any: it has the tables and the most layers
        a.table_blocks = static_cast<unsigned>(tables);
        hipLaunchKernelGGL(k_kv_reorder, dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
        if (int rc = launch_status()) return rc;
    }
    return 0;
}
