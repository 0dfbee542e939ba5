// k_attn_chunk.hip — attention of each sequence's new tokens against its paged
// keys and values, in float32 or as bytes with a scale a row and head:
//
//   s_j = alpha q . k_j - slope (p - j),  j <= p, the token's position,
//   m = max_j s_j,  l = sum_j exp(s_j - m),  O = sum_j exp(s_j - m) v_j / l.
//
// A sequence's rows are its (token, query head) pairs that read one key head. A
// workgroup takes a block of them and one range of the positions that its last
// token sees; where there are several ranges a second kernel joins them in
// order.
#include "attn_chunk.hpp"

#include <algorithm>

namespace nnhip
{
namespace
{

// Sequences of up to kNarrowRows rows.
template <int BITS, int KS, bool VEC> __global__ __launch_bounds__(256, VEC ? 2 : 1) void k_attn_chunk(ChunkArgs a)
{
    __shared__ WalkShared<KS> sh;
    Part part;
    if (!narrow_part(a, part, 4 * kTile)) return;
    // Ranges of an 8-bit cache are joined in the order of k_attn_chunk8.
    if (part.n_rows <= kTile) walk<BITS, KS, VEC, 1, BITS == 8>(a, part, 1, sh);
    else walk<BITS, KS, VEC, 2, BITS == 8>(a, part, 1, sh);
}

// In place of the factor of a range of l = 0, whose O is anything. A factor that underflows to 0 is one: a value of its
// range that is not finite makes O one that is not, as within a range.
constexpr float kNoRange = -1.0f;

// Joins the ranges of a row in order: a wave a row. narrow, wide: the ranges of the rows of either kernel.
__global__ __launch_bounds__(256) void k_attn_chunk_join(ChunkArgs a, unsigned narrow, unsigned wide)
{
    const unsigned at = blockIdx.x * 4 + threadIdx.x / 64;
    const unsigned n = at / a.q_heads, h = at - n * a.q_heads;
    if (n >= a.tokens) return;
    const int lane = threadIdx.x & 63, dim = a.c.t.dim;
    const int b = last_of(a.c.t.batch, [&](unsigned i) { return length_of(a.start[i], a.tokens) <= (int)n; });
    if (b < 0) return;
    const Chunk c = chunk_of(a, b);
    if (n >= c.first + c.n) return;   // no sequence's
    const bool is_wide = c.n * (int)a.by_per.d > a.wide_from, log2 = is_wide || a.c.K;   // m is a score times log2(e)
    const unsigned ranges = is_wide ? wide : narrow;
    const float to_log2 = log2 ? 1.0f : kLog2e;
    if (ranges == 1) return;   // written already
    const float* ml = a.part_ml + 2 * (size_t)at * a.slots;
    const float* po = a.part_o + (size_t)at * a.slots * dim;
    float m = kLowest, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (unsigned i = lane; i < ranges; i += 64)
        if (ml[2 * i + 1] != 0.0f) m = fmax_std(m, ml[2 * i]);
    m = wave_max(m);
    for (unsigned c0 = 0; c0 < ranges; c0 += 64)
    {
        float w = kNoRange;
        if (c0 + lane < ranges && ml[2 * (c0 + lane) + 1] != 0.0f)
        {
            w = __builtin_amdgcn_exp2f((ml[2 * (c0 + lane)] - m) * to_log2);
            l += ml[2 * (c0 + lane) + 1] * w;
        }
        const int nc = min(ranges - c0, 64u);
        for (int i = 0; i < nc; ++i)
        {
            const float f = __shfl(w, i, 64);
#pragma unroll
            for (int y = 0; y < 2; ++y)
            {
                const float x = po[(size_t)(c0 + i) * dim + min(lane + 64 * y, dim - 1)];
                o[y] += f == kNoRange ? 0.0f : x * f;
            }
        }
    }
    l = wave_sum(l);
#pragma unroll
    for (int y = 0; y < 2; ++y)
    {
        const int d = lane + 64 * y;
        if (d < dim) a.O[(long)n * a.o_t + ((long)h * dim + d) * a.o_f] = l == 0.0f ? 0.0f : o[y] / l;
    }
    if (lane == 0 && a.m) a.m[at] = log2 && m != kLowest ? m * kLn2 : m;
    if (lane == 0 && a.l) a.l[at] = l;
}

// A call's sizes, whichever cache it is over.
struct ChunkCall
{
    Pages8 c;
    int bits;
    bool vec;          // rows can be read in pieces of 4 values
    bool wide_bytes;   // and 16 bytes
    size_t q_heads, tokens, most;
};

struct ChunkPlan
{
    int wide_from;
    unsigned narrow, wide;   // ranges of the two kernels' rows, 0: it is not launched
    size_t blocks, wide_row_blocks, wide_blocks;
    unsigned slots() const { return std::max(narrow, wide); }
};

constexpr size_t kNarrowRows = 32;   // of a sequence and key head that the walk takes

// How a call is cut, from its sizes alone: the lengths are on the device.
ChunkPlan chunk_plan(const ChunkCall& c)
{
    ChunkPlan p{};
    const size_t per = c.q_heads / c.c.t.heads, batch = c.c.t.batch, heads = c.c.t.heads;
    const size_t positions = (size_t)c.c.t.width * c.c.t.page.d, cus = device_cus();
    p.wide_from = kNarrowRows;
    const size_t want = (4 * cus + batch * heads - 1) / (batch * heads), most_ranges = (positions + 63) / 64;
    p.narrow = static_cast<unsigned>(std::min<size_t>(std::min(want, most_ranges), 256));
    p.blocks = batch * heads * p.narrow;
    if (c.most * per > kNarrowRows)
    {
        p.wide_row_blocks = c.tokens * per / kWideRows + batch;
        const size_t others = heads * std::max<size_t>(c.tokens * per / kWideRows, 1), most_wide = (positions + 255) / 256;
        p.wide = static_cast<unsigned>(std::min<size_t>(std::min(std::max<size_t>(2 * cus / others, 1), most_wide), 256));
        p.wide_blocks = (p.wide_row_blocks * heads * p.wide + 7) / 8 * 8;
        if (batch == 1) p.narrow = 0, p.wide_from = 0;   // one launch, however few tokens the sequence has
    }
    return p;
}

// m and l of every row and range, in whole 16 bytes.
size_t ml_floats(const ChunkCall& c, const ChunkPlan& p) { return (2 * c.tokens * c.q_heads * p.slots() + 3) / 4 * 4; }
size_t chunk_workspace(const ChunkCall& c, const ChunkPlan& p)
{
    return p.slots() == 1 ? 0 : (ml_floats(c, p) + c.tokens * c.q_heads * p.slots() * c.c.t.dim) * sizeof(float);
}

bool chunk_ok(const ChunkCall& c, size_t heads)
{
    return c.q_heads > 0 && c.q_heads % heads == 0 && c.q_heads <= kMaxIndex && c.tokens > 0 && c.tokens <= kMaxIndex && c.most > 0 &&
           c.most <= c.tokens && c.tokens * c.q_heads < (size_t)0x80000000u;
}
bool chunk_call(const nnhip_kv_pages* c, size_t q_heads, size_t tokens, size_t most, ChunkCall& out)
{
    if (!pages_ok(c, kChunkMaxDim)) return false;
    out = {Pages8{pages_of(*c), nullptr, nullptr, nullptr, nullptr}, 32, c->dim % 4 == 0 && c->row % 4 == 0 && aligned16(c->K) && aligned16(c->V), false,
           q_heads, tokens, most};
    return chunk_ok(out, c->heads);
}
bool chunk_call(const nnhip_kv8_pages* c, size_t q_heads, size_t tokens, size_t most, ChunkCall& out)
{
    if (!pages8_ok(c, kChunkMaxDim)) return false;
    const uintptr_t at = reinterpret_cast<uintptr_t>(c->K) | reinterpret_cast<uintptr_t>(c->V);
    out = {pages8_of(*c), 8, c->dim % 4 == 0 && c->row % 4 == 0 && (at & 3) == 0, c->dim % 16 == 0 && c->row % 16 == 0 && (at & 15) == 0,
           q_heads, tokens, most};
    return chunk_ok(out, c->heads);
}

template <int BITS, bool VEC> void chunk_launch(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s)
{
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.blocks)), dim3(256), 0, s, a); };
    switch ((a.c.t.dim + 31) / 32)
    {
    case 1: go(k_attn_chunk<BITS, 2, VEC>); break;
    case 2: go(k_attn_chunk<BITS, 4, VEC>); break;
    case 3: go(k_attn_chunk<BITS, 6, VEC>); break;
    default: go(k_attn_chunk<BITS, 8, VEC>); break;
    }
}

template <class C> size_t chunk_bytes(const C* c, size_t q_heads, size_t tokens, size_t most)
{
    ChunkCall call;
    return chunk_call(c, q_heads, tokens, most, call) ? chunk_workspace(call, chunk_plan(call)) : 0;
}

template <class C>
int attn_chunk(const C* c, const float* q, long q_t, long q_f, size_t q_heads, size_t tokens, const float* start, size_t most,
               const float* len, const float* slopes, float alpha, float* O, long o_t, long o_f, float* m, float* l, void* workspace,
               size_t workspace_bytes, void* stream)
{
    ChunkCall call;
    if (!chunk_call(c, q_heads, tokens, most, call) || !q || !start || !len || !O || q_t < 0 || q_f < 0 || o_t < 0 || o_f < 0) return -1;
    const ChunkPlan p = chunk_plan(call);
    const size_t need = chunk_workspace(call, p);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return -1;
    if (p.blocks > kGridMost || p.wide_blocks > kGridMost || tokens * q_heads / 4 + 1 > kGridMost) return -1;
    auto* ws = static_cast<float*>(workspace);
    ChunkArgs a{};
    a.c = call.c;
    a.q = q;
    a.q_t = q_t;
    a.q_f = q_f;
    a.start = start;
    a.len = len;
    a.slopes = slopes;
    a.O = O;
    a.o_t = o_t;
    a.o_f = o_f;
    a.m = m;
    a.l = l;
    a.part_ml = ws;
    if (p.slots() > 1) a.part_o = ws + ml_floats(call, p);
    a.q_heads = static_cast<unsigned>(q_heads);
    a.tokens = static_cast<unsigned>(tokens);
    a.most = static_cast<unsigned>(most);
    a.ranges = p.narrow;
    a.slots = p.slots();
    a.wide_from = p.wide_from;
    a.by_per = FastDiv(static_cast<unsigned>(q_heads / c->heads));
    a.by_heads = FastDiv(call.c.t.heads);
    a.by_ranges = FastDiv(std::max(p.narrow, 1u));
    a.q_rows = q_f == 1 && q_t % 4 == 0 && aligned16(q) && c->dim % 4 == 0;
    a.page4 = c->page % 4 == 0;
    a.vec = call.vec;
    a.alpha = alpha;
    auto s = static_cast<hipStream_t>(stream);
    if (p.narrow)
    {
        if (call.bits == 32) call.vec ? chunk_launch<32, true>(a, p, s) : chunk_launch<32, false>(a, p, s);
        else if (call.wide_bytes) chunk8(a, static_cast<unsigned>(p.blocks), s);
        else chunk_launch<8, false>(a, p, s);
        if (int rc = launch_status()) return rc;
    }
    if (p.wide)
    {
        ChunkArgs w = a;
        w.ranges = p.wide;
        w.by_ranges = FastDiv(p.wide);
        w.by_row_blocks = FastDiv(static_cast<unsigned>(p.wide_row_blocks));
        chunk_wide(w, call.bits, static_cast<unsigned>(p.wide_blocks), s);
        if (int rc = launch_status()) return rc;
    }
    if (p.slots() == 1) return 0;
    hipLaunchKernelGGL(k_attn_chunk_join, dim3(static_cast<unsigned>((tokens * q_heads + 3) / 4)), dim3(256), 0, s, a, p.narrow, p.wide);
    return launch_status();
}

} // namespace
} // namespace nnhip

using namespace nnhip;

extern "C" size_t nnhip_attn_chunk_workspace_bytes(const nnhip_kv_pages* c, size_t q_heads, size_t tokens, size_t most)
{
    return chunk_bytes(c, q_heads, tokens, most);
}
extern "C" size_t nnhip_attn_chunk8_workspace_bytes(const nnhip_kv8_pages* c, size_t q_heads, size_t tokens, size_t most)
{
    return chunk_bytes(c, q_heads, tokens, most);
}
extern "C" int nnhip_attn_chunk(const nnhip_kv_pages* c, const float* q, long q_t, long q_f, size_t q_heads, size_t tokens,
                                const float* start, size_t most, const float* len, const float* slopes, float alpha, float* O, long o_t,
                                long o_f, float* m, float* l, void* workspace, size_t workspace_bytes, void* stream)
{
    return attn_chunk(c, q, q_t, q_f, q_heads, tokens, start, most, len, slopes, alpha, O, o_t, o_f, m, l, workspace, workspace_bytes, stream);
}
extern "C" int nnhip_attn_chunk8(const nnhip_kv8_pages* c, const float* q, long q_t, long q_f, size_t q_heads, size_t tokens,
                                 const float* start, size_t most, const float* len, const float* slopes, float alpha, float* O, long o_t,
                                 long o_f, float* m, float* l, void* workspace, size_t workspace_bytes, void* stream)
{
    return attn_chunk(c, q, q_t, q_f, q_heads, tokens, start, most, len, slopes, alpha, O, o_t, o_f, m, l, workspace, workspace_bytes, stream);
}
