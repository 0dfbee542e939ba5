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

// Sequences of up to 16 RT rows, bound by the cache's bytes: 32 single tokens behind 3000 positions, 12 heads of 64, take 100 us
// (460 MB, 4.6 TB/s), 48 of 4000 to 8000, 8 heads of 128, 400 (5.9); five tokens of one sequence behind 700, 7 and the join's
// 3 of latency.
template <int BITS, int KS, bool VEC, int RT> __global__ __launch_bounds__(256, VEC ? 2 : 1) void k_attn_chunk(ChunkArgs a)
{
    __shared__ WalkShared<KS> sh;
    Part part;
    if (!narrow_part(a, part, 4 * kTile)) return;
    // Ranges of an 8-bit cache are joined in the order of k_attn_chunk8.
    if (RT == 1 || part.n_rows <= kTile) walk<BITS, KS, VEC, 1, BITS == 8>(a, part, 1, sh);
    else walk<BITS, KS, VEC, RT, BITS == 8>(a, part, 1, sh);
}

// In place of the factor of a range of l = 0, whose O is anything. A factor that underflows to 0 is one: a value of its
// range that is not finite makes O one that is not, as within a range.
constexpr float kNoRange = -1.0f;
constexpr size_t kMostRanges = 256;

// The joins: narrow, wide: the ranges of the rows of either kernel. A row's ranges, 0 where it has nothing to join: written
// already, or no sequence's token; and the place of their results.
struct Joined
{
    unsigned ranges;
    bool log2;   // m is a score times log2(e)
    bool is_wide;
    size_t at;
};
__device__ __forceinline__ Joined joined(const ChunkArgs& a, unsigned n, unsigned h, unsigned narrow, unsigned wide)
{
    const int b = last_of(a.c.t.batch, [&](unsigned i) { return length_of(a.start[i], a.tokens) <= (int)n; });
    if (b < 0) return {};
    const Chunk c = chunk_of(a, b);
    if (n >= c.first + c.n) return {};
    const bool is_wide = c.n * (int)a.by_per.d > a.wide_from;
    const unsigned ranges = is_wide ? wide : narrow, kh = a.by_per.div(h);
    return {ranges == 1 ? 0 : ranges, is_wide || a.c.K, is_wide,
            is_wide ? (size_t)n * a.q_heads + h : result_of(a, results_of(a, b, kh, c.first), n - c.first, h - kh * a.by_per.d)};
}

// Row i of a join's grid: token and head, and, where the grid's order does not say it (wide), what is joined. Where rows of the
// wide kernel are whole already, or there are none (wide 1), the grid is of the others alone, kNarrowRows for each sequence and key head; i is past
// them where it has fewer.
__device__ __forceinline__ bool row_of_join(const ChunkArgs& a, unsigned i, unsigned narrow, unsigned wide, unsigned& n, unsigned& h,
                                            Joined& r)
{
    if (wide != 1)
    {
        n = a.by_q_heads.div(i);
        h = i - n * a.q_heads;
        if (n >= a.tokens) return false;
        if (wide) r = joined(a, n, h, narrow, wide);
        else r.at = i;
        return !wide || r.ranges > 0;
    }
    const unsigned piece = i / kNarrowRows, row = i - piece * kNarrowRows, b = a.by_heads.div(piece), kh = piece - b * a.c.t.heads;
    if (b >= a.c.t.batch) return false;
    const Chunk c = chunk_of(a, b);
    const int rows = c.n * (int)a.by_per.d;
    if (rows > a.wide_from || (int)row >= rows) return false;
    const unsigned t = a.by_per.div(row);
    n = c.first + t;
    h = kh * a.by_per.d + (row - t * a.by_per.d);
    r = {narrow, a.c.K != nullptr, false, i};
    return true;
}

// Up to kFewParts ranges: a wave a row, everything it needs on its way at once, the search for the token's sequence too. With
// rows of both kernels the search comes first: most rows may have nothing to join, or few ranges (seven prompts' chunks of
// 3900 tokens, 16 heads of 80, none of whose rows are cut: 67 us of reads that are not needed, 12 of searches alone, 3 by narrow rows).
constexpr unsigned kFewParts = 16;
__global__ __launch_bounds__(256) void k_attn_chunk_join_few(ChunkArgs a, unsigned narrow, unsigned wide)
{
    unsigned n, h;
    Joined r{};
    if (!row_of_join(a, (blockIdx.y * gridDim.x + blockIdx.x) * 4 + threadIdx.x / 64, narrow, wide, n, h, r)) return;
    const unsigned slots = wide ? r.ranges : narrow, last = slots - 1;
    const int lane = threadIdx.x & 63, dim = a.c.t.dim;
    const float2 own = reinterpret_cast<const float2*>(r.is_wide ? a.wide_ml : a.part_ml)[r.at * slots + min((unsigned)lane, last)];
    const float* po = (r.is_wide ? a.wide_o : a.part_o) + r.at * slots * dim;
    float x[kFewParts][2];
#pragma unroll
    for (unsigned i = 0; i < kFewParts; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y) x[i][y] = po[(size_t)min(i, last) * dim + min(lane + 64 * y, dim - 1)];
    if (!wide) r = joined(a, n, h, narrow, wide);
    if (r.ranges == 0) return;
    const bool any = lane < (int)r.ranges && own.y != 0.0f;
    const float m = wave_max(any ? own.x : kLowest);
    const float w = any ? __builtin_amdgcn_exp2f((own.x - m) * (r.log2 ? 1.0f : kLog2e)) : kNoRange;
    const float l = wave_sum(any ? own.y * w : 0.0f);
    float o[2] = {0.0f, 0.0f};
#pragma unroll
    for (unsigned i = 0; i < kFewParts; ++i)
    {
        const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
#pragma unroll
        for (int y = 0; y < 2; ++y) o[y] += f == kNoRange ? 0.0f : x[i][y] * f;
    }
#pragma unroll
    for (int y = 0; y < 2; ++y)
    {
        const int d = lane + 64 * y;
        if (d < dim) a.O[(long)n * a.o_t + ((long)h * dim + d) * a.o_f] = l == 0.0f ? 0.0f : o[y] / l;
    }
    const size_t to = (size_t)n * a.q_heads + h;
    if (lane == 0 && a.m) a.m[to] = r.log2 && m != kLowest ? m * kLn2 : m;
    if (lane == 0 && a.l) a.l[to] = l;
}

// More: a workgroup a row. The ranges' factors go to LDS, then 2 or 4 groups of threads sum every 2nd or 4th range.
__global__ __launch_bounds__(256) void k_attn_chunk_join(ChunkArgs a, unsigned narrow, unsigned wide)
{
    static_assert(kMostRanges <= 256);
    __shared__ float w_s[256], red[2][4], o_s[256];
    unsigned n, h;
    Joined r{};
    if (!row_of_join(a, blockIdx.y * gridDim.x + blockIdx.x, narrow, wide, n, h, r)) return;
    if (!wide) r = joined(a, n, h, narrow, wide);
    if (r.ranges == 0) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, dim = a.c.t.dim;
    const int cols = dim <= 64 ? 64 : 128, groups = 256 / cols, d = t % cols, g = t / cols;
    const float2 own = reinterpret_cast<const float2*>(r.is_wide ? a.wide_ml : a.part_ml)[r.at * r.ranges + min((unsigned)t, r.ranges - 1)];
    const float* po = (r.is_wide ? a.wide_o : a.part_o) + r.at * r.ranges * dim + (d < dim ? d : 0);
    const bool any = t < (int)r.ranges && own.y != 0.0f;
    float m = wave_max(any ? own.x : kLowest);
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmax_std(fmax_std(red[0][0], red[0][1]), fmax_std(red[0][2], red[0][3]));
    const float w = any ? __builtin_amdgcn_exp2f((own.x - m) * (r.log2 ? 1.0f : kLog2e)) : kNoRange;
    float l = wave_sum(any ? own.y * w : 0.0f), o = 0.0f;
    w_s[t] = w;
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
#pragma unroll 8
    for (int i = g; i < (int)r.ranges; i += groups)
    {
        const float x = po[(size_t)i * dim], f = w_s[i];
        o += f == kNoRange ? 0.0f : x * f;
    }
    o_s[t] = o;
    __syncthreads();
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    if (t < dim)
    {
        o = 0.0f;
        for (int i = 0; i < groups; ++i) o += o_s[i * cols + t];
        a.O[(long)n * a.o_t + ((long)h * dim + t) * a.o_f] = l == 0.0f ? 0.0f : o / l;
    }
    const size_t to = (size_t)n * a.q_heads + h;
    if (t == 0 && a.m) a.m[to] = r.log2 && m != kLowest ? m * kLn2 : m;
    if (t == 0 && a.l) a.l[to] = l;
}

// A call's sizes, whichever cache it is over.
struct ChunkCall
{
    Pages8 c;
    int bits;
    bool vec;          // rows can be read in pieces of 4 values
    int bytes;         // 8 bits: and in pieces of so many bytes, 16, 8 or 4, or 1
    size_t q_heads, tokens, most;
};

struct ChunkPlan
{
    int wide_from;
    unsigned narrow, wide;   // ranges of the two kernels' rows, 0: it is not launched
    size_t blocks, wide_row_blocks, wide_blocks;
    bool wide_by_seqs;
    size_t image_slots, image_tiles, image_pieces;   // of the parts; pieces that are formed at a time
    unsigned most_ranges() const { return std::max(narrow, wide); }
};

// Parts of keys and values that are formed at a time, or those of one piece: past this a call takes several launches. They are
// as large as the float32 cache of the sequences with many rows, which may be any of the batch's.
constexpr size_t kImageBytes = (size_t)2 << 30;

// How a call is cut, from its sizes alone: the lengths are on the device.
ChunkPlan chunk_plan(const ChunkCall& c)
{
    ChunkPlan p{};
    const size_t per = c.q_heads / c.c.t.heads, batch = c.c.t.batch, heads = c.c.t.heads;
    const size_t positions = (size_t)c.c.t.width * c.c.t.page.d, cus = device_cus();
    // No sequence has more rows: those of up to 16 have a kernel that holds fewer registers.
    p.wide_from = static_cast<int>(std::min<size_t>(kNarrowRows, (c.most * per + kTile - 1) / kTile * kTile));
    // Workgroups a CU. Where the key heads alone fill the CUs, float32 caches stream best with 8 (48 sequences of 4000 to 8000
    // positions, 8 heads of 128: 466 us with 2, 440 with 4, 400 with 8), bytes with 4 (143 us with 2 to 8; 5 rows a head 192
    // with 2, 188 with 4, 213 with 8); where they do not, ranges are more results to join (one sequence of 60000: 95 to 103
    // us with 2 and 3, 107 with 8; in bytes 34 and 36, 50 with 8; 4 of 3000, 12 heads of 64: 22 and 20, 25 with 8).
    const size_t pieces = batch * heads, per_cu = pieces < cus ? 3 : c.bits == 32 ? 8 : 4;
    const size_t want = (per_cu * cus + pieces - 1) / pieces, most_ranges = (positions + 63) / 64;
    p.narrow = static_cast<unsigned>(std::min<size_t>(std::min(want, most_ranges), kMostRanges));
    p.blocks = (batch * p.narrow + 7) / 8 * 8 * heads;
    if (c.most * per > kNarrowRows)
    {
        // Numbers of blocks of rows: fewer by the sequences' numbers where these are few, else by rows alone.
        const size_t by_seqs = c.tokens * per / kWideRows + batch, by_rows = c.tokens * per / (kNarrowRows + 1) + 1;
        p.wide_by_seqs = by_seqs <= by_rows || batch == 1;
        p.wide_row_blocks = p.wide_by_seqs ? by_seqs : by_rows;
        // Ranges for two workgroups a CU, of 128 positions at least (200 tokens behind 300, 12 heads: 32 us with 256, 27 with 128,
        // 25 with 64; chunks of up to 60 of four sequences over bytes 32, 28, 29; 40 tokens behind 6000 87, 83, 83; 16 sequences of
        // 12 behind 2000 213, 224, 226).
        const size_t others = heads * ((c.tokens * per + kWideRows - 1) / kWideRows), most_wide = (positions + 127) / 128;
        p.wide = static_cast<unsigned>(std::min<size_t>(std::min(std::max<size_t>(2 * cus / others, 1), most_wide), kMostRanges));
        p.wide_blocks = (p.wide_row_blocks * heads * p.wide + 7) / 8 * 8;
        if (batch == 1) p.narrow = 0, p.wide_from = 0;   // one launch, however few tokens the sequence has
        p.image_slots = std::min(batch, c.tokens * per / (kNarrowRows + 1) + 1);
        p.image_tiles = (positions + 31) / 32;
        p.image_pieces = std::min(p.image_slots * heads, std::max<size_t>(kImageBytes / (p.image_tiles * chunk_image_bytes(c.bits, c.c.t.dim)), 1));
    }
    return p;
}

// The workspace: the ranges' results of the rows of either kernel (m and l, then O), and the parts; floats, each in whole 16
// bytes. Beside prompts, and where most tokens are padding, the narrow kernel's are those of kNarrowRows for each sequence and
// key head: its ranges are chosen for that many, and of every token they would be gigabytes that nothing writes (two prompts
// of 8192 tokens, 32 heads on 8 of 128: 12 GiB, and 12 MiB so).
struct ChunkSpace
{
    size_t narrow_o, wide_ml, wide_o, images;
    size_t bytes;
    bool few_rows;
};
ChunkSpace chunk_space(const ChunkCall& c, const ChunkPlan& p)
{
    const size_t all = c.tokens * c.q_heads, few = (size_t)c.c.t.batch * c.c.t.heads * kNarrowRows;
    const bool few_rows = p.wide || all > few;
    const size_t narrow = p.narrow > 1 ? (few_rows ? few : all) * p.narrow : 0, wide = p.wide > 1 ? all * p.wide : 0, dim = c.c.t.dim;
    auto whole = [](size_t n) { return (n + 3) / 4 * 4; };
    ChunkSpace s{};
    s.few_rows = few_rows;
    s.narrow_o = whole(2 * narrow);
    s.wide_ml = s.narrow_o + whole(narrow * dim);
    s.wide_o = s.wide_ml + whole(2 * wide);
    s.images = s.wide_o + whole(wide * dim);
    s.bytes = s.images * sizeof(float) + p.image_pieces * p.image_tiles * chunk_image_bytes(c.bits, c.c.t.dim);
    return s;
}

bool chunk_ok(const ChunkCall& c, size_t heads)
{
    return c.q_heads > 0 && c.q_heads % heads == 0 && c.q_heads <= kMaxIndex && c.tokens > 0 && c.tokens <= kMaxIndex && c.most > 0 &&
           c.most <= c.tokens && c.tokens * c.q_heads < (size_t)0x80000000u;
}
bool chunk_call(const nnhip_kv_pages* c, size_t q_heads, size_t tokens, size_t most, ChunkCall& out)
{
    if (!pages_ok(c, kChunkMaxDim)) return false;
    out = {Pages8{pages_of(*c), nullptr, nullptr, nullptr, nullptr}, 32, c->dim % 4 == 0 && c->row % 4 == 0 && aligned16(c->K) && aligned16(c->V), 0,
           q_heads, tokens, most};
    return chunk_ok(out, c->heads);
}
bool chunk_call(const nnhip_kv8_pages* c, size_t q_heads, size_t tokens, size_t most, ChunkCall& out)
{
    if (!pages8_ok(c, kChunkMaxDim)) return false;
    const uintptr_t at = reinterpret_cast<uintptr_t>(c->K) | reinterpret_cast<uintptr_t>(c->V) | c->dim | c->row;
    const int bytes = at % 16 == 0 ? 16 : at % 8 == 0 ? 8 : at % 4 == 0 ? 4 : 1;
    out = {pages8_of(*c), 8, bytes >= 4, bytes,
           q_heads, tokens, most};
    return chunk_ok(out, c->heads);
}

template <int BITS, bool VEC, int RT> void chunk_launch(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s)
{
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.blocks)), dim3(256), 0, s, a); };
    switch ((a.c.t.dim + 31) / 32)
    {
    case 1: go(k_attn_chunk<BITS, 2, VEC, RT>); break;
    case 2: go(k_attn_chunk<BITS, 4, VEC, RT>); break;
    case 3: go(k_attn_chunk<BITS, 6, VEC, RT>); break;
    default: go(k_attn_chunk<BITS, 8, VEC, RT>); break;
    }
}
template <int BITS, bool VEC> void chunk_launch(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s)
{
    if (a.wide_from <= kTile) chunk_launch<BITS, VEC, 1>(a, p, s);
    else chunk_launch<BITS, VEC, 2>(a, p, s);
}

template <class C> size_t chunk_bytes(const C* c, size_t q_heads, size_t tokens, size_t most)
{
    ChunkCall call;
    return chunk_call(c, q_heads, tokens, most, call) ? chunk_space(call, chunk_plan(call)).bytes : 0;
}

template <class C>
int attn_chunk(const C* c, const float* q, long q_t, long q_f, size_t q_heads, size_t tokens, const float* start, size_t most,
               const float* len, const float* slopes, float alpha, float* O, long o_t, long o_f, float* m, float* l, void* workspace,
               size_t workspace_bytes, void* stream)
{
    ChunkCall call;
    if (!chunk_call(c, q_heads, tokens, most, call) || !q || !start || !len || !O || q_t < 0 || q_f < 0 || o_t < 0 || o_f < 0) return -1;
    const ChunkPlan p = chunk_plan(call);
    const ChunkSpace space = chunk_space(call, p);
    if (space.bytes > 0 && (!workspace || workspace_bytes < space.bytes || !aligned16(workspace))) return -1;
    if (p.blocks > kGridMost || p.wide_blocks > kGridMost) return -1;
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
    a.part_o = ws + space.narrow_o;
    a.wide_ml = ws + space.wide_ml;
    a.wide_o = ws + space.wide_o;
    a.few_rows = space.few_rows;
    a.result_step = static_cast<unsigned>(space.few_rows ? q_heads / c->heads : q_heads);
    a.q_heads = static_cast<unsigned>(q_heads);
    a.tokens = static_cast<unsigned>(tokens);
    a.most = static_cast<unsigned>(most);
    a.ranges = p.narrow;
    a.wide_from = p.wide_from;
    a.by_per = FastDiv(static_cast<unsigned>(q_heads / c->heads));
    a.by_heads = FastDiv(call.c.t.heads);
    a.by_q_heads = FastDiv(a.q_heads);
    a.by_ranges = FastDiv(std::max(p.narrow, 1u));
    a.q_rows = q_f == 1 && q_t % 4 == 0 && aligned16(q) && c->dim % 4 == 0;
    a.page4 = c->page % 4 == 0;
    a.vec = call.vec;
    a.alpha = alpha;
    auto s = static_cast<hipStream_t>(stream);
    if (p.narrow)
    {
        if (call.bits == 32) call.vec ? chunk_launch<32, true>(a, p, s) : chunk_launch<32, false>(a, p, s);
        else if (call.bytes >= 4) chunk8(a, call.bytes, static_cast<unsigned>(p.blocks), s);
        else chunk_launch<8, false>(a, p, s);
        if (int rc = launch_status()) return rc;
    }
    if (p.wide)
    {
        ChunkArgs w = a;
        w.ranges = p.wide;
        w.part_ml = a.wide_ml;
        w.part_o = a.wide_o;
        w.few_rows = 0;
        w.result_step = a.q_heads;
        w.by_ranges = FastDiv(p.wide);
        w.by_row_blocks = FastDiv(static_cast<unsigned>(p.wide_row_blocks));
        w.by_block_rows = FastDiv(p.wide_by_seqs ? kWideRows : kNarrowRows + 1);
        w.block_seqs = p.wide_by_seqs;
        w.images = reinterpret_cast<char*>(ws + space.images);
        w.tiles = static_cast<unsigned>(p.image_tiles);
        w.slots_by_batch = p.image_slots == call.c.t.batch;
        // Workgroups: of several slots most may have nothing to do.
        const size_t all = p.image_slots * call.c.t.heads, heads_of_one = call.c.t.heads;
        for (size_t at = 0; at < all; at += p.image_pieces)
        {
            const size_t pieces = std::min(p.image_pieces, all - at), each = std::min(p.image_tiles, ((all == heads_of_one ? 8 : 32) * device_cus() + pieces - 1) / pieces);
            w.first_piece = static_cast<unsigned>(at);
            w.pieces = static_cast<unsigned>(pieces);
            chunk_parts(w, call.bits, w.pieces, static_cast<unsigned>(each), s);
            if (int rc = launch_status()) return rc;
            chunk_wide(w, call.bits, static_cast<unsigned>(p.wide_blocks), s);
            if (int rc = launch_status()) return rc;
        }
    }
    if (p.most_ranges() == 1) return 0;
    const bool few = p.most_ranges() <= kFewParts;
    const unsigned wide = p.wide == 0 && space.few_rows ? 1 : p.wide;   // no wide rows, or whole ones: the others' grid
    const size_t rows = wide == 1 ? call.c.t.batch * (size_t)call.c.t.heads * kNarrowRows : tokens * q_heads;
    const size_t blocks = few ? (rows + 3) / 4 : rows, x = std::min(blocks, (size_t)1 << 20);
    const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>((blocks + x - 1) / x));
    hipLaunchKernelGGL(few ? k_attn_chunk_join_few : k_attn_chunk_join, grid, dim3(256), 0, s, a, p.narrow, wide);
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
