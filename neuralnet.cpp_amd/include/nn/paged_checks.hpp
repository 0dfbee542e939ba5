// paged_checks.hpp — the shapes that every engine asks for in the paged-cache and
// beam-search calls (nn::ComputeEngine::kv_append, attn_paged, beam_select,
// kv_reorder).
#pragma once

#include "compute_engine.hpp"

namespace nn::paged
{

constexpr std::size_t kMaxIndex = std::size_t{1} << 24;   // integers that a float holds

// Head width of a cache, 0 where its shapes do not fit.
inline std::size_t dim_of(const KvPages& c)
{
    if (c.page == 0 || c.heads == 0 || c.K.rows() == 0 || c.K.rows() % c.page != 0 || c.K.cols() == 0 ||
        c.K.cols() % c.heads != 0 || c.V.rows() != c.K.rows() || c.V.cols() != c.K.cols() || c.table.size() == 0 ||
        c.K.rows() / c.page > kMaxIndex || c.K.rows() > 0x7fffffffu || c.page > kMaxIndex || c.table.rows() > kMaxIndex ||
        c.table.cols() > kMaxIndex || c.table.cols() * c.page > kMaxIndex)
        return 0;
    return c.K.cols() / c.heads;
}

// kv_append: query heads (0 without q) and half the turned width.
struct Append
{
    std::size_t dim, q_heads, half;
};
inline Result<Append> check_append(const KvPages& c, const Tensor& k, const Tensor& v, const Tensor* q, const Tensor& pos,
                                   const Tensor* seq, const Tensor* cos, const Tensor* sin)
{
    const std::size_t d = dim_of(c), n = k.cols();
    if (d == 0 || d > 256) return fail("kv_append: cache shapes do not fit (or heads wider than 256)");
    if (k.rows() != c.K.cols() || v.rows() != c.K.cols() || v.cols() != n) return fail("kv_append: k, v shape mismatch");
    if (pos.size() != n || (seq && seq->size() != n)) return fail("kv_append: one position (and sequence) a token required");
    if (q && (q->cols() != n || q->rows() == 0 || q->rows() % d != 0)) return fail("kv_append: q shape mismatch");
    if ((cos == nullptr) != (sin == nullptr)) return fail("kv_append: cos and sin go together");
    if (cos && (cos->rows() == 0 || cos->cols() == 0 || cos->rows() != sin->rows() || cos->cols() != sin->cols() ||
                2 * cos->cols() > d))
        return fail("kv_append: cos, sin shape mismatch");
    return Append{d, q ? q->rows() / d : 0, cos ? cos->cols() : 0};
}

// attn_paged: head width.
inline Result<std::size_t> check_attn(const KvPages& c, const Tensor& q, const Tensor& len, const Tensor* shared,
                                      std::size_t group, const Tensor* slopes)
{
    const std::size_t d = dim_of(c), batch = c.table.rows();
    if (d == 0 || d > 128) return fail("attn_paged: cache shapes do not fit (or heads wider than 128)");
    if (q.cols() != batch || q.rows() == 0 || q.rows() % d != 0 || (q.rows() / d) % c.heads != 0)
        return fail("attn_paged: q shape mismatch");
    if (len.size() != batch) return fail("attn_paged: one length a sequence required");
    if (group == 0 || batch % group != 0 || (shared && shared->size() != batch / group))
        return fail("attn_paged: groups do not fit the batch");
    if (slopes && slopes->size() != q.rows() / d) return fail("attn_paged: one slope a head required");
    return d;
}

// beam_select: beams of a group.
inline Result<std::size_t> check_select(const Tensor& logits, const Tensor& scores, const Tensor* done, std::size_t groups,
                                        std::size_t take, std::size_t eos)
{
    const std::size_t n = logits.cols(), vocab = logits.rows();
    if (groups == 0 || n == 0 || n % groups != 0 || n / groups > 1024 || n > kMaxIndex || vocab == 0 || vocab > kMaxIndex)
        return fail("beam_select: groups do not fit the logits");
    if (scores.size() != n || (done && done->size() != n)) return fail("beam_select: one score (and done) a beam required");
    if (n / groups * vocab >= (std::size_t{1} << 31) - (std::size_t{1} << 20))
        return fail("beam_select: beams * vocab too large");
    if (take == 0 || take > 256 || take > n / groups * vocab) return fail("beam_select: take out of range");
    if (done && eos >= vocab) return fail("beam_select: eos out of range");
    return n / groups;
}

inline Result<void> check_reorder(std::span<const KvPages> layers, const Tensor& parent, const Tensor& len,
                                  const Tensor* fresh)
{
    if (layers.empty()) return fail("kv_reorder: no layers");
    const KvPages& c = layers[0];
    for (const KvPages& x : layers)
        if (dim_of(x) == 0 || x.K.rows() != c.K.rows() || x.K.cols() != c.K.cols() || x.page != c.page ||
            x.heads != c.heads || x.table.rows() != c.table.rows() || x.table.cols() != c.table.cols())
            return fail("kv_reorder: cache shapes do not fit");
    if (len.size() != c.table.rows()) return fail("kv_reorder: one length a sequence required");
    if (parent.size() == 0 || parent.size() > kMaxIndex || (fresh && fresh->size() != parent.size()))
        return fail("kv_reorder: parent and fresh do not fit");
    return {};
}

} // namespace nn::paged
