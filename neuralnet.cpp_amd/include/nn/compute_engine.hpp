// compute_engine.hpp — the op-level engine interface (the drop-in boundary).
//
// Same virtual surface, argument meaning, defaults and op codes as the
// reference's nn::ComputeEngine (include/neuralnet.cpp/compute_engine.hpp:87-410).
// Default arguments live only on this base declaration, so callers go
// through ComputeEngine& exactly as the reference's layers do. Layers hold
// the algorithms; engines implement only these primitives.
//
// Shape conventions shared by every engine (reference :130-200):
//   * all tensors are row-major fp32; index tensors hold integers as floats;
//   * batched ops split A/B into `batch` consecutive row blocks;
//     A_b is (M,K), or (K,M) stored when transA; B_b is (K,N), or (N,K) when transB;
//   * masks are dense (M,N) float tensors shared by all batches:
//     -inf excludes a position, a finite value is added to the score.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <span>

#include "core_errors.hpp"
#include "expr_spec.hpp"
#include "tensor.hpp"

namespace nn
{

// Op codes keep the reference's numeric values (compute_engine.hpp:43-82);
// they are also the op ids of the kernel C-ABI.
enum class UnaryOp : std::uint32_t { Neg = 0, Exp = 1, Log = 2, Sqrt = 3, Rsqrt = 4, Abs = 5, Tanh = 6 };
enum class BinaryOp : std::uint32_t { Add = 0, Sub = 1, Mul = 2, Div = 3, Max = 4, Min = 5 };
enum class CompareOp : std::uint32_t { Lt = 0, Le = 1, Gt = 2, Ge = 3, Eq = 4, Ne = 5 };
enum class ReduceOp : std::uint32_t { Sum = 0, Max = 1, Min = 2 };

// Keys and values of a batch of sequences in pages (nnhip_kv_pages, nnhip_kernels.h): K and V (pages * page,
// heads * dim), table (batch, width) of page numbers. No reference counterpart.
struct KvPages
{
    Tensor K, V, table;
    std::size_t page = 1, heads = 1;
};

// The same with a byte a value (nnhip_kv8_pages): K and V (pages * page, at least heads * dim / 4 floats, each of four
// bytes), a scale a row and head (pages * page, heads).
struct KvPages8
{
    Tensor K, V, K_scale, V_scale, table;
    std::size_t page = 1, heads = 1, dim = 1;
};

class ComputeEngine
{
public:
    virtual ~ComputeEngine() = default;

    [[nodiscard]] virtual Device device() const noexcept = 0;

    // Batch / expression regions (reference :93-118).
    [[nodiscard]] virtual Result<void> begin_batch() = 0;
    [[nodiscard]] virtual Result<void> end_batch() = 0;
    [[nodiscard]] virtual Result<void> begin_expr() = 0;
    [[nodiscard]] virtual Result<void> end_expr() = 0;
    [[nodiscard]] virtual Result<void> flush_batch() { return {}; }

    // Factories and transfers (reference :121-131).
    [[nodiscard]] virtual Tensor create_tensor(std::size_t rows, std::size_t cols) = 0;
    [[nodiscard]] virtual Result<Tensor> from_matrix(const Matrix& m) = 0;
    [[nodiscard]] virtual Result<Matrix> to_matrix(const Tensor& t) = 0;
    // to_matrix into the caller's t.size() floats (no reference counterpart: its hosts take the Matrix).
    [[nodiscard]] virtual Result<void> read_into(const Tensor& t, Scalar* out)
    {
        NN_TRY(m, to_matrix(t));
        std::copy(m.data(), m.data() + m.size(), out);
        return {};
    }
    [[nodiscard]] virtual Result<void> copy_from(Tensor& dst, const Matrix& src) = 0;
    [[nodiscard]] virtual Result<Tensor> clone(const Tensor& src) = 0;

    // Row slices (reference :136-143).
    [[nodiscard]] virtual Result<Tensor> slice_rows(const Tensor& src, std::size_t start_row, std::size_t count) = 0;
    [[nodiscard]] virtual Result<void> insert_rows(Tensor& dst, std::size_t dst_start_row, const Tensor& src) = 0;

    // Row gather / scatter-add by float-encoded indices (reference :151-161).
    [[nodiscard]] virtual Result<Tensor> gather_rows(const Tensor& table, const Tensor& indices) = 0;
    [[nodiscard]] virtual Result<void> scatter_add_rows(Tensor& dst, const Tensor& indices, const Tensor& grad) = 0;

    // (M, B*N) <-> (B*M, N) (reference :170-172) and 2-D transpose (:175).
    [[nodiscard]] virtual Result<Tensor> rearrange_3d(const Tensor& x, std::size_t M, std::size_t B, std::size_t N,
                                                      bool inverse = false) = 0;
    [[nodiscard]] virtual Result<Tensor> transpose(const Tensor& A) = 0;

    // GEMMs (reference :182-199).
    [[nodiscard]] virtual Result<Tensor> matmul(const Tensor& A, const Tensor& B, bool transA = false,
                                                bool transB = false) = 0;
    [[nodiscard]] virtual Result<Tensor> batched_matmul(const Tensor& A, const Tensor& B, std::size_t batch,
                                                        bool transA = false, bool transB = false,
                                                        Scalar alpha = Scalar{1}) = 0;

    // Fused attention primitives (reference :217-276).
    [[nodiscard]] virtual Result<Tensor> batched_matmul_reduce(const Tensor& A, const Tensor& B, std::size_t batch,
                                                               ReduceOp op, bool transA, bool transB, Scalar alpha,
                                                               bool reduce_cols = true,
                                                               const Tensor* mask = nullptr) = 0;
    [[nodiscard]] virtual Result<Tensor> batched_matmul_softmax_denom(const Tensor& A, const Tensor& B,
                                                                      const Tensor& row_max, std::size_t batch,
                                                                      bool transA, bool transB, Scalar alpha,
                                                                      const Tensor* mask = nullptr) = 0;
    [[nodiscard]] virtual Result<Tensor> batched_matmul_softmax_apply(const Tensor& A, const Tensor& B,
                                                                      const Tensor& V, const Tensor& row_max,
                                                                      const Tensor& denom, std::size_t batch,
                                                                      bool transA, bool transB, Scalar alpha,
                                                                      const Tensor* mask = nullptr) = 0;
    [[nodiscard]] virtual Result<Tensor> batched_matmul_softmax_backward_q(
        const Tensor& A, const Tensor& B, const Tensor& P, const Tensor& row_max, const Tensor& denom,
        std::size_t batch, bool transA, bool transB, Scalar alpha, Tensor& r_out,
        const Tensor* mask = nullptr) = 0;
    [[nodiscard]] virtual Result<Tensor> batched_matmul_softmax_backward_kv(
        const Tensor& A, const Tensor& B, const Tensor& P, const Tensor& G, const Tensor& R,
        const Tensor& row_max, const Tensor& denom, std::size_t batch, bool transA, bool transB, Scalar alpha,
        Tensor& grad_v_out, const Tensor* mask = nullptr) = 0;

    // Column softmax primitives for cross-entropy (reference :289-303).
    [[nodiscard]] virtual Result<Tensor> col_softmax_denom(const Tensor& logits, const Tensor& col_max) = 0;
    [[nodiscard]] virtual Result<Tensor> col_softmax_sparse_forward(const Tensor& logits, const Tensor& labels,
                                                                    const Tensor* mask, std::size_t vocab_size,
                                                                    Scalar inv_num_valid,
                                                                    Tensor& loss_vec_out) = 0;

    // In-place updates (reference :306-316).
    [[nodiscard]] virtual Result<void> add_inplace(Tensor& A, const Tensor& B) = 0;
    [[nodiscard]] virtual Result<void> scale_inplace(Tensor& A, Scalar s) = 0;
    [[nodiscard]] virtual Result<void> axpy_inplace(Tensor& A, Scalar scalar, const Tensor& B) = 0;
    [[nodiscard]] virtual Result<void> zero(Tensor& A) = 0;

    // Reductions (reference :324-336).
    [[nodiscard]] virtual Result<Tensor> row_reduce_sum(const Tensor& A) = 0;
    [[nodiscard]] virtual Result<Tensor> col_reduce_sum(const Tensor& A) = 0;
    [[nodiscard]] virtual Result<Tensor> row_reduce_max(const Tensor& A) = 0;
    [[nodiscard]] virtual Result<Tensor> col_reduce_max(const Tensor& A) = 0;

    // Broadcasts (reference :344-350).
    [[nodiscard]] virtual Result<void> broadcast_row_inplace(Tensor& A, const Tensor& row_vec, BinaryOp op) = 0;
    [[nodiscard]] virtual Result<void> broadcast_col_inplace(Tensor& A, const Tensor& col_vec, BinaryOp op) = 0;

    // Elementwise (reference :357-378).
    [[nodiscard]] virtual Result<Tensor> elementwise_unary(UnaryOp op, const Tensor& A) = 0;
    [[nodiscard]] virtual Result<Tensor> elementwise_binary(BinaryOp op, const Tensor& A, const Tensor& B) = 0;
    [[nodiscard]] virtual Result<Tensor> elementwise_binary_scalar(BinaryOp op, const Tensor& A, Scalar s,
                                                                   bool scalar_first = false) = 0;
    [[nodiscard]] virtual Result<Tensor> elementwise_select_scalar_cond(CompareOp cmp, const Tensor& A,
                                                                        Scalar scalar_b, const Tensor& then_t,
                                                                        Scalar scalar_else) = 0;

    // Expression evaluation (reference :392-409).
    [[nodiscard]] virtual Result<Tensor> eval_expr(const ExprSpec& spec, std::span<const Tensor> inputs,
                                                   std::size_t rows, std::size_t cols) = 0;
    [[nodiscard]] virtual Result<Tensor> eval_expr_reduce(const ExprSpec& spec, std::span<const Tensor> inputs,
                                                          std::size_t rows, std::size_t cols)
    {
        (void)spec;
        (void)inputs;
        (void)rows;
        (void)cols;
        return fail("eval_expr_reduce: not supported by this engine");
    }

    // Paged caches and beam search (no reference counterpart; nnhip_kernels.h has the definitions). Activations are
    // (features, tokens): k, v (heads * dim, N), q (q_heads * dim, N); index tensors hold integers as floats.
    // Stores the tokens' keys and values at pos (N) of the sequences seq (N; null: token n of sequence n), k and q
    // turned by rows pos of cos and sin (rows, rope_dim / 2) when these are set; gives q so turned (empty without q).
    [[nodiscard]] virtual Result<Tensor> kv_append(KvPages& cache, const Tensor& k, const Tensor& v, const Tensor* q,
                                                   const Tensor& pos, const Tensor* seq, const Tensor* cos,
                                                   const Tensor* sin)
    {
        (void)cache, (void)k, (void)v, (void)q, (void)pos, (void)seq, (void)cos, (void)sin;
        return fail("kv_append: not supported by this engine");
    }
    // Attention of one query per sequence over its first len (batch) positions; shared (batch / group), when set,
    // counts the positions that each group's sequences have in common. O (q_heads * dim, batch).
    [[nodiscard]] virtual Result<Tensor> attn_paged(const KvPages& cache, const Tensor& q, const Tensor& len,
                                                    const Tensor* shared, std::size_t group, const Tensor* slopes,
                                                    Scalar alpha)
    {
        (void)cache, (void)q, (void)len, (void)shared, (void)group, (void)slopes, (void)alpha;
        return fail("attn_paged: not supported by this engine");
    }
    // The best `take` continuations of each group's beams: logits (vocab, groups * beams), scores and done (size
    // groups * beams; done may be null). Totals (groups, take), and the beams and tokens.
    [[nodiscard]] virtual Result<Tensor> beam_select(const Tensor& logits, const Tensor& scores, const Tensor* done,
                                                     std::size_t groups, std::size_t take, std::size_t eos,
                                                     Tensor& beams_out, Tensor& tokens_out)
    {
        (void)logits, (void)scores, (void)done, (void)groups, (void)take, (void)eos, (void)beams_out, (void)tokens_out;
        return fail("beam_select: not supported by this engine");
    }
    // The page tables of the sequences that continue parent (their tail pages copied into the pages fresh, which may
    // be null); layers share the table. New table, and its lengths in len_out.
    [[nodiscard]] virtual Result<Tensor> kv_reorder(std::span<KvPages> layers, const Tensor& parent, const Tensor& len,
                                                    const Tensor* fresh, Tensor& len_out)
    {
        (void)layers, (void)parent, (void)len, (void)fresh, (void)len_out;
        return fail("kv_reorder: not supported by this engine");
    }
    // Attention of a chunk of new tokens of every sequence: q (q_heads * dim, tokens), of which sequence b has start[b] ..
    // start[b + 1) (start: batch + 1 numbers), at most `most`, the last of its len[b] positions; each sees the positions
    // up to its own. O (q_heads * dim, tokens), zeros for tokens that no sequence has.
    [[nodiscard]] virtual Result<Tensor> attn_chunk(const KvPages& cache, const Tensor& q, const Tensor& start,
                                                    std::size_t most, const Tensor& len, const Tensor* slopes, Scalar alpha)
    {
        (void)cache, (void)q, (void)start, (void)most, (void)len, (void)slopes, (void)alpha;
        return fail("attn_chunk: not supported by this engine");
    }
    // kv_append into 8-bit pages; what they hold of tokens' positions, k and v (heads * dim, tokens), zeros where there is
    // no such row; attn_chunk over them.
    [[nodiscard]] virtual Result<Tensor> kv8_append(KvPages8& cache, const Tensor& k, const Tensor& v, const Tensor* q,
                                                    const Tensor& pos, const Tensor* seq, const Tensor* cos,
                                                    const Tensor* sin)
    {
        (void)cache, (void)k, (void)v, (void)q, (void)pos, (void)seq, (void)cos, (void)sin;
        return fail("kv8_append: not supported by this engine");
    }
    [[nodiscard]] virtual Result<Tensor> kv8_read(const KvPages8& cache, const Tensor& pos, const Tensor* seq, Tensor& v_out)
    {
        (void)cache, (void)pos, (void)seq, (void)v_out;
        return fail("kv8_read: not supported by this engine");
    }
    [[nodiscard]] virtual Result<Tensor> attn_chunk8(const KvPages8& cache, const Tensor& q, const Tensor& start,
                                                     std::size_t most, const Tensor& len, const Tensor* slopes, Scalar alpha)
    {
        (void)cache, (void)q, (void)start, (void)most, (void)len, (void)slopes, (void)alpha;
        return fail("attn_chunk8: not supported by this engine");
    }
    // Which drafted tokens stand, and the token that comes after them (nnhip_draft_verify): the logits (vocab, tokens), or
    // (tokens, vocab) if token_major; start (batch + 1). draft may be null (tokens without probabilities), accept (tokens)
    // and pick (batch) where temperature is 0. Numbers of tokens that stand (batch), and the drawn ones in tokens_out.
    [[nodiscard]] virtual Result<Tensor> draft_verify(const Tensor& target, const Tensor* draft, bool token_major,
                                                      const Tensor& fed, const Tensor& start, std::size_t most,
                                                      Scalar temperature, const Tensor* accept, const Tensor* pick,
                                                      Tensor& tokens_out)
    {
        (void)target, (void)draft, (void)token_major, (void)fed, (void)start, (void)most, (void)temperature, (void)accept;
        (void)pick, (void)tokens_out;
        return fail("draft_verify: not supported by this engine");
    }

    // Queues everything t's values depend on, as a read through the engine
    // would, without waiting (engines that defer work; others have nothing
    // to do). No reference counterpart: the reference reads through to_matrix.
    [[nodiscard]] virtual Result<void> settle_for_read(const Tensor& t)
    {
        (void)t;
        return {};
    }
};

} // namespace nn
