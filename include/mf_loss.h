/*
 * mf_loss.h — C-ABI of the losses over the tied output table.
 *
 * The dense head (mf_dense_head_f16) answers with the table; these entry
 * points train it and score with it: softmax cross entropy over the whole
 * vocabulary and distillation from a teacher's top logits, each with its
 * gradients.  The scores of the vocabulary are made in pieces and never kept.
 * No counterpart in the reference, which only decodes.
 *
 *   s[r][v] = hidden[r] . embedding[v]                      (FP32)
 *   cross entropy  loss[r] = lse[r] - s[r][target[r]],
 *                  lse[r] = log sum_v exp(s[r][v])
 *   distillation   q[r] = softmax of the teacher's logits / T over the row's
 *                  set, lse[r] = log sum_v exp(s[r][v] / T),
 *                  loss[r] = T^2 KL(q[r] || softmax(s[r] / T))
 *                          = T^2 sum_k q_k (log q_k - s[r][id_k] / T + lse[r])
 *   gradients      with g = grad_losses, p[r][v] = exp(s[r][v] / T - lse[r]) and
 *                  d[r][v] = T g[r] (p[r][v] - q[r][v])  (T = 1 and q one at
 *                  the target for cross entropy):
 *                  d_hidden = d . embedding, d_embedding = d^T . hidden
 *
 * MF_LOSS_MAX_ROWS: the tensor core's sums lose up to 4e-9 a product of a sum
 * that grows steadily, so d_embedding of more rows in one call would lose what
 * its type holds; larger batches go in slices whose gradients the caller adds.
 *
 * Scores come from the tensor cores: relative to a score, an error of up to
 * about 3e-9 a product of its width remains (bfloat16 2e-9).  A target's own score is summed
 * with rounding to nearest.  A call's losses, lse and gradients are made of the
 * same scores, so where p and q are nearly equal, p - q is good to lse's
 * rounding to f32, 2^-24 |lse|, and the loss to a few 2^-24.
 * Scores over T beyond 1e9 in magnitude may give infinities.
 *
 * Types: _f16 takes fp16 and _bf16 bfloat16 hidden rows and table; gradients
 * have the type of what they are the gradient of.  Losses, lse, grad_losses
 * and teacher logits are f32, every sum is held in FP32, and d is rounded once
 * to the 16-bit type for the two gradient products (up to 64 rows: to the sum
 * of two such numbers).
 * fp16 gradients beyond 65504 become infinite; in d_embedding, what a row of a
 * small weight adds is good to 2^-25 of the call's largest weight, which fp16
 * keeps of a hidden element times its row's share of that weight.
 *
 * Arguments are validated as mf_head.h says, before any launch, with these
 * additions: hidden_size is a multiple of 8 up to MF_LOSS_MAX_HIDDEN, rows at
 * most MF_LOSS_MAX_ROWS, vocab at most MF_LOSS_MAX_VOCAB, entries at most
 * MF_LOSS_MAX_ENTRIES (MF_RESOURCE_LIMIT otherwise); hidden, embedding,
 * d_hidden and d_embedding are 16-byte aligned and the workspace 256-byte (as
 * cudaMalloc gives it), and no output and no workspace overlaps another buffer
 * (MF_INVALID_ARGUMENT otherwise).  The current device must be the one that
 * owns the buffers and the stream.
 *
 * Rows: a cross entropy row whose target is MF_INVALID_TOKEN (what the heads
 * write for a row without a candidate), and a distillation row with an empty
 * set or only -inf teacher logits, is ignored: loss 0, no gradient.  A row
 * with any other target >= vocab, an id outside the vocabulary, ids that do
 * not ascend strictly (the same id twice included), a NaN or +inf teacher
 * logit, or offsets that decrease or leave [0, entries], is invalid: loss NaN,
 * no gradient.  Neither kind, nor a row whose grad_losses is 0, takes part in
 * the gradients: its d_hidden row is 0 and what its hidden row holds (NaN
 * included) does not reach d_embedding.  lse is written for every row.
 * Elsewhere a score of NaN or +inf gives its row a NaN loss and NaN gradients.
 * A score of -inf (a table row masked by a bias column) has p = 0: it adds
 * nothing to lse, and a loss that asks for it is +inf; so do scores over T below
 * -1.5e9 beside others that are not.  A row whose scores are all -inf has lse
 * -inf and a NaN loss.  Products with an infinite table element make d_hidden
 * NaN as 0 times it is; a masked table that trains holds a large negative
 * number, whose products with 0 are 0.
 *
 * Every wait inside the kernels is bounded (100 ms); one that runs out gives
 * NaN in the outputs it covers, and the context stays usable.
 *
 * The workspace needs no initialisation and holds nothing between calls; calls
 * that share one must not overlap on the GPU.  All calls may be captured
 * into a CUDA graph, and results do not change from run to run.
 */
#ifndef MF_LOSS_H
#define MF_LOSS_H

#include "mf_head.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MF_LOSS_MAX_ROWS (1u << 16)
#define MF_LOSS_MAX_VOCAB (1u << 24)
#define MF_LOSS_MAX_HIDDEN 8192u
/* of a teacher's sets: 32-bit indices that step past their end stay positive */
#define MF_LOSS_MAX_ENTRIES ((1u << 31) - 1024u)

/* Bytes of device memory that a forward call and a backward call of at most
 * `rows` rows need; 0 for sizes outside the limits.  A backward call's holds up
 * to two pieces of d of at most 128 MiB, a copy of the hidden rows (two up to 64
 * rows), and FP32 sums of d_hidden of at most 128 MiB (4 bytes an element above
 * 32 Mi elements). */
MF_API uint64_t mf_dense_loss_workspace_bytes(uint64_t rows, uint64_t hidden_size, uint64_t vocab);
MF_API uint64_t mf_dense_loss_backward_workspace_bytes(uint64_t rows, uint64_t hidden_size,
                                                       uint64_t vocab);

/* Cross entropy.  hidden [rows, hidden_size], embedding [vocab, hidden_size],
 * targets u32 [rows]; losses f32 [rows], lse f32 [rows].  With one row this is
 * the log-probability (negated) of one chosen token. */
MF_API mf_status mf_dense_xent_f16(const void* hidden, uint64_t hidden_bytes,
                                   const void* embedding, uint64_t embedding_bytes,
                                   const void* targets, uint64_t targets_bytes, void* losses,
                                   uint64_t losses_bytes, void* lse, uint64_t lse_bytes,
                                   void* workspace, uint64_t workspace_bytes, uint64_t rows,
                                   uint64_t hidden_size, uint64_t vocab, void* stream);
MF_API mf_status mf_dense_xent_bf16(const void* hidden, uint64_t hidden_bytes,
                                    const void* embedding, uint64_t embedding_bytes,
                                    const void* targets, uint64_t targets_bytes, void* losses,
                                    uint64_t losses_bytes, void* lse, uint64_t lse_bytes,
                                    void* workspace, uint64_t workspace_bytes, uint64_t rows,
                                    uint64_t hidden_size, uint64_t vocab, void* stream);

/* Its gradients.  lse as the forward call wrote it for the same hidden rows
 * and table; grad_losses f32 [rows]; d_hidden [rows, hidden_size] and
 * d_embedding [vocab, hidden_size] are overwritten, either may be NULL (0
 * bytes), not both. */
MF_API mf_status mf_dense_xent_backward_f16(
    const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,
    const void* targets, uint64_t targets_bytes, const void* lse, uint64_t lse_bytes,
    const void* grad_losses, uint64_t grad_losses_bytes, void* d_hidden, uint64_t d_hidden_bytes,
    void* d_embedding, uint64_t d_embedding_bytes, void* workspace, uint64_t workspace_bytes,
    uint64_t rows, uint64_t hidden_size, uint64_t vocab, void* stream);
MF_API mf_status mf_dense_xent_backward_bf16(
    const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,
    const void* targets, uint64_t targets_bytes, const void* lse, uint64_t lse_bytes,
    const void* grad_losses, uint64_t grad_losses_bytes, void* d_hidden, uint64_t d_hidden_bytes,
    void* d_embedding, uint64_t d_embedding_bytes, void* workspace, uint64_t workspace_bytes,
    uint64_t rows, uint64_t hidden_size, uint64_t vocab, void* stream);

/* Distillation.  The teacher's top logits are a ragged CSR batch, as the
 * allowed sets of mf_head_restricted_csr_f16: row r's entries are
 * [offsets[r], offsets[r+1]) of ids (i32, ascending strictly within the row)
 * and teacher_logits (f32).  offsets i32 [rows + 1].  temperature T is finite
 * and > 0.  A batch without entries passes NULL ids and logits. */
MF_API mf_status mf_dense_distill_f16(
    const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,
    const void* offsets, uint64_t offsets_bytes, const void* ids, uint64_t ids_bytes,
    const void* teacher_logits, uint64_t teacher_logits_bytes, float temperature, void* losses,
    uint64_t losses_bytes, void* lse, uint64_t lse_bytes, void* workspace,
    uint64_t workspace_bytes, uint64_t rows, uint64_t hidden_size, uint64_t vocab, void* stream);
MF_API mf_status mf_dense_distill_bf16(
    const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,
    const void* offsets, uint64_t offsets_bytes, const void* ids, uint64_t ids_bytes,
    const void* teacher_logits, uint64_t teacher_logits_bytes, float temperature, void* losses,
    uint64_t losses_bytes, void* lse, uint64_t lse_bytes, void* workspace,
    uint64_t workspace_bytes, uint64_t rows, uint64_t hidden_size, uint64_t vocab, void* stream);

/* Its gradients; lse as the forward call wrote it with the same temperature. */
MF_API mf_status mf_dense_distill_backward_f16(
    const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,
    const void* offsets, uint64_t offsets_bytes, const void* ids, uint64_t ids_bytes,
    const void* teacher_logits, uint64_t teacher_logits_bytes, float temperature, const void* lse,
    uint64_t lse_bytes, const void* grad_losses, uint64_t grad_losses_bytes, void* d_hidden,
    uint64_t d_hidden_bytes, void* d_embedding, uint64_t d_embedding_bytes, void* workspace,
    uint64_t workspace_bytes, uint64_t rows, uint64_t hidden_size, uint64_t vocab, void* stream);
MF_API mf_status mf_dense_distill_backward_bf16(
    const void* hidden, uint64_t hidden_bytes, const void* embedding, uint64_t embedding_bytes,
    const void* offsets, uint64_t offsets_bytes, const void* ids, uint64_t ids_bytes,
    const void* teacher_logits, uint64_t teacher_logits_bytes, float temperature, const void* lse,
    uint64_t lse_bytes, const void* grad_losses, uint64_t grad_losses_bytes, void* d_hidden,
    uint64_t d_hidden_bytes, void* d_embedding, uint64_t d_embedding_bytes, void* workspace,
    uint64_t workspace_bytes, uint64_t rows, uint64_t hidden_size, uint64_t vocab, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MF_LOSS_H */
