/*
 * fusionvocab.h — C ABI of libfusionmoe.so, continued: the vocabulary operators
 * at the two ends of a model, the token embedding in front of the blocks and the
 * losses behind them that multiply the hidden states with the vocabulary's weight
 * without keeping the logits.
 *
 * The conventions, status codes and dtype codes are those of fusionmoe.h:
 * borrowed device pointers, asynchronous on `stream`, no allocation, no
 * synchronisation, a status instead of an exception.  Indices are int32 or int64
 * (index64 = 0 or 1).
 */
#ifndef FUSIONVOCAB_H
#define FUSIONVOCAB_H

#include "fusionmoe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FMOE_VOCAB_MAX_DIM 16384
#define FMOE_VOCAB_MAX_TOKENS 16777216 /* rows of one call */
#define FMOE_VOCAB_MAX_VOCAB 16777216
#define FMOE_VOCAB_MAX_ELEMENTS 8589934592LL /* of an operand: rows * dim, vocab * dim */
#define FMOE_SCALE_MAX_TENSORS 8
#define FMOE_VOCAB_MAX_TOP 1024        /* listed logits of a teacher per row */

/* ---------------------------------------------------------------------------
 * Token embedding: y[t] = scale * weight[ids[t]], one rounding to y's dtype, which
 * is weight's (dtype).  Row v of weight [vocab, dim] starts at weight + v * ldw; y
 * [T, dim] is dense.  An id outside 0 .. vocab - 1 gives a row of NaN (nothing is read).
 * Pointers need the alignment of their element type only.
 * ------------------------------------------------------------------------- */
int fmoe_embedding_fwd(const void* ids, int index64, const void* weight, int dtype, int64_t ldw,
                       int64_t T, int64_t vocab, int64_t dim, float scale, void* y, void* stream);

/* Its backward: d_weight[v] = scale * sum of dy[t] over the t with ids[t] = v, every row
 * written (zeros where v has no token).  A row is summed in fp32, in a fixed order, without atomics: the
 * same bits every run (up to 64 tokens in their order; more are sorted by id, stably, and an id with many
 * is summed in pieces of 16).  Rows of padding_idx (-1: none) stay zero, ids out of range add nothing.
 * Row t of dy starts at dy + t * lddy.  workspace: 256-byte aligned (up to 64 tokens need none: 0 bytes). */
size_t fmoe_embedding_bwd_workspace_bytes(int64_t T, int64_t vocab, int64_t dim);
int fmoe_embedding_bwd(const void* ids, int index64, const void* dy, int dy_dtype, int64_t lddy,
                       int64_t T, int64_t vocab, int64_t dim, float scale, int64_t padding_idx,
                       void* d_weight, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Losses over a vocabulary.  With s[t, v] = logit_scale / temperature * sum_c hidden[t, c] weight[v, c]
 * and log p[t] = s[t] - logsumexp(s[t]):
 *   cross entropy (teacher NULL, top = 1, temperature 1):  loss[t] = -log p[t, index[t]]
 *   distillation from a teacher's listed logits:  q[t] = softmax(teacher[t] / temperature) over the row's
 *     entries,  loss[t] = temperature^2 * sum_k q[t, k] (log q[t, k] - log p[t, index[t, k]])
 * index [T, top]; an entry whose index is ignore_index, or whose teacher logit is -infinity, is none,
 * and a row without entries has no loss, no gradient, and its hidden state is not read.  An index listed twice
 * counts twice.  Any other index outside 0 .. vocab - 1 makes the row's loss NaN (and with it the gradients).
 * temperature lies in 2^-63 .. 2^63, and |logit_scale| times it or its inverse below 2^126 (factors in fp32).
 * reduction: loss [T] (0 in rows without entries), or one value, the mean over the rows with entries
 * (NaN where there are none) or their sum.
 *
 * The rows with entries are packed, and tiles of the logits are formed on the matrix units, reduced to
 * a maximum and a sum of exponentials per row and dropped; fmoe_vocab_loss_bwd forms them again, a piece
 * of the vocabulary at a time, as G = (p - q) times the row's weight, and multiplies
 *   d_hidden = G weight,  d_weight = G^T hidden.
 * planes = 1: operands and G are bf16 (fp32 operands are rounded), sums fp32.  planes = 3: fp32
 * operands (both), whose rows are taken as two scaled fp16 numbers each for the logits (three products) and, like G, as
 * three bf16 numbers for the gradients (the six largest products; 24 bits of elements down to 2^-109): fp32 precision; up to 64 rows the logits and d_hidden are fp32 products.
 * Long lists of a distillation read their logits from a piece of at most 256 MB in the workspace.
 * The forward's workspace holds a maximum and a sum per row and 128 columns (T vocab / 16 bytes), the backward's a piece of G (2 GiB,
 * or 256 columns) and fp32 sums of d_hidden where there are several.
 * Deterministic, no atomics.
 *
 * state keeps what the backward needs (fmoe_vocab_loss_state_bytes); it belongs to one forward call.
 * workspaces and state: 256-byte aligned.  hidden rows lie ldh apart, weight rows ldw.
 * ------------------------------------------------------------------------- */
enum fmoe_reduction { FMOE_REDUCE_NONE = 0, FMOE_REDUCE_MEAN = 1, FMOE_REDUCE_SUM = 2 };

size_t fmoe_vocab_loss_state_bytes(int64_t T, int64_t dim, int64_t top, int planes);
/* 1 where the products read a copy of weight, made a piece at a time, rather than weight as it lies
 * (bf16 rows of a multiple of 64 elements at 16-byte addresses): an argument of the size queries. */
int fmoe_vocab_loss_packs(const void* weight, int w_dtype, int64_t ldw, int64_t dim, int planes);
size_t fmoe_vocab_loss_fwd_workspace_bytes(int64_t T, int64_t dim, int64_t vocab, int64_t top, int planes, int packs);
int fmoe_vocab_loss_fwd(const void* hidden, int h_dtype, int64_t ldh, const void* weight, int w_dtype,
                        int64_t ldw, const void* index, int index64, const void* teacher, int t_dtype,
                        int64_t T, int64_t dim, int64_t vocab, int64_t top, int64_t ignore_index,
                        double logit_scale, double temperature, int planes, int reduction, float* loss,
                        void* state, size_t state_bytes, void* workspace, size_t workspace_bytes,
                        void* stream);

/* Backward of the call that wrote state, whose sizes and options are repeated here.  d_loss: one fp32 value, or T
 * of them where reduction is none.  d_hidden [T, dim] and d_weight [vocab, dim] are dense and written whole; either may be NULL (not
 * wanted). */
size_t fmoe_vocab_loss_bwd_workspace_bytes(int64_t T, int64_t dim, int64_t vocab, int planes, int packs);
int fmoe_vocab_loss_bwd(const float* d_loss, const void* weight, int w_dtype, int64_t ldw, int64_t T,
                        int64_t dim, int64_t vocab, int64_t top, int distill, double logit_scale,
                        double temperature, int planes, int reduction, const void* state,
                        size_t state_bytes, void* d_hidden, int dh_dtype, void* d_weight, int dw_dtype,
                        void* workspace, size_t workspace_bytes, void* stream);

/* The forward and the gradients of a loss of one value (mean or sum, for d_loss = 1) in one call, without
 * forming the logits twice: a piece of the rows at a time, whose exponentials 2^(s - o), o the logit of the row's
 * target (or the largest listed one), are G up to a factor per row.  Those factors go into d_hidden, and with hidden into
 * the product of d_weight: with planes = 1 the scaled hidden states are rounded to bf16 once more.  Rows whose
 * sum of such exponentials leaves 2^-60 .. 2^60 (a loss of 41.6; or is no number) make their piece be formed in the ordinary way.
 * d_hidden and d_weight as in fmoe_vocab_loss_bwd.  The size query returns 0 where this form is not taken (up to 64
 * rows; vocabularies of which no piece of 2048 rows fits 2 GiB): FMOE_ERR_SHAPE.  There is no state. */
size_t fmoe_vocab_loss_grad_workspace_bytes(int64_t T, int64_t dim, int64_t vocab, int64_t top, int planes, int packs);
int fmoe_vocab_loss_fwd_grad(const void* hidden, int h_dtype, int64_t ldh, const void* weight, int w_dtype,
                             int64_t ldw, const void* index, int index64, const void* teacher, int t_dtype,
                             int64_t T, int64_t dim, int64_t vocab, int64_t top, int64_t ignore_index,
                             double logit_scale, double temperature, int planes, int reduction, float* loss,
                             void* d_hidden, int dh_dtype, void* d_weight, int dw_dtype, void* workspace,
                             size_t workspace_bytes, void* stream);

/* dst[i] = scale[0] * src[i] for up to FMOE_SCALE_MAX_TENSORS tensors of n[i] elements of dtype[i] (host arrays; fp32
 * arithmetic, one rounding).  src[i] == dst[i]: in place, and nothing is touched where scale[0] is 1 (gradients
 * whose loss's gradient arrives later). */
int fmoe_scale(const float* scale, const void* const* src, void* const* dst, const int* dtype, const int64_t* n,
               int n_tensors, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FUSIONVOCAB_H */
