/*
 * ds41 logits for MI355X (gfx950): C ABI of what stands between the head and the samplers
 * (ds41_accept_gfx950.h), and between the samplers and the drafter's next training step:
 *   token table    counts and marks of the tokens a sequence holds
 *   control        penalties, biases and grammar masks on the rows that the samplers read
 *   top logits     the k largest logits of a row, its log-sum-exp, the chosen token's log-probability
 *   distillation   loss and gradient of a drafter's rows against a teacher's top logits
 *   policy loss    loss and gradient of a drafter's or model's rows against how its answers were rated
 *   gradients      their global norm, and clipping
 * No counterparts in the reference (its logits go to the host and from there to the sampler,
 * engine/src/hotpath/batch.inc:496,553). All buffers are caller-owned DEVICE memory; `stream` is a
 * hipStream_t passed as void*; every entry returns a hipError_t value as int, invalid arguments
 * hipErrorInvalidValue (1) before any launch. No entry allocates or synchronises, and every one may be
 * captured into a graph. vocab 1 .. 1,048,576 (as the samplers), rows and sequences 1 .. 65,535 (ds41_logits_control: 1 .. 64
 * rows a sequence).
 * A row stride (ld) counts elements and is at least vocab; rows need the alignment of their element only.
 */
#ifndef DS41_LOGITS_GFX950_H
#define DS41_LOGITS_GFX950_H
#include <stddef.h>
#include <stdint.h>
#include "ds41_accept_gfx950.h"
#ifdef __cplusplus
extern "C" {
#endif

/* Element types of logits, gradients and products. */
enum { DS41_TYPE_F32 = 0, DS41_TYPE_BF16 = 1 };

/* ---- token table --------------------------------------------------------------------
 * Row t of the table is one sequence's: counts uint32 [table_rows][vocab], how often the answer has
 * generated each token, and seen uint32 [table_rows][(vocab + 31) / 32], bit v % 32 of word v / 32 set
 * for every token v that the prompt or the answer holds (so counts[v] > 0 implies the bit). Sequence i of
 * a call is table row table_index[i] (device int32 [n]; NULL: row i); a sequence whose row is outside the
 * table is left out, and so is a token outside the vocabulary. Two sequences of one call may name the same
 * row: their tokens are added to it (integer atomics, so the order of the adds changes nothing). Calls that
 * touch one table must be ordered. */
int ds41_token_counts_clear(uint32_t *counts, uint32_t *seen, int table_rows, int vocab,
                            const int32_t *table_index, int n, void *stream);
/* Sequence i adds tokens[offsets[i] .. offsets[i + 1]) (device int32 [total] and [n + 1]; parts outside
 * 0 .. total are left out): marked, and counted where generated != 0. total may be 0. */
int ds41_token_counts_add(uint32_t *counts, uint32_t *seen, int table_rows, int vocab,
                          const int32_t *table_index, const int32_t *tokens, const int32_t *offsets, int n,
                          int total, int generated, void *stream);
/* Adds what a verify step emitted, read from its device results [n] (ds41_spark_result): tokens[0 .. emitted),
 * counted and marked. A result with emitted < 0 adds nothing. No host wait between verify and commit. */
int ds41_token_counts_commit(uint32_t *counts, uint32_t *seen, int table_rows, int vocab,
                             const int32_t *table_index, const ds41_spark_result *results, int n,
                             void *stream);

/* ---- penalties, biases and grammar masks ---------------------------------------------
 * Logits F32, row s * rows + j of [sequences * rows] for row j of sequence s (a verify step's target rows, or
 * the rows its drafts are drawn from), ld_in apart, to out, ld_out apart. out may be logits (with ld_out ==
 * ld_in; entries that nothing touches are then not written) and must not overlap it otherwise.
 * With c the entry's count in the sequence's table row plus its occurrences among the sequence's drafts
 * before row j (drafts int32 [sequences][draft_ld], the first j of them; entries outside the vocabulary are
 * left out), s whether its mark is set or it occurs among those drafts, and penalties[s] = {repetition,
 * frequency, presence} (F32 [sequences][3]):
 *   x1 = s ? (x > 0 ? x / repetition : x * repetition) : x
 *   x2 = x1 - frequency * c - (c > 0 ? presence : 0)
 *   x3 = x2 + bias
 * in fp32. bias: entries bias_offsets[s] .. bias_offsets[s + 1) (int32 [sequences + 1], clamped to 0 ..
 * bias_total) of bias_ids / bias_values; where an id is listed twice the later entry holds; ids outside the
 * vocabulary are left out. An entry that any of this touches is kept at or above masked_value / 2
 * (-FLT_MAX where masked_value is -infinity), so that a bias of -infinity never pushes an allowed token
 * below the masked ones; NaN stays NaN.
 * mask: uint32 [mask_rows] of mask_ld words, bit set: the grammar allows the token. Row r takes mask row
 * mask_index[r] (int32 [sequences * rows]; NULL: row r), none where that is negative. What is masked becomes
 * masked_value whatever stood there (NaN and infinities too). A row whose mask allows nothing, or whose
 * mask_index is not below mask_rows, becomes NaN throughout, which the samplers reject (emitted -1, token
 * -1), and status bit 8 is set (ds41_take_status). masked_value: -infinity or at most -1e30; the samplers
 * of ds41_accept_gfx950.h reject rows with non-finite entries, so rows meant for them take a finite one
 * (-FLT_MAX).
 * Nullable: counts (NULL: 0 before the drafts), seen (NULL: a token is marked where c > 0), drafts,
 * penalties ({1, 0, 0}), bias_ids, mask. With seen, counts are read only where the mark is set. */
int ds41_logits_control(const float *logits, size_t ld_in, float *out, size_t ld_out, int sequences, int rows,
                        int vocab, const uint32_t *counts, const uint32_t *seen, int table_rows,
                        const int32_t *table_index, const int32_t *drafts, int draft_ld,
                        const float *penalties, const int32_t *bias_ids, const float *bias_values,
                        const int32_t *bias_offsets, int bias_total, const uint32_t *mask, size_t mask_ld,
                        int mask_rows, const int32_t *mask_index, float masked_value, void *stream);

/* ---- top logits --------------------------------------------------------------------
 * For every row of logits (type DS41_TYPE_*, [rows] of ld): its k largest entries in descending order, equal
 * ones by ascending id (-0 equals +0, and is given as +0), as ids int32 [rows][k] and values F32 [rows][k];
 * lse F32 [rows] = log sum exp(x / temperature); logprob F32 [rows] = x[chosen] / temperature - lse for
 * chosen int32 [rows], NaN where that is outside the vocabulary; it is formed from the row's maximum, so that it holds
 * where lse is beyond fp32 (an infinity). ids and values may both be NULL, so may lse,
 * and chosen with logprob. -infinity is an ordinary smallest value; a row with NaN or +infinity gives ids -1
 * and NaN. k 1 .. 128 and at most vocab; temperature from
 * FLT_MIN to 1e38.
 * workspace: ds41_top_logits_workspace_bytes(rows, vocab, k) device bytes, 256-byte aligned, which cover every call of
 * no more rows, entries and k; calls that share one must be ordered. */
size_t ds41_top_logits_workspace_bytes(int rows, int vocab, int k);
int ds41_top_logits(const void *logits, int type, size_t ld, int rows, int vocab, int k, float temperature,
                    int32_t *ids, float *values, float *lse, const int32_t *chosen, float *logprob,
                    void *workspace, size_t workspace_bytes, void *stream);

/* ---- distillation from a teacher's top logits -------------------------------------------
 * For every row: the teacher's top set (teacher_ids int32, teacher_logits F32, both [rows][k], as
 * ds41_top_logits gives them; an entry with an id outside the vocabulary or a logit of -infinity is left out,
 * the probabilities of an id listed twice add up), z the student's row / temperature, q = softmax(z):
 *   p_i = exp(t_i / temperature) / sum over the set           (teacher_lse NULL: renormalised), or
 *   p_i = exp(t_i / temperature - teacher_lse[row])           (teacher_lse F32 [rows], the log-sum-exp of the
 *         teacher's whole row at this temperature); the rest p_r = max(0, 1 - sum p_i) is one more class,
 *         matched with q_r, the student's mass outside the set (0 where the set is the whole vocabulary)
 *   loss = sum p_i (log p_i - log q_i) [+ p_r (log p_r - log q_r)]
 *   d loss / d logit_j = (q_j - p_j) / temperature in the set, and outside it q_j / temperature
 *         [times 1 - p_r / q_r, whose p_r q_j / q_r stays of p_r's size where the set holds nearly all of q]
 * Where every logit outside the set is -infinity, log q_r is -infinity, the loss +infinity if p_r > 0, and the gradient
 * outside 0. What a grammar masks of the student belongs in the renormalised form, or the teacher's rest pulls on it.
 * A row with nothing in its set has loss 0 and gradient 0 whatever its logits hold (padding). loss F32
 * [rows]; stats F32 [rows][2] = {log sum exp z, log q_r (0 when renormalised) + what rounding left of the first},
 * which the backward call takes; both 0 for such a row. The backward call's q are off by the second's own rounding, 2^-25
 * of |log q_r|, and with a rest class by 2^-25 of |log sum exp z| too for bf16 rows and where it writes over the logits;
 * where the two are above 8,192 together one workgroup a row forms them again. A step has none of this. grad: grad_loss[row] (F32 [rows]) times the derivative, in the logits' type, ld_grad
 * apart; grad may be logits (with ld_grad == ld) and must not overlap it otherwise. k 1 .. 128; temperature
 * 0.01 .. 100. ds41_distill_step is forward and backward in one call, for a grad_loss known beforehand.
 * workspace: ds41_distill_workspace_bytes(rows, vocab) device bytes, 256-byte aligned, which cover every call of no
 * more rows and entries; calls that share one must be ordered. */
size_t ds41_distill_workspace_bytes(int rows, int vocab);
int ds41_distill_forward(const void *logits, int type, size_t ld, int rows, int vocab,
                         const int32_t *teacher_ids, const float *teacher_logits, int k,
                         const float *teacher_lse, float temperature, float *loss, float *stats,
                         void *workspace, size_t workspace_bytes, void *stream);
int ds41_distill_backward(const void *logits, int type, size_t ld, int rows, int vocab,
                          const int32_t *teacher_ids, const float *teacher_logits, int k,
                          const float *teacher_lse, float temperature, const float *stats,
                          const float *grad_loss, void *grad, size_t ld_grad, void *stream);
int ds41_distill_step(const void *logits, int type, size_t ld, int rows, int vocab,
                      const int32_t *teacher_ids, const float *teacher_logits, int k,
                      const float *teacher_lse, float temperature, const float *grad_loss, float *loss,
                      float *stats, void *grad, size_t ld_grad, void *workspace, size_t workspace_bytes,
                      void *stream);

/* ---- clipped policy loss with a KL term ------------------------------------------------
 * For every row: z the logits / temperature, a = tokens[row] (int32) the token that was chosen there, log p its
 * log-softmax, old its log-probability when it was chosen and A its advantage (old_logprob, advantage F32 [rows]), ref its
 * log-probability under a reference model (ref_logprob F32 [rows]; not read, and may be NULL, where kl_coef is 0):
 *   r = exp(log p - old)
 *   loss = -min(r A, min(max(r, 1 - clip_low), 1 + clip_high) A) + kl_coef (exp(ref - log p) - (ref - log p) - 1)
 *   d loss / d log p = -r A (0 where the clipped term is the smaller) + kl_coef (1 - exp(ref - log p))
 *   d log p / d logit_j = ((j == a) - softmax(z)_j) / temperature
 * A row whose token is outside the vocabulary (padding) has loss, log p and gradient 0 whatever it holds, and a row with
 * grad_loss 0 or nothing left by the clipping has gradient 0. -infinity is an ordinary logit of a token that is not the
 * chosen one; a row with NaN or +infinity gives NaN.
 * loss, logprob F32 [rows]; stats F32 [rows][3] (the largest of the other logits, the sum of their exponentials from there, the
 * chosen token's logit), which the backward call takes: it forms the step's gradient. grad: grad_loss[row] (F32 [rows]) times the
 * derivative, in the logits' type, ld_grad apart; grad may be logits (with ld_grad == ld). Outputs (the workspace among them) that
 * otherwise share a byte with an input or with another output are refused.
 * clip_low 0 .. 1, clip_high and kl_coef finite and not negative, temperature 0.01 .. 100. ds41_policy_step is forward and
 * backward in one call.
 * workspace: ds41_policy_workspace_bytes(rows, vocab) device bytes, 256-byte aligned, which cover every call of no
 * more rows and entries; calls that share one must be ordered. */
size_t ds41_policy_workspace_bytes(int rows, int vocab);
int ds41_policy_forward(const void *logits, int type, size_t ld, int rows, int vocab, const int32_t *tokens,
                        const float *old_logprob, const float *advantage, const float *ref_logprob,
                        float kl_coef, float clip_low, float clip_high, float temperature, float *loss,
                        float *logprob, float *stats, void *workspace, size_t workspace_bytes, void *stream);
int ds41_policy_backward(const void *logits, int type, size_t ld, int rows, int vocab, const int32_t *tokens,
                         const float *old_logprob, const float *advantage, const float *ref_logprob,
                         float kl_coef, float clip_low, float clip_high, float temperature,
                         const float *stats, const float *grad_loss, void *grad, size_t ld_grad,
                         void *stream);
int ds41_policy_step(const void *logits, int type, size_t ld, int rows, int vocab, const int32_t *tokens,
                     const float *old_logprob, const float *advantage, const float *ref_logprob, float kl_coef,
                     float clip_low, float clip_high, float temperature, const float *grad_loss, float *loss,
                     float *logprob, float *stats, void *grad, size_t ld_grad, void *workspace,
                     size_t workspace_bytes, void *stream);

/* ---- global gradient norm and clipping --------------------------------------------------
 * grads: a HOST array of n descriptions (read before the call returns) of device tensors: count contiguous elements of type
 * DS41_TYPE_*, aligned to their element; count may be 0. n 1 .. DS41_GRAD_MAX, 2^42 elements in all.
 * ds41_grad_norm: norm F32 [1] = sqrt(sum of all squares), square_sum F64 [1] (nullable) the sum itself, for adding over
 * processes. Squares are formed and added in fp64 in a fixed order: the same bits every call for the same list.
 * ds41_grad_clip: out = grad * min(1, max_norm / (*norm + 1e-6)) with norm read on the device; out NULL or grad: in place,
 * where nothing is written if the factor is 1. Factor and product are formed in fp64, rounded to fp32 and, of bf16 gradients,
 * from there to bf16. A norm of infinity gives a factor of 0 (so infinities become NaN), a norm of NaN gives NaN everywhere.
 * ds41_grad_norm_clip: both in one call, with the factor of the norm before its rounding to fp32: infinite only where a
 * gradient is, not where finite gradients have a norm beyond fp32 (then *norm alone is infinity).
 * Outputs that overlap each other, a gradient that is not their own, norm, square_sum or the workspace are refused, as
 * ds41_grad_norm's are over a gradient or each other. max_norm finite and not negative.
 * workspace: ds41_grad_workspace_bytes(n) device bytes, 256-byte aligned; calls that share one must be ordered. */
enum { DS41_GRAD_MAX = 65535 };
typedef struct {
  void *grad;
  void *out;
  uint64_t count;
  int32_t type, reserved;
} ds41_grad;
size_t ds41_grad_workspace_bytes(int n);
int ds41_grad_norm(const ds41_grad *grads, int n, float *norm, double *square_sum, void *workspace,
                   size_t workspace_bytes, void *stream);
int ds41_grad_clip(const ds41_grad *grads, int n, const float *norm, float max_norm, void *stream);
int ds41_grad_norm_clip(const ds41_grad *grads, int n, float max_norm, float *norm, double *square_sum,
                        void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
