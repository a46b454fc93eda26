/*
 * zg_hip_topk.h -- operators built on the k largest values of a row: selection and its gradient, the loss of a student
 * against a teacher's k largest logits, and layers of experts in which each row goes to the k experts its router scores
 * highest.  No counterparts in the reference, whose selection ends at the single maximum (argmax along a dimension), whose
 * losses take one-hot or integer labels and whose Linear layers apply one weight matrix to all rows.
 *
 * The conventions of zg_hip.h hold: fp32 values, uint64_t indices (device memory or zg_hip_host_alloc memory, 8-byte
 * aligned), dense row-major arrays at any 4-byte alignment, asynchronous calls in order on the context's stream, arguments
 * checked on the host before any launch, ZG_HIP_E* codes.  These calls hold nothing back: what waits in the context is
 * launched first, their own kernels before they return.  They can be recorded into an execution graph; where a comment says
 * that a call uses the context's workspace, run it once eagerly with the same sizes first.  Results do not depend on
 * scheduling: no call adds through atomics.  An output may not overlap another operand of its call (ZG_HIP_EINVAL).
 */
#ifndef ZG_HIP_TOPK_H
#define ZG_HIP_TOPK_H
#include "zg_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    ZG_HIP_TOPK_MAX_K = 512,       /* k of selection and of distillation */
    ZG_HIP_EXPERTS_MAX = 1024,     /* experts of a layer */
    ZG_HIP_EXPERTS_MAX_K = 64,     /* experts per row */
};

/* ---------------------------------------------------------------------------------------------
 * selection.  values[r, :] = the k largest of x[r, :] in descending order, indices[r, :] their columns.  Equal values
 * (+0 and -0 are equal) come in the order of their columns; a NaN counts as larger than any number, as in zg_hip_max_fwd.
 * 1 <= k <= min(cols, ZG_HIP_TOPK_MAX_K), cols < 2^31; no rows: nothing to do.  Few long rows use the workspace.
 * ------------------------------------------------------------------------------------------- */
int zg_hip_topk_fwd(zg_hip_ctx *ctx, const float *x, float *values, uint64_t *indices, size_t rows, size_t cols, size_t k);
/* x_g[r, indices[r, j]] += y_g[r, j]; accumulate == 0: x_g is written, zero in every place that was not chosen.  Indices that
 * are not below cols take part in nothing; the gradients of an index that stands in a row more than once are added in the
 * order of j. */
int zg_hip_topk_bwd(zg_hip_ctx *ctx, const uint64_t *indices, const float *y_g, float *x_g, size_t rows, size_t cols,
                    size_t k, int accumulate);

/* ---------------------------------------------------------------------------------------------
 * distillation from a teacher's k largest logits (values and columns, as zg_hip_topk_fwd gives them; 1 <= k <=
 * ZG_HIP_TOPK_MAX_K).  With q = softmax(teacher[r, :] / temperature) over the k kept logits and p = softmax(logits[r, :] /
 * temperature) over all classes:
 *   row_loss[r] = temperature^2 sum_j q_j (log q_j - log p_{indices[r, j]})
 *   loss        = sum_r w_r row_loss[r]              w = row_weights (finite), or 1 / rows each when row_weights is null
 *   grad[r, c] += w_r temperature (p_c - sum of the q_j whose index is c)      accumulate == 0: grad is written, not read
 * An index that is not below cols is padding: its logit is left out of q.  A row adds exactly nothing (row_loss 0, gradient
 * 0, whatever its logits hold) when its weight is 0, when it has no teacher logit above -inf, or when all its logits
 * are -inf.  A class of p = 0 that the teacher wants (q > 0) makes the row's loss infinite and leaves its gradient finite.
 * stats[r, :] = { max_c logits, log sum_c exp((logits - max) / temperature) }, {-inf, 0} for a row whose logits are all -inf,
 * {0, 0} for a row of weight 0 (its logits are not read): what zg_hip_distill_bwd needs of the row.  1e-18 <=
 * temperature <= 1e18; cols < 2^31.  As with the other losses the forward calls refuse an empty matrix and the backward does
 * nothing on one.
 * ------------------------------------------------------------------------------------------- */
int zg_hip_distill_fwd(zg_hip_ctx *ctx, const float *logits, const float *teacher, const uint64_t *indices,
                       const float *row_weights, float *stats, float *row_loss, float *loss, size_t rows, size_t cols,
                       size_t k, float temperature);
int zg_hip_distill_bwd(zg_hip_ctx *ctx, const float *logits, const float *teacher, const uint64_t *indices,
                       const float *row_weights, const float *stats, float *grad, size_t rows, size_t cols, size_t k,
                       float temperature, int accumulate);
/* forward and the backward of the scalar loss (upstream gradient 1) in one call; rows of up to 65536 columns are read once,
 * longer ones twice */
int zg_hip_distill_fwd_bwd(zg_hip_ctx *ctx, const float *logits, const float *teacher, const uint64_t *indices,
                           const float *row_weights, float *stats, float *row_loss, float *loss, float *grad, size_t rows,
                           size_t cols, size_t k, float temperature, int accumulate);

/* ---------------------------------------------------------------------------------------------
 * rows to experts and back.  Entry i = t * k + j says that row t goes to experts[i] with weight weights[i]; an expert that is
 * not below n_experts drops the entry (a full expert, a padding row).
 *   expert_sort      orders the entries by expert, those of one expert by i: slots[i] = the entry's place in that order,
 *                    UINT64_MAX for a dropped one; expert e owns the places offsets[e] .. offsets[e + 1] - 1.  offsets has
 *                    n_experts + 1 entries.  1 <= n_experts <= ZG_HIP_EXPERTS_MAX, n_entries < 2^32 - 1.  Uses the workspace
 *                    beyond 2048 entries.
 *   expert_dispatch  y[slots[t * k + j], :] = x[t, :].  y has n_tokens * k rows; those behind the last place are left as they were.
 *   expert_dispatch_bwd  x_g[t, :] += sum over j of y_g[slots[t * k + j], :], in the order of j; accumulate == 0: written.
 *   expert_combine   out[t, :] = sum over j of weights[t, j] y[slots[t * k + j], :], in the order of j (zeros for a row with no
 *                    entry).
 *   expert_combine_bwd  y_g[slots[t * k + j], :] = weights[t, j] out_g[t, :] and weights_g[t, j] = <out_g[t, :], y[slots[t * k + j], :]>
 *                    (0 for a dropped entry); y_g or weights_g may be null, y too when weights_g is.  Rows of y_g behind the last
 *                    place are left as they were.
 * A slot that is not below n_tokens * k counts as dropped; the slots below it must differ.  1 <= k <= ZG_HIP_EXPERTS_MAX_K;
 * no tokens or a width of 0: nothing to do (expert_sort of no entries writes offsets of 0).
 * ------------------------------------------------------------------------------------------- */
int zg_hip_expert_sort(zg_hip_ctx *ctx, const uint64_t *experts, uint64_t *offsets, uint64_t *slots, size_t n_entries,
                       size_t n_experts);
int zg_hip_expert_dispatch(zg_hip_ctx *ctx, const float *x, const uint64_t *slots, float *y, size_t n_tokens, size_t k,
                           size_t width);
int zg_hip_expert_dispatch_bwd(zg_hip_ctx *ctx, const float *y_g, const uint64_t *slots, float *x_g, size_t n_tokens, size_t k,
                               size_t width, int accumulate);
int zg_hip_expert_combine(zg_hip_ctx *ctx, const float *y, const uint64_t *slots, const float *weights, float *out,
                          size_t n_tokens, size_t k, size_t width);
int zg_hip_expert_combine_bwd(zg_hip_ctx *ctx, const float *out_g, const float *y, const uint64_t *slots, const float *weights,
                              float *y_g, float *weights_g, size_t n_tokens, size_t k, size_t width);

/* ---------------------------------------------------------------------------------------------
 * the experts' Linear layers: zg_hip_linear_fwd and zg_hip_linear_bwd with weights w[e, fan_out, fan_in] and bias[e, fan_out]
 * for the rows offsets[e] .. offsets[e + 1] - 1 (as zg_hip_expert_sort leaves them in device memory: the host never needs the
 * counts).  Rows behind offsets[n_experts] are neither read nor written; offsets beyond n_rows are taken as n_rows and a range that ends
 * before it begins as empty.  The ranges must not overlap, which offsets that never decrease can not: where they do, what the rows of y and
 * gx in the overlapping ranges hold afterwards is undefined (gw_e and gb_e are sums over expert e's range all the same, and nothing
 * outside the ranges is touched).  n_rows < 2^31, fan_in and fan_out < 2^21, n_experts <= ZG_HIP_EXPERTS_MAX.
 *   forward   y = x w_e^T + bias_e (null: none), max(0, .) when relu
 *   backward  gw_e += gy_e^T x_e;  gb_e += column sums of gy_e (null: none);  gx = gy w_e, zero where act_in <= 0 (gx null: no
 *             input gradient, w is not read; act_in null: no mask).  accumulate == 0: gw and gb are written, zero for an
 *             expert without rows.  A layer without inputs or outputs: nothing to do.  Uses the workspace when there
 *             are more than 64 experts, when gb is given, and for layers so small that the rows are cut into parts.
 * ------------------------------------------------------------------------------------------- */
int zg_hip_expert_linear_fwd(zg_hip_ctx *ctx, const float *x, const float *w, const float *bias, float *y,
                             const uint64_t *offsets, size_t n_rows, size_t n_experts, size_t fan_in, size_t fan_out, int relu);
int zg_hip_expert_linear_bwd(zg_hip_ctx *ctx, const float *gy, const float *x, const float *w, const float *act_in, float *gw,
                             float *gb, float *gx, const uint64_t *offsets, size_t n_rows, size_t n_experts, size_t fan_in,
                             size_t fan_out, int accumulate);

#ifdef __cplusplus
}
#endif
#endif
