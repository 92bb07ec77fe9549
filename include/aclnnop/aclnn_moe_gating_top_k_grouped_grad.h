/*
 * aclnnMoeGatingTopKGroupedGrad — the gradient with respect to a router's logits, of the weights of the experts that aclnnMoeGatingTopKGrouped (or
 * aclnnMoeGatingTopKSoftmaxV2) picked, of aclnnMoeBalanceLoss, or of both in one pass.
 * An operator of this library without a counterpart among the entry points it replaces.
 *
 * Per row, p = softmax(x) (scoreType 0) or sigmoid(x) (scoreType 1), ids expertIdx_1..k, dy = yGrad (the choice itself has no gradient, and neither has
 * the bias that steers it):
 *   dp_e = sum over the j with id e of routedScalingFactor * (renorm 0: dy_j;  renorm 1: (dy_j - sum_i dy_i p_i / t) / t with t = sum_i p_i + eps)
 *   xGrad = p (dp - sum_e dp_e p_e)  (softmax),  p (1 - p) dp  (sigmoid)
 * and, for rows of sequence s, with r and n as in aclnn_moe_balance_loss.h, added to it:
 *   dr_e = lossGrad_s * E / (k n^2) * counts_se
 *   r (dr - sum_e dr_e r_e)  (softmax),  r (1 - p) (dr - sum_e dr_e r_e)  (sigmoid)
 * A row whose first id lies outside [0, E) has zeros; another such id has no part in the sums; with renorm a row whose picked p are all zero in 64 bits (the
 * choice has its weights in them) has dp = 0; picked p that only fp32 loses have their shares all the same.
 * Rows in no sequence have no gradient of the loss.  Everything is fp32, rounded once to xGrad's type.
 *
 * x, expertIdx, seqOffsetsOptional: as aclnnMoeBalanceLoss takes them; yGradOptional of x's type or FLOAT, expertIdx's extents; lossGradOptional FLOAT [S],
 * countsOptional INT32 [S, E] and rowsOptional INT32 [S], the three together; yGrad or these or both; seqOffsets only with these.  xGradOut of x's type or
 * FLOAT, x's extents.  renorm, routedScalingFactor and eps belong to yGrad.  Inputs may be strided views; xGradOut is contiguous and shares no memory with
 * an input.
 */
#ifndef OPS_TRANSFORMER_AMD_ACLNN_MOE_GATING_TOP_K_GROUPED_GRAD_H_
#define OPS_TRANSFORMER_AMD_ACLNN_MOE_GATING_TOP_K_GROUPED_GRAD_H_

#include "acl/acl.h"

#ifdef __cplusplus
extern "C" {
#endif

ACLNN_API aclnnStatus aclnnMoeGatingTopKGroupedGradGetWorkspaceSize(
    const aclTensor* x, const aclTensor* expertIdx, const aclTensor* yGradOptional, const aclTensor* lossGradOptional, const aclTensor* countsOptional,
    const aclTensor* rowsOptional, const aclTensor* seqOffsetsOptional, int64_t scoreType, int64_t renorm, double routedScalingFactor, double eps,
    const aclTensor* xGradOut, uint64_t* workspaceSize, aclOpExecutor** executor);

ACLNN_API aclnnStatus aclnnMoeGatingTopKGroupedGrad(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream);

#ifdef __cplusplus
}
#endif

#endif  /* OPS_TRANSFORMER_AMD_ACLNN_MOE_GATING_TOP_K_GROUPED_GRAD_H_ */
