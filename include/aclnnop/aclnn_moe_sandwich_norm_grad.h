/*
 * aclnnMoeSandwichNormGrad — the gradients of aclnnMoeSandwichNorm's sumOut and normOut (aclnn_moe_sandwich_norm.h; its int8 rows have none).
 * An operator of this library without a counterpart among the entry points it replaces.
 *
 * Per row, in fp32, with x^ = x * postRstd, s^ = sum * preRstd, g and u as there, ds = sumGrad, dn = normGrad (absent ones are zero):
 *   dS = ds + preRstd * (dn preGamma - s^ * mean(dn preGamma s^))
 *   residualGrad = residualScale * dS                                                                  -> residualGradOutOptional
 *   dv = branchScale * dS;  dg = dv u, times g (1 - g) for gateType 1;  du = dv g
 *   xGrad = postRstd * (du postGamma - x^ * mean(du postGamma x^));  du without postGamma              -> xGradOutOptional
 * and over all rows: postGammaGrad = sum of du x^, preGammaGrad = sum of dn s^, gateGrad = dg summed as the gate was shared (over the rows for a value
 * per channel, over the channels for a value per row).  Column sums are taken in fp32 over up to 512 rows, those sums in 64 bits in a fixed order: equal
 * calls give equal bits.
 *
 * x, sum, sumGradOptional, normGradOptional, residualGradOutOptional, xGradOutOptional: FLOAT, FLOAT16 or BF16 (equal), rank 2 or 3, equal extents, at
 * most 2^26 rows of at most 2^24 values; gammas and gate as there.  normGrad, preGamma and preRstd belong together, and sum with them (not read without),
 * postGamma and postRstd do; sumGrad or normGrad or both.  postRstdOptional, preRstdOptional FLOAT of x's extents without the last.  postGammaGradOutOptional and
 * preGammaGradOutOptional FLOAT [H]; gateGradOutOptional FLOAT of the gate's extents where it is shared, of x's type where it is not; each with its input
 * only.  At least one output.  Inputs may be strided views; outputs are contiguous and share no memory with an input or with each other.  The workspace is
 * 16-byte aligned and one per stream.
 */
#ifndef OPS_TRANSFORMER_AMD_ACLNN_MOE_SANDWICH_NORM_GRAD_H_
#define OPS_TRANSFORMER_AMD_ACLNN_MOE_SANDWICH_NORM_GRAD_H_

#include "acl/acl.h"

#ifdef __cplusplus
extern "C" {
#endif

ACLNN_API aclnnStatus aclnnMoeSandwichNormGradGetWorkspaceSize(
    const aclTensor* x, const aclTensor* sumOptional, const aclTensor* sumGradOptional, const aclTensor* normGradOptional,
    const aclTensor* postGammaOptional, const aclTensor* gateOptional, const aclTensor* preGammaOptional, const aclTensor* postRstdOptional,
    const aclTensor* preRstdOptional, int64_t gateType, double residualScale, double branchScale, const aclTensor* xGradOutOptional,
    const aclTensor* residualGradOutOptional, const aclTensor* postGammaGradOutOptional, const aclTensor* gateGradOutOptional,
    const aclTensor* preGammaGradOutOptional, uint64_t* workspaceSize, aclOpExecutor** executor);

ACLNN_API aclnnStatus aclnnMoeSandwichNormGrad(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream);

#ifdef __cplusplus
}
#endif

#endif  /* OPS_TRANSFORMER_AMD_ACLNN_MOE_SANDWICH_NORM_GRAD_H_ */
