/*
 * aclnnMoeRouterLogits — the router's product: logits = x @ weight^T in fp32.
 * An operator of this library without a counterpart among the entry points it replaces: what makes the logits that
 * aclnnMoeGatingTopKSoftmaxV2 and aclnnMoeGatingTopKGrouped take, from the rows of aclnnMoeAddRmsNormQuant.
 *
 *   logitsOut[..., e] = sum over h of x[..., h] * weight[e, h], products and sums in fp32
 * Router weights are often kept in 32 bits next to 16-bit hidden states: neither side is rounded to fewer bits than it has.
 * (Where x is FLOAT or FLOAT16 next to FLOAT weights both are sums of bf16 parts, and products of parts that are left out come to at most 2^-23 of |x w|.)
 * Results are the same bits on every launch.  A row with a NaN or an infinity gives NaN or infinities; so does, where x is FLOAT or
 * FLOAT16 next to FLOAT weights, a FLOAT value of 2^128 (1 - 2^-9) or more.
 *
 * x: FLOAT, FLOAT16 or BF16, rank 2 or 3, at most 2^26 rows, last extent H; weight: of x's type or FLOAT, [E, H], 1 <= E <= 4096;
 * logitsOut: FLOAT of x's extents with the last replaced by E, contiguous, apart from the inputs' memory.  Inputs may be
 * strided views (copied into the workspace first).  Two calls may not share a workspace on different streams.
 */
#ifndef OPS_TRANSFORMER_AMD_ACLNN_MOE_ROUTER_LOGITS_H_
#define OPS_TRANSFORMER_AMD_ACLNN_MOE_ROUTER_LOGITS_H_

#include "acl/acl.h"

#ifdef __cplusplus
extern "C" {
#endif

ACLNN_API aclnnStatus aclnnMoeRouterLogitsGetWorkspaceSize(const aclTensor* x, const aclTensor* weight, const aclTensor* logitsOut,
                                                           uint64_t* workspaceSize, aclOpExecutor** executor);

ACLNN_API aclnnStatus aclnnMoeRouterLogits(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream);

#ifdef __cplusplus
}
#endif
#endif
