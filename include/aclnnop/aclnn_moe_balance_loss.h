/*
 * aclnnMoeBalanceLoss — how evenly a router spreads a batch over its experts: picks per expert, mean probability per expert, and the loss that
 * their product is, for each sequence of the batch.
 * An operator of this library beside aclnnMoeGatingTopKGrouped and aclnnMoeGatingTopKSoftmaxV2, whose logits and expert ids it takes.  Its gradient is
 * aclnnMoeGatingTopKGroupedGrad (aclnn_moe_gating_top_k_grouped_grad.h).
 *
 * The T rows of x are cut into S sequences: sequence s holds rows seqOffsets[s] to seqOffsets[s + 1] - 1; rows in front of the first and behind the last
 * count nowhere; without seqOffsets all rows are one sequence.  A row whose first expert id lies outside [0, E) (the gating operators write E into
 * finished rows) counts nowhere either.  Over the n rows of a sequence that count:
 *   r = softmax(x) (scoreType 0), or sigmoid(x) divided by its sum over the row (scoreType 1)
 *   counts_e = how often e is among their k ids (an id outside [0, E) is none, one that comes twice counts twice)       -> countsOut
 *   prob_e = mean of r_e                                                                                                -> probOutOptional
 *   loss = E / (k n) * sum over e of counts_e prob_e   (1 where both are even)                                          -> lossOut;  n -> rowsOut
 * A sequence without such rows has zeros.  A logit of -inf has r = 0, a row of nothing else r = 0 throughout; NaN (and under softmax +inf) makes its row's r
 * NaN.  Probabilities are summed in fp32 over up to 4096 rows, those sums in 64 bits, all in a fixed order: equal calls
 * give equal bits.
 *
 * x: FLOAT, FLOAT16 or BF16, rank 2 or 3, at most 2^26 rows and 2048 experts; expertIdx INT32 of x's extents with the last replaced by k, 1 to 64, at most
 * 2^31 - 1 ids in all, of which one expert may be every one;
 * seqOffsetsOptional INT32 or INT64 [S + 1], S from 1 to 2^20, not falling (else: unspecified values, no access outside the tensors); lossOut FLOAT [S]; countsOut
 * INT32 [S, E]; rowsOut INT32 [S]; probOutOptional FLOAT [S, E] ([1] and [1, E] without seqOffsets).  Inputs may be strided views; outputs are contiguous
 * and share no memory with an input or with each other.  The workspace is 16-byte aligned and one per stream.
 */
#ifndef OPS_TRANSFORMER_AMD_ACLNN_MOE_BALANCE_LOSS_H_
#define OPS_TRANSFORMER_AMD_ACLNN_MOE_BALANCE_LOSS_H_

#include "acl/acl.h"

#ifdef __cplusplus
extern "C" {
#endif

ACLNN_API aclnnStatus aclnnMoeBalanceLossGetWorkspaceSize(const aclTensor* x, const aclTensor* expertIdx, const aclTensor* seqOffsetsOptional,
                                                          int64_t scoreType, const aclTensor* lossOut, const aclTensor* countsOut,
                                                          const aclTensor* rowsOut, const aclTensor* probOutOptional, uint64_t* workspaceSize,
                                                          aclOpExecutor** executor);

ACLNN_API aclnnStatus aclnnMoeBalanceLoss(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream);

#ifdef __cplusplus
}
#endif

#endif  /* OPS_TRANSFORMER_AMD_ACLNN_MOE_BALANCE_LOSS_H_ */
