/* Log probabilities of given tokens, with entropy and the most likely alternatives, and their gradient: what a model's logits say.
 * Extension (no counterpart in the reference).
 *
 * With z = scale * logits of a row, in float32:
 *     lse = log(sum exp(z)),  logProb = z[token] - lse,  p = exp(z - lse),  entropy = -sum p * (z - lse) (0 where p is 0);
 *     logProb is 0 where the token is outside [0, V) (padding).
 * topTokens are the K tokens of the largest logits, the largest first, of equal ones (+0 and -0 are) the lowest first, a NaN before
 * all numbers; topValues their log probabilities. A row whose logits are all -infinity: lse and all log probabilities are -infinity (0
 * for padding), entropy 0. A row with NaN or +infinity: NaN, except topTokens and padding's 0.
 * Gradient, with g = gradOut (0 for padding) and h = gradEntropy (0 without it):
 *     gradLogits[j] = scale * (g * ([j == token] - p_j) - h * p_j * ((z_j - lse) + entropy)), 0 where p_j is 0 and j is not the token, or lse = -infinity.
 * Results are rounded once. Sums are made in the same order in every call.
 *
 * logits, gradLogits : n rows of V elements, strided as rows in cvcuda/LayerNorm.h; F32, F16 or BF16 (NVCVX_DATA_TYPE_BF16), of one type
 *                      and shape. gradLogits may be logits, or must not overlap it.
 * tokens             : S32 or S64, dense, n elements.
 * out, entropy, lse, gradOut, gradEntropy: F32, dense, n elements. Of the forward call's results entropy and lse may be NULL. gradEntropy may be
 *                      NULL, and entropy with it.
 * topValues          : F32, topTokens: S32, dense, [n, K], K 1 to 32 and at most V; NULL together.
 * scale: finite, positive. n below 2^31, V 1 to 2^30. Tensors may be larger than 2^32 bytes.
 * Status: INVALID_ARGUMENT for any type / shape / stride problem. */
#ifndef CVCUDA_LOG_PROBS_H
#define CVCUDA_LOG_PROBS_H

#include "Operator.h"
#include "Types.h"

#include <nvcv/Status.h>
#include <nvcv/Tensor.h>

#ifdef __cplusplus
extern "C"
{
#endif

#define CVCUDAX_LOG_PROBS_MOST_TOP 32

CVCUDA_PUBLIC NVCVStatus cvcudaxLogProbsCreate(NVCVOperatorHandle *handle);

CVCUDA_PUBLIC NVCVStatus cvcudaxLogProbsSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle logits,
                                               NVCVTensorHandle tokens, NVCVTensorHandle out, NVCVTensorHandle entropy,
                                               NVCVTensorHandle lse, NVCVTensorHandle topValues, NVCVTensorHandle topTokens,
                                               float scale);

CVCUDA_PUBLIC NVCVStatus cvcudaxLogProbsGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle logits,
                                                   NVCVTensorHandle tokens, NVCVTensorHandle lse, NVCVTensorHandle entropy,
                                                   NVCVTensorHandle gradOut, NVCVTensorHandle gradEntropy,
                                                   NVCVTensorHandle gradLogits, float scale);

#ifdef __cplusplus
}
#endif

#endif /* CVCUDA_LOG_PROBS_H */
