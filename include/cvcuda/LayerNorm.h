/* Layer norm of rows, and its gradient. Extension (no counterpart in the reference).
 *
 * A row is the last dimension of a tensor of any rank; its elements follow one another, the dimensions before it may be
 * strided as long as at most two of them cannot be merged into one. With D elements in a row, all in float32:
 *     mean = sum(x) / D,  rstd = 1 / sqrt(sum((x - mean)^2) / D + epsilon),  out = (x - mean) * rstd * gamma + beta.
 * Gradient, with h = (x - mean) * rstd and w = gradOut * gamma:
 *     gradIn = rstd * (w - sum(w) / D - h * sum(w * h) / D),
 *     gradGamma = sum over rows of gradOut * h,  gradBeta = sum over rows of gradOut.
 * Results are rounded once, to the nearest even. The sums over rows are made in the same order in every call.
 *
 * in, out, gradOut, gradIn: F32, F16 or BF16 (NVCVX_DATA_TYPE_BF16), one type for all, of one shape. out may be in and
 *                           gradIn may be gradOut or in.
 * gamma, beta             : [D] (or any shape of D elements), both F32 or both of in's type; NULL stands for 1 and 0.
 * gradGamma, gradBeta     : [D], both F32 or both of in's type; either may be NULL.
 * mean, rstd              : F32, one element per row, dense; outputs of the forward call (either may be NULL there), inputs
 *                           of the gradient.
 * workspace               : U8, dense, at least as many elements as cvcudaxLayerNormGradWorkspace gives, aligned to 16 bytes. It
 *                           belongs to the call until the stream has passed it; NULL where 0 bytes are needed, or without gradGamma and
 *                           gradBeta. Of CVCUDAX_LAYER_NORM_UNTOUCHED_WORKSPACE bytes (gradients of few rows, made in one launch) it has to be
 *                           given, but is not touched: calls on any streams may share one.
 * Rows: below 2^31, row elements: 2^30 at most. Tensors may be larger than 2^32 bytes. Tensors without elements are allowed: sums
 * over no rows are 0.
 * Status: INVALID_ARGUMENT for any type / shape / stride problem. */
#ifndef CVCUDA_LAYER_NORM_H
#define CVCUDA_LAYER_NORM_H

#include "Operator.h"
#include "Types.h"

#include <nvcv/Status.h>
#include <nvcv/Tensor.h>

#ifdef __cplusplus
extern "C"
{
#endif

#define CVCUDAX_LAYER_NORM_UNTOUCHED_WORKSPACE 16

CVCUDA_PUBLIC NVCVStatus cvcudaxLayerNormCreate(NVCVOperatorHandle *handle);

CVCUDA_PUBLIC NVCVStatus cvcudaxLayerNormSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle in,
                                                NVCVTensorHandle gamma, NVCVTensorHandle beta, NVCVTensorHandle out,
                                                NVCVTensorHandle mean, NVCVTensorHandle rstd, float epsilon);

CVCUDA_PUBLIC NVCVStatus cvcudaxLayerNormGradWorkspace(int64_t rows, int64_t columns, int64_t *bytes);

CVCUDA_PUBLIC NVCVStatus cvcudaxLayerNormGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle gradOut,
                                                    NVCVTensorHandle in, NVCVTensorHandle gamma, NVCVTensorHandle mean,
                                                    NVCVTensorHandle rstd, NVCVTensorHandle gradIn,
                                                    NVCVTensorHandle gradGamma, NVCVTensorHandle gradBeta,
                                                    NVCVTensorHandle workspace);

#ifdef __cplusplus
}
#endif

#endif /* CVCUDA_LAYER_NORM_H */
