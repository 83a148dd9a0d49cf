/* One step of AdamW over many tensors at once. Extension (no counterpart in the reference).
 *
 * For each element of each tensor, in float32, every operation rounded by itself and in this order; the coefficients in
 * brackets are computed in 64 bits and rounded to float32, t being `step`:
 *     g = gradScale * grad
 *     m = [beta1] * m + g * [1 - beta1]
 *     v = [beta2] * v + (g * [1 - beta2]) * g
 *     p = p * [1 - lr * weightDecay] - (m / (sqrt(v) * [1 / sqrt(1 - beta2^t)] + [epsilon])) * [lr / (1 - beta1^t)]
 *
 * params    : F32, F16 or BF16 (NVCVX_DATA_TYPE_BF16); updated, rounded once.
 * grads     : F32, F16 or BF16.
 * copies    : NULL, or for each tensor NULL or one of F16 or BF16 that receives the new params, rounded once from float32.
 * moments, variances: m and v, updated. F32, or in 8 bits: moments S8 and variances U8, for which momentScales and
 *             varianceScales hold an F32 for each block of 256 elements, in the tensor's order. With a the block's scale, the
 *             largest magnitude of its values, codes stand for
 *                 m = (t * |t|) * a, t = q * [1 / 127]         v = ((t * t) * (t * t)) * a, t = q * [1 / 255]
 *             and are the nearest: q = rint(sqrt(|m| / a) * 127) with m's sign, q = rint(sqrt(sqrt(v / a)) * 255), but 1 at
 *             least where v > 0, so that no step is divided by epsilon alone; 0 where a is 0. The step itself uses the values
 *             of m and v before they become codes. A block in which a value is not finite has NaN as its scale, and
 *             stands for NaN from then on.
 * gradScale : NULL (1), or an F32 tensor of one element, read on the device: the factor of a clipped or scaled gradient.
 * All tensors of one index have the same number of elements and are dense; their shapes do not matter. Types may differ from
 * index to index. Tensors without elements are allowed; no tensor may overlap another.
 * cvcudaxAdamWUnpackSubmit gives the values that 8-bit states stand for, as F32: moments for S8, variances for U8.
 * Status: INVALID_ARGUMENT for any type / shape / stride problem, before any tensor is changed. */
#ifndef CVCUDA_ADAMW_H
#define CVCUDA_ADAMW_H

#include "Operator.h"
#include "Types.h"

#include <nvcv/Status.h>
#include <nvcv/Tensor.h>

#ifdef __cplusplus
extern "C"
{
#endif

#define CVCUDAX_ADAMW_BLOCK 256

typedef struct CVCUDAXAdamWRec
{
    double  lr;
    double  beta1, beta2; /* in [0, 1) */
    double  epsilon;
    double  weightDecay;
    int64_t step; /* 1 for the first */
} CVCUDAXAdamW;

CVCUDA_PUBLIC NVCVStatus cvcudaxAdamWCreate(NVCVOperatorHandle *handle);

CVCUDA_PUBLIC NVCVStatus cvcudaxAdamWSubmit(NVCVOperatorHandle handle, hipStream_t stream, int32_t count,
                                            const NVCVTensorHandle *params, const NVCVTensorHandle *moments,
                                            const NVCVTensorHandle *variances, const NVCVTensorHandle *grads,
                                            const NVCVTensorHandle *copies, const NVCVTensorHandle *momentScales,
                                            const NVCVTensorHandle *varianceScales, NVCVTensorHandle gradScale,
                                            const CVCUDAXAdamW *args);

CVCUDA_PUBLIC NVCVStatus cvcudaxAdamWUnpackSubmit(NVCVOperatorHandle handle, hipStream_t stream, int32_t count,
                                                  const NVCVTensorHandle *codes, const NVCVTensorHandle *scales,
                                                  const NVCVTensorHandle *out);

#ifdef __cplusplus
}
#endif

#endif /* CVCUDA_ADAMW_H */
