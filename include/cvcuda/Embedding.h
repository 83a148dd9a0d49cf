/* Lookup of rows of a table by token, with scaling, and the table's gradient. Extension (no counterpart in the reference).
 *
 *     out[i] = scale * table[tokens[i]], in float32, rounded once; zeros where tokens[i] is outside [0, V).
 * Gradient: gradTable[v] = scale * (sum of gradOut[i] over the i with tokens[i] == v, in float32); with `accumulate` it is
 * added to what gradTable holds, in float32 and rounded once, and rows of tokens that do not occur are left as they are,
 * without it they are set to zero. Tokens outside [0, V) and tokens equal to `padding` have no part in it. The tokens are
 * sorted, each row is summed in an order that depends on them alone: the same call gives the same bits.
 *
 * table, gradTable: [V, D], rows of elements that follow one another; F32, F16 or BF16 (NVCVX_DATA_TYPE_BF16).
 * tokens          : S32 or S64, dense, any shape of n elements.
 * out, gradOut    : n rows of D elements, strided as rows in cvcuda/LayerNorm.h.
 * out has the table's type, or F16 or BF16 beside a table of F32. gradTable has gradOut's type, or F32.
 * padding         : a token, or -1 for none.
 * workspace       : U8, dense, at least as many elements as cvcudaxEmbeddingGradWorkspace gives, aligned to 16 bytes. It
 *                   belongs to the call until the stream has passed it; NULL where 0 bytes are needed.
 * n, V: below 2^31 each, D: 2^30 at most. Tensors may be larger than 2^32 bytes.
 * Status: INVALID_ARGUMENT for any type / shape / stride problem. */
#ifndef CVCUDA_EMBEDDING_H
#define CVCUDA_EMBEDDING_H

#include "Operator.h"
#include "Types.h"

#include <nvcv/Status.h>
#include <nvcv/Tensor.h>

#ifdef __cplusplus
extern "C"
{
#endif

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingCreate(NVCVOperatorHandle *handle);

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle table,
                                                NVCVTensorHandle tokens, NVCVTensorHandle out, float scale);

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingGradWorkspace(int64_t tokens, int64_t vocabulary, int64_t columns, int64_t *bytes);

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle gradOut,
                                                    NVCVTensorHandle tokens, NVCVTensorHandle gradTable,
                                                    NVCVTensorHandle workspace, float scale, int64_t padding,
                                                    int8_t accumulate);

#ifdef __cplusplus
}
#endif

#endif /* CVCUDA_EMBEDDING_H */
