/* Attention over packed sequences, with grouped heads, and its gradient. Extension (no counterpart in the reference).
 *
 * Rows offsets[b] to offsets[b + 1] - 1 of q and out are those of sequence b; its keys are the rows from keyOffsets[b] on (NULL: as the
 * queries'): as many as keyLengths[b] says, and at most those before keyOffsets[b + 1] (NULL: those). So keys lie packed, or in
 * places with room, as a cache has them. With Lq rows and Lk keys, row i of a sequence sees keys j < Lk, with `causal` those of
 * j <= i + Lk - Lq: the last row sees all. Query head h reads key head h / (Hq / Hk). Over the keys that a row sees, in float32:
 *     s_j = scale * (q . k_j),  lse = log(sum exp(s_j)),  out = sum exp(s_j - lse) * v_j;
 * a row that sees none, or only scores of -infinity: out = 0, lse = -infinity. Gradient, with p_j = exp(s_j - lse) and d = gradOut . out:
 *     t_j = p_j * (gradOut . v_j - d),
 *     gradQ = scale * sum over j of t_j * k_j,  gradK_j = scale * sum of t_j * q,  gradV_j = sum of p_j * gradOut,
 * the latter two over the rows, and heads of its group, that see key j. p and t take part in the products rounded to the inputs'
 * type (F16: times a power of two, so that small ones are kept); sums and exponentials are 32 bits wide, results are rounded once.
 * Every result is the same in every call.
 *
 * Rows of no sequence, and keys' places that none of them has, are left as they are in out, lse, gradQ, gradK and gradV, and not read
 * elsewhere. Values that are not finite reach the rows that see them, and in the gradient the rows and keys that these are summed over; no
 * others. (Such calls take longer.) Offsets are read on the device: those below 0 or beyond the tensors count as the border, a sequence whose
 * end lies before its begin as empty.
 *
 * q, out, gradOut, gradQ  : [Tq, Hq, D]; k, v, gradK, gradV: [Tk, Hk, D]; F16 or BF16 (NVCVX_DATA_TYPE_BF16), one type for all. Hk
 *                           divides Hq. D: a multiple of 8, at most 128. A row's elements follow one another; heads, and
 *                           tokens, lie at distances of whole 16 bytes, aligned to 16 bytes, each token behind all heads of the one before (such
 *                           as parts of one projection's result), within 2^24 bytes of it.
 *                           Outputs must not overlap inputs nor each other.
 * offsets, keyOffsets     : S32, dense, B + 1 elements each, ascending; keyLengths: S32, B elements, only beside keyOffsets.
 * lse                     : F32, [Hq, Tq], dense. NULL if not wanted; an input of the gradient.
 * workspace               : U8, dense, at least as many elements as cvcudaxAttentionWorkspace or ...GradWorkspace gives (for any lengths of
 *                           the sequences), aligned to 16 bytes. It belongs to the call until the stream has passed it; NULL
 *                           where 0 bytes are needed.
 * scale: positive, at most 1e30. Tq * Hq and Tk * Hk below 2^29, B * Hk below 2^21; tensors may be larger than 2^32 bytes.
 * Status: INVALID_ARGUMENT for any type / shape / stride problem. */
#ifndef CVCUDA_ATTENTION_H
#define CVCUDA_ATTENTION_H

#include "Operator.h"
#include "Types.h"

#include <nvcv/Status.h>
#include <nvcv/Tensor.h>

#ifdef __cplusplus
extern "C"
{
#endif

CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionCreate(NVCVOperatorHandle *handle);

CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionWorkspace(int64_t rows, int64_t keys, int64_t sequences, int32_t heads,
                                                   int32_t keyHeads, int32_t dims, int64_t *bytes);

CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle q,
                                                NVCVTensorHandle k, NVCVTensorHandle v, NVCVTensorHandle offsets,
                                                NVCVTensorHandle keyOffsets, NVCVTensorHandle keyLengths,
                                                NVCVTensorHandle out, NVCVTensorHandle lse, NVCVTensorHandle workspace,
                                                float scale, int8_t causal);

CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionGradWorkspace(int64_t rows, int64_t keys, int64_t sequences, int32_t heads,
                                                       int32_t keyHeads, int32_t dims, int64_t *bytes);

CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle gradOut,
                                                    NVCVTensorHandle q, NVCVTensorHandle k, NVCVTensorHandle v,
                                                    NVCVTensorHandle out, NVCVTensorHandle lse, NVCVTensorHandle offsets,
                                                    NVCVTensorHandle keyOffsets, NVCVTensorHandle keyLengths,
                                                    NVCVTensorHandle gradQ, NVCVTensorHandle gradK, NVCVTensorHandle gradV,
                                                    NVCVTensorHandle workspace, float scale, int8_t causal);

#ifdef __cplusplus
}
#endif

#endif /* CVCUDA_ATTENTION_H */
