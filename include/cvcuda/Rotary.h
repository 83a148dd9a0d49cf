/* Rotary positions of queries and keys. Extension (no counterpart in the reference).
 *
 * Each row of a head is turned, in pairs of its first `dims` elements, by angles that grow with its token's position. Pair i has
 * the frequency
 *     f = base^(-2 i / dims), with `original` > 0 changed to f * (g + (1 - g) / factor), where
 *         g = clamp((original * f / (2 pi) - low) / (high - low), 0, 1):
 *         pairs that turn at least `high` times over `original` positions keep their frequency, those of at most `low` turns
 *         have it divided by `factor`; with `original` = 0 it is f / factor for all,
 * and with c = magnitude * cos(position * f), s = magnitude * sin(position * f):
 *     out[a] = in[a] * c - in[b] * s,  out[b] = in[a] * s + in[b] * c,
 * a and b being elements 2 i and 2 i + 1 (`interleaved`) or i and i + dims / 2. Elements from `dims` on are copied. `inverse` takes -s
 * for s: the gradient of in from that of out.
 *
 * An angle's whole turns are taken off in 64-bit arithmetic before the sine and cosine, which have errors of some 2^-24, and of up to
 * position * 2^-52 for the 64 bits of a frequency (2^-24 at 2^28, 2^-21 at 2^31); results are computed in float32 and rounded once.
 *
 * in, out   : [T, H, D], F32, F16 or BF16 (NVCVX_DATA_TYPE_BF16), of one type and shape; a row's elements follow one another, tokens
 *             and heads may have gaps, each token lies behind all heads of the one before. out may be in, or must not overlap it.
 * positions : S32 or S64, dense, T elements, any numbers.
 * dims      : even, 2 to 256, at most D. base, factor, magnitude: finite and positive. original >= 0; with it 0 <= low < high.
 * T * H below 2^31, D at most 2^20; tensors may be larger than 2^32 bytes.
 * Status: INVALID_ARGUMENT for any type / shape / stride / parameter problem. */
#ifndef CVCUDA_ROTARY_H
#define CVCUDA_ROTARY_H

#include "Operator.h"
#include "Types.h"

#include <nvcv/Status.h>
#include <nvcv/Tensor.h>

#ifdef __cplusplus
extern "C"
{
#endif

typedef struct CVCUDAXRotaryRec
{
    double  base;
    double  factor, original, low, high; /* 1, 0, 0, 0: frequencies as they are */
    double  magnitude;
    int32_t dims;
    int8_t  interleaved, inverse;
} CVCUDAXRotary;

CVCUDA_PUBLIC NVCVStatus cvcudaxRotaryCreate(NVCVOperatorHandle *handle);

CVCUDA_PUBLIC NVCVStatus cvcudaxRotarySubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle in,
                                             NVCVTensorHandle positions, NVCVTensorHandle out, const CVCUDAXRotary *args);

#ifdef __cplusplus
}
#endif

#endif /* CVCUDA_ROTARY_H */
