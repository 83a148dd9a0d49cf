// What the operators on rows of floating-point values share (layer norm, embedding, AdamW): element types and their
// conversions, runs of 16 bytes per lane, sums over a wave and the rows of a strided tensor.
#ifndef CVCUDA_AMD_ROWOPS_HPP
#define CVCUDA_AMD_ROWOPS_HPP

#include "DeviceUtils.hpp"
#include "OpCommon.hpp"

#include <nvcv/DataType.h>

namespace cvamd {

using Half  = _Float16;
using Bf16  = __bf16;
using Bytes = const uint8_t *;

enum RowElem
{
    kRowF32,
    kRowF16,
    kRowBf16,
    kRowNone
};

inline RowElem RowElemOf(NVCVDataType dt)
{
    return dt == NVCV_DATA_TYPE_F32 ? kRowF32 : dt == NVCV_DATA_TYPE_F16 ? kRowF16 : dt == NVCVX_DATA_TYPE_BF16 ? kRowBf16 : kRowNone;
}

inline int RowElemSize(RowElem e)
{
    return e == kRowF32 ? 4 : 2;
}

// N elements at an address that is aligned to one of them: moved as wide as N allows.
template<class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Run
{
    T v[N];
};

// Elements of T in 16 bytes.
template<class T>
constexpr int kRunOf = 16 / (int)sizeof(T);

template<class T>
__device__ __forceinline__ T FromFloat(float v)
{
    return (T)v; // to the nearest even
}

// Sum over the 64 lanes, in every lane: halves of the wave in turn, so the order is the same in all of them.
__device__ __forceinline__ float WaveSum(float v)
{
#pragma unroll
    for (int s = 32; s > 0; s >>= 1)
    {
        v += __shfl_xor(v, s);
    }
    return v;
}

// Elements of a row: a lane's first column stays a 32-bit number also behind the end of the row.
constexpr int64_t kMostColumns = 1 << 30;

// ---- rows of a tensor --------------------------------------------------------------------------------------------
// Row r begins at base + (r / inner) * outerStride + (r % inner) * innerStride bytes.
struct RowsView
{
    uint8_t *base;
    int64_t  outerStride, innerStride;
    int32_t  rows, columns, inner;
    RowElem  elem;
};

// The same for a kernel.
struct RowPlaces
{
    uint8_t *base;
    int64_t  outerStride, innerStride;
    DivBy    inner;

    explicit RowPlaces(const RowsView &v)
        : base(v.base)
        , outerStride(v.outerStride)
        , innerStride(v.innerStride)
        , inner((uint32_t)(v.inner > 0 ? v.inner : 1))
    {
    }

    __device__ __forceinline__ uint8_t *at(uint32_t row) const
    {
        const uint32_t o = inner.Quotient(row);
        return base + (int64_t)o * outerStride + (int64_t)(row - o * inner.d) * innerStride;
    }
};

// A tensor as rows of its last dimension. Throws INVALID_ARGUMENT where that is not possible.
RowsView RequireRows(NVCVTensorHandle h, const char *what);

// A dense tensor as one run of elements of `dt` (NVCV_DATA_TYPE_NONE: any type).
struct DenseView
{
    uint8_t     *base;
    int64_t      count;
    NVCVDataType dtype;
};

DenseView RequireDense(NVCVTensorHandle h, const char *what, NVCVDataType dt);

// The memory of a workspace of `bytes` (nullptr where none is needed).
uint8_t *RequireWorkspace(NVCVTensorHandle h, int64_t bytes);

} // namespace cvamd

#endif // CVCUDA_AMD_ROWOPS_HPP
