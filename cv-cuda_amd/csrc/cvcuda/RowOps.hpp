// What the operators on rows of floating-point values share (layer norm, embedding, AdamW): element types and their
// conversions, runs of 16 bytes per lane, sums over a wave and the rows of a strided tensor.
#ifndef CVCUDA_AMD_ROWOPS_HPP
#define CVCUDA_AMD_ROWOPS_HPP

#include "DeviceUtils.hpp"
#include "OpCommon.hpp"

#include <nvcv/DataType.h>

namespace cvamd {

using Half = _Float16;
using Bf16 = __bf16;

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

// Runs of 16 bytes that a kernel reads or writes once. PAST: with the hint that the caches need not keep them, for calls that move more
// than half of what the memory-side cache holds (256 MB). Their inputs and outputs are gone from there before they are wanted again, and what is
// kept of them costs places: the gradient of 512 MB of logits 174 us, 164 with the hint; in buffers that take turns 128 MB of logits 45 and
// 42, 64 MB 24 and 22. Smaller calls find their inputs there, and their outputs are found: 16 MB 6.8 us, with the hint 7.4.
inline bool MovesPastCaches(int64_t bytes)
{
    return bytes > 128 << 20;
}

using Unit16 = uint32_t __attribute__((ext_vector_type(4)));

template<bool PAST, class T, int N>
__device__ __forceinline__ Run<T, N> LoadRun(const T *from)
{
    if constexpr (PAST && sizeof(Run<T, N>) == sizeof(Unit16))
    {
        using Unit = Unit16 __attribute__((aligned(sizeof(T))));
        return __builtin_bit_cast(Run<T, N>, __builtin_nontemporal_load(reinterpret_cast<const Unit *>(from)));
    }
    else
    {
        return *reinterpret_cast<const Run<T, N> *>(from);
    }
}

template<bool PAST, class T, int N>
__device__ __forceinline__ void StoreRun(T *to, const Run<T, N> &run)
{
    if constexpr (PAST && sizeof(Run<T, N>) == sizeof(Unit16))
    {
        using Unit = Unit16 __attribute__((aligned(sizeof(T))));
        __builtin_nontemporal_store(__builtin_bit_cast(Unit16, run), reinterpret_cast<Unit *>(to));
    }
    else
    {
        *reinterpret_cast<Run<T, N> *>(to) = run;
    }
}

// Elements of T in 16 bytes.
template<class T>
constexpr int kRunOf = 16 / (int)sizeof(T);

template<class T>
__device__ __forceinline__ T FromFloat(float v)
{
    return (T)v; // to the nearest even
}

// What lane `of the step` has, 0 where there is none: the steps of a reduction over the wave by cross-lane moves alone (within
// rows of 16 lanes, then from each row's last lane to the next row). After the last one lane 63 has it all.
template<int STEP>
__device__ __forceinline__ uint32_t LaneStep(uint32_t v)
{
    constexpr int ctrl[] = {0x111, 0x112, 0x114, 0x118, 0x142, 0x143}; // row_shr 1, 2, 4, 8, row_bcast 15, 31
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl[STEP], STEP == 4 ? 0xA : STEP == 5 ? 0xC : 0xF, 0xF, false);
}

// Sum over the 64 lanes, as one number.
__device__ __forceinline__ float WaveSum(float v)
{
    v += __uint_as_float(LaneStep<0>(__float_as_uint(v)));
    v += __uint_as_float(LaneStep<1>(__float_as_uint(v)));
    v += __uint_as_float(LaneStep<2>(__float_as_uint(v)));
    v += __uint_as_float(LaneStep<3>(__float_as_uint(v)));
    v += __uint_as_float(LaneStep<4>(__float_as_uint(v)));
    v += __uint_as_float(LaneStep<5>(__float_as_uint(v)));
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

// The largest of the 64 lanes' numbers, as one. Of magnitudes by their bits: a NaN is larger than all others.
__device__ __forceinline__ uint32_t WaveLargest(uint32_t v)
{
    v = max(v, LaneStep<0>(v));
    v = max(v, LaneStep<1>(v));
    v = max(v, LaneStep<2>(v));
    v = max(v, LaneStep<3>(v));
    v = max(v, LaneStep<4>(v));
    v = max(v, LaneStep<5>(v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The wave's number in its workgroup, as what it is to the compiler: the same in all lanes.
__device__ __forceinline__ uint32_t WaveOfGroup()
{
    return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
