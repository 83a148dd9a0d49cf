#include "RowOps.hpp"

namespace cvamd {

namespace {

void RequireAligned(const void *p, int bytes, const char *what)
{
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must be aligned to its elements of %d bytes", what, bytes);
    }
}

int64_t CountOf(const NVCVTensorData &d, const char *what)
{
    // (extents of 0 first: the others' product may be anything)
    for (int i = 0; i < d.rank; ++i)
    {
        if (d.shape[i] == 0)
        {
            return 0;
        }
    }
    int64_t n = 1;
    for (int i = 0; i < d.rank; ++i)
    {
        if (__builtin_mul_overflow(n, d.shape[i], &n))
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s has too many elements", what);
        }
    }
    return n;
}

} // namespace

RowsView RequireRows(NVCVTensorHandle h, const char *what)
{
    NVCVTensorData d;
    ExportTensor(h, d, what);
    RowsView v = {};
    v.base     = d.buffer.strided.basePtr;
    v.elem     = RowElemOf(d.dtype);
    if (v.elem == kRowNone)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must hold F32, F16 or BF16 values", what);
    }
    const int      es = RowElemSize(v.elem);
    const int64_t *st = d.buffer.strided.strides;
    RequireAligned(v.base, es, what);
    const int64_t columns = d.shape[d.rank - 1];
    if (columns > 1 && st[d.rank - 1] != es)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have rows of elements that follow one another", what);
    }
    if (columns > kMostColumns)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s has rows of too many elements", what);
    }
    // the dimensions before the last, from the inside out, merged where one continues the other
    int64_t extent[2] = {1, 1}, stride[2] = {columns * es, 0}, rows = 1;
    int     levels = 0;
    for (int i = 0; i < d.rank - 1; ++i)
    {
        rows = d.shape[i] == 0 ? 0 : rows;
    }
    for (int i = d.rank - 2; i >= 0 && rows > 0; --i)
    {
        if (d.shape[i] == 1)
        {
            continue;
        }
        if (st[i] % es != 0)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have strides of whole elements", what);
        }
        if (levels > 0 && st[i] == stride[levels - 1] * extent[levels - 1])
        {
            extent[levels - 1] *= d.shape[i];
        }
        else if (levels < 2)
        {
            extent[levels] = d.shape[i];
            stride[levels] = st[i];
            ++levels;
        }
        else
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s has rows at distances of more than two kinds", what);
        }
        if (__builtin_mul_overflow(rows, d.shape[i], &rows) || rows > INT32_MAX)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s has too many rows", what);
        }
    }
    v.rows        = (int32_t)rows;
    v.columns     = (int32_t)columns;
    v.inner       = (int32_t)extent[0];
    v.innerStride = stride[0];
    v.outerStride = levels == 2 ? stride[1] : 0;
    return v;
}

DenseView RequireDense(NVCVTensorHandle h, const char *what, NVCVDataType dt)
{
    NVCVTensorData d;
    ExportTensor(h, d, what);
    if (dt != NVCV_DATA_TYPE_NONE && d.dtype != dt)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must hold values of type %s", what, nvcvDataTypeGetName(dt));
    }
    int32_t es = RowElemOf(d.dtype) != kRowNone ? RowElemSize(RowElemOf(d.dtype)) : 0; // (the others' sizes are looked up)
    if (es == 0)
    {
        CheckCore(nvcvDataTypeGetStrideBytes(d.dtype, &es));
    }
    DenseView v = {d.buffer.strided.basePtr, CountOf(d, what), d.dtype};
    int64_t   want = es;
    for (int i = d.rank - 1; i >= 0 && v.count > 0; --i)
    {
        if (d.shape[i] > 1 && d.buffer.strided.strides[i] != want)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must be dense", what);
        }
        want *= d.shape[i];
    }
    RequireAligned(v.base, es, what);
    return v;
}

uint8_t *RequireWorkspace(NVCVTensorHandle h, int64_t bytes)
{
    if (bytes == 0)
    {
        return nullptr;
    }
    const DenseView v = RequireDense(h, "Workspace", NVCV_DATA_TYPE_U8);
    if (v.count < bytes)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Workspace must hold %ld bytes at least, not %ld", (long)bytes, (long)v.count);
    }
    RequireAligned(v.base, 16, "Workspace");
    return v.base;
}

} // namespace cvamd
