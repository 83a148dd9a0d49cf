#include "HeadOps.hpp"

namespace cvamd {

HeadsView RequireHeads(NVCVTensorHandle h, const char *what, int align)
{
    NVCVTensorData d;
    ExportTensor(h, d, what);
    HeadsView v = {};
    v.elem      = RowElemOf(d.dtype);
    if (v.elem == kRowNone)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must hold F32, F16 or BF16 values", what);
    }
    if (d.rank != 3)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have 3 dimensions (tokens, heads, elements), not %d", what, d.rank);
    }
    const int64_t es = RowElemSize(v.elem), whole = align > es ? align : es;
    const auto   &st = d.buffer.strided.strides;
    v.base           = d.buffer.strided.basePtr;
    if (reinterpret_cast<uintptr_t>(v.base) % whole != 0)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must be aligned to %ld bytes", what, (long)whole);
    }
    if (d.shape[2] > 1 && st[2] != es)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have rows of elements that follow one another", what);
    }
    if (d.shape[2] > (1 << 20) || d.shape[0] > INT32_MAX || d.shape[1] > INT32_MAX || (d.shape[0] > 0 && d.shape[1] > INT32_MAX / d.shape[0]))
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s has too many elements in a row, or rows", what);
    }
    v.tokens = (int32_t)d.shape[0];
    v.heads  = (int32_t)d.shape[1];
    v.dims   = (int32_t)d.shape[2];
    // (distances between one and the same are never gone; a token behind the only one is still another place)
    v.headStride  = v.heads > 1 ? st[1] : 0;
    v.tokenStride = v.tokens > 1 ? st[0] : v.heads > 1 ? v.headStride * v.heads : v.dims * es;
    if (v.tokenStride % whole != 0 || v.headStride % whole != 0)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have tokens and heads at distances of whole %ld bytes", what, (long)whole);
    }
    return v;
}

void RequireSameHeads(const HeadsView &a, const HeadsView &b, const char *what)
{
    if (a.elem != b.elem || a.tokens != b.tokens || a.heads != b.heads || a.dims != b.dims)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have the same type and shape as what it belongs to", what);
    }
}

} // namespace cvamd
