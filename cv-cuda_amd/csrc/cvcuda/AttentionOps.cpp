#include "AttentionOps.hpp"

#include <algorithm>

namespace cvamd {

namespace {

constexpr int kMostDims = 128, kAlign = 16;

// Numbers of rows and keys, and what is added to them, stay below 2^31, and a launch's threads below 2^32.
constexpr int64_t kMostRows = 1 << 29, kMostSequences = 1 << 21;

const int32_t *TakeNumbers(NVCVTensorHandle h, const char *what, int64_t count)
{
    const DenseView v = RequireDense(h, what, NVCV_DATA_TYPE_S32);
    if (v.count != count)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have %ld elements, not %ld", what, (long)count, (long)v.count);
    }
    return reinterpret_cast<const int32_t *>(v.base);
}

HeadsView TakeHeads(NVCVTensorHandle h, const char *what)
{
    const HeadsView v = RequireHeads(h, what, kAlign);
    if (v.elem == kRowF32)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must hold F16 or BF16 values", what);
    }
    if (v.tokenStride > kMostStride || v.headStride > kMostStride / std::max(v.heads, 1))
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have tokens, and all heads, within %ld bytes of one another", what, (long)kMostStride);
    }
    return v;
}

} // namespace

void RequireAttentionSizes(int64_t rows, int64_t keys, int64_t sequences, int64_t heads, int64_t keyHeads, int64_t dims)
{
    if (rows < 0 || keys < 0 || sequences < 0 || heads < 1 || keyHeads < 1 || heads % keyHeads != 0)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT,
                      "Rows, keys and sequences must not be negative, heads a multiple of the key heads, not %ld, %ld, %ld, %ld and %ld", (long)rows,
                      (long)keys, (long)sequences, (long)heads, (long)keyHeads);
    }
    if (rows > (kMostRows - 1) / heads || keys > (kMostRows - 1) / keyHeads || sequences > (kMostSequences - 1) / keyHeads)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Too many rows, keys or sequences");
    }
    if (dims < 8 || dims > kMostDims || dims % 8 != 0)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "A head must have a multiple of 8 elements, at most %d, not %ld", kMostDims, (long)dims);
    }
}

HeadsView TakeHeadsLike(NVCVTensorHandle h, const HeadsView &as, const char *what)
{
    const HeadsView v = TakeHeads(h, what);
    RequireSameHeads(as, v, what);
    return v;
}

AttentionInputs TakeAttention(NVCVTensorHandle hq, NVCVTensorHandle hk, NVCVTensorHandle hv, NVCVTensorHandle hoffsets,
                              NVCVTensorHandle hkeyOffsets, NVCVTensorHandle hkeyLengths, NVCVTensorHandle hlse, bool lseOptional, float scale)
{
    AttentionInputs in = {TakeHeads(hq, "Queries"), TakeHeads(hk, "Keys"), TakeHeads(hv, "Values"), {}, nullptr};
    RequireSameHeads(in.k, in.v, "Values");
    if (in.q.elem != in.k.elem || in.q.dims != in.k.dims)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Queries and keys must have one type and as many elements in a head");
    }
    const DenseView offsets = RequireDense(hoffsets, "Offsets", NVCV_DATA_TYPE_S32);
    if (offsets.count < 1)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Offsets must have one element more than there are sequences");
    }
    RequireAttentionSizes(in.q.tokens, in.k.tokens, offsets.count - 1, in.q.heads, in.k.heads, in.q.dims);
    in.sequences = {reinterpret_cast<const int32_t *>(offsets.base), nullptr, nullptr, (int32_t)(offsets.count - 1), in.q.tokens, in.k.tokens};
    if (hkeyOffsets != nullptr)
    {
        in.sequences.keyOffsets = TakeNumbers(hkeyOffsets, "Key offsets", offsets.count);
    }
    if (hkeyLengths != nullptr)
    {
        if (hkeyOffsets == nullptr)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Key lengths go beside key offsets");
        }
        in.sequences.keyLengths = TakeNumbers(hkeyLengths, "Key lengths", offsets.count - 1);
    }
    if (hlse != nullptr || !lseOptional)
    {
        const DenseView lse = RequireDense(hlse, "Lse", NVCV_DATA_TYPE_F32);
        if (lse.count != (int64_t)in.q.tokens * in.q.heads)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Lse must have one element for each of %d heads and %d rows, not %ld", in.q.heads, in.q.tokens,
                          (long)lse.count);
        }
        in.lse = reinterpret_cast<float *>(lse.base);
    }
    if (!(scale > 0) || !(scale <= 1e30f))
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Scale must be positive, at most 1e30, not %g", (double)scale);
    }
    return in;
}

} // namespace cvamd
