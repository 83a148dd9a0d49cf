// What attention and its gradient take (cvcuda/Attention.h), and what the host checks of it.
#ifndef CVCUDA_AMD_ATTENTIONOPS_HPP
#define CVCUDA_AMD_ATTENTIONOPS_HPP

#include "HeadOps.hpp"

namespace cvamd {

// Bytes from one token to the next, or of all heads: a tile's addresses are 32-bit numbers.
constexpr int64_t kMostStride = 1 << 24;

struct AttentionSequences
{
    const int32_t *offsets, *keyOffsets, *keyLengths; // the latter two: nullptr as in cvcuda/Attention.h
    int32_t        count, rows, keys;                 // sequences; tokens of q and of k

    __device__ __forceinline__ int firstRow(int b) const
    {
        return min(max(offsets[b], 0), rows);
    }

    __device__ __forceinline__ int rowsOf(int b, int first) const
    {
        return max(min(max(offsets[b + 1], 0), rows) - first, 0);
    }

    __device__ __forceinline__ int firstKey(int b) const
    {
        return min(max((keyOffsets != nullptr ? keyOffsets : offsets)[b], 0), keys);
    }

    __device__ __forceinline__ int keysOf(int b, int first) const
    {
        const int n = max(min(max((keyOffsets != nullptr ? keyOffsets : offsets)[b + 1], 0), keys) - first, 0);
        return keyLengths != nullptr ? min(max(keyLengths[b], 0), n) : n;
    }
};

class AttentionOperator final : public IOperator
{
};

struct AttentionInputs
{
    HeadsView          q, k, v;
    AttentionSequences sequences;
    float             *lse;
};

// Shared by the forward call and the gradient. Throws INVALID_ARGUMENT.
AttentionInputs TakeAttention(NVCVTensorHandle q, NVCVTensorHandle k, NVCVTensorHandle v, NVCVTensorHandle offsets, NVCVTensorHandle keyOffsets,
                              NVCVTensorHandle keyLengths, NVCVTensorHandle lse, bool lseOptional, float scale);

// A tensor like `as`, aligned as attention's tensors are.
HeadsView TakeHeadsLike(NVCVTensorHandle h, const HeadsView &as, const char *what);

void RequireAttentionSizes(int64_t rows, int64_t keys, int64_t sequences, int64_t heads, int64_t keyHeads, int64_t dims);

} // namespace cvamd

#endif // CVCUDA_AMD_ATTENTIONOPS_HPP
