// What the operators on tensors of tokens, heads and a head's elements share (rotary positions, attention).
#ifndef CVCUDA_AMD_HEADOPS_HPP
#define CVCUDA_AMD_HEADOPS_HPP

#include "RowOps.hpp"

namespace cvamd {

// [T, H, D]: the row of a token's head begins at base + token * tokenStride + head * headStride bytes. A token lies behind all heads of the one before,
// as the library's tensors have no smaller pitch than what lies within it (nvcvTensorWrapDataConstruct).
struct HeadsView
{
    uint8_t *base;
    int64_t  tokenStride, headStride;
    int32_t  tokens, heads, dims;
    RowElem  elem;
};

// Throws INVALID_ARGUMENT where a tensor isn't one of that kind; `align`: bytes that its address and distances must be multiples of (0: an element).
HeadsView RequireHeads(NVCVTensorHandle h, const char *what, int align);

// Throws INVALID_ARGUMENT unless `b` has a's type and shape.
void RequireSameHeads(const HeadsView &a, const HeadsView &b, const char *what);

} // namespace cvamd

#endif // CVCUDA_AMD_HEADOPS_HPP
