// Lookup of rows of a table by token, and the table's gradient (formulas: cvcuda/Embedding.h).
#include "RowOps.hpp"

#include <cvcuda/Embedding.h>

#include <algorithm>
#include <cmath>

namespace cvamd {

namespace {

struct LookupArgs
{
    RowPlaces   table, out;
    const void *tokens;
    int32_t     wide; // tokens of 64 bits
    int32_t     count, vocabulary, columns;
    float       scale;
};

struct GradArgs
{
    RowPlaces   grad, table;
    const void *tokens;
    int32_t     wide, accumulate;
    int32_t     count, vocabulary, columns;
    int64_t     padding;
    float       scale;
};

__device__ __forceinline__ int64_t TokenAt(const void *tokens, int wide, int64_t i)
{
    return wide ? static_cast<const int64_t *>(tokens)[i] : static_cast<const int32_t *>(tokens)[i];
}

// A workgroup per token.
template<class T, class O>
__global__ __launch_bounds__(256) void EmbeddingKernel(const LookupArgs a)
{
    for (uint32_t i = blockIdx.x; i < (uint32_t)a.count; i += gridDim.x)
    {
        const int64_t t = TokenAt(a.tokens, a.wide, i);
        O            *y = reinterpret_cast<O *>(a.out.at(i));
        const bool    known = t >= 0 && t < a.vocabulary;
        const T      *row   = reinterpret_cast<const T *>(a.table.at(known ? (uint32_t)t : 0));
        for (int c = threadIdx.x; c < a.columns; c += 256)
        {
            y[c] = FromFloat<O>(known ? (float)row[c] * a.scale : 0.f);
        }
    }
}

// A workgroup per row of the table and 256 columns looks through all tokens and adds the rows of its own in their order.
template<class T, class O>
__global__ __launch_bounds__(256) void EmbeddingGradKernel(const GradArgs a)
{
    __shared__ uint64_t found[4];
    const uint32_t      tiles = (a.columns + 255) / 256;
    for (uint64_t k = blockIdx.x; k < (uint64_t)a.vocabulary * tiles; k += gridDim.x)
    {
        const int64_t       v = k / tiles;
        const int           c = (int)(k % tiles) * 256 + threadIdx.x;
        float               s = 0;
        bool                any = false;
        for (int first = 0; first < a.count && v != a.padding; first += 256)
        {
            const int      i    = first + threadIdx.x;
            const uint64_t mine = __ballot(i < a.count && TokenAt(a.tokens, a.wide, i) == v);
            __syncthreads();
            if ((threadIdx.x & 63) == 0)
            {
                found[threadIdx.x >> 6] = mine;
            }
            __syncthreads();
            for (int w = 0; w < 4; ++w)
            {
                for (uint64_t f = found[w]; f != 0; f &= f - 1)
                {
                    any = true;
                    s += c < a.columns ? (float)reinterpret_cast<const T *>(a.grad.at(first + 64 * w + __ffsll((unsigned long long)f) - 1))[c] : 0.f;
                }
            }
        }
        O *out = reinterpret_cast<O *>(a.table.at((uint32_t)v));
        if (c < a.columns && (any || !a.accumulate))
        {
            out[c] = FromFloat<O>(a.accumulate ? (float)out[c] + s * a.scale : s * a.scale);
        }
    }
}

// Workgroups of a launch: a dimension of the grid holds fewer than 2^32 threads.
constexpr int kMostGroups = 1 << 20;

// ---- host ----------------------------------------------------------------------------------------------------------
int64_t GradWorkspace(int64_t, int64_t, int64_t)
{
    return 0;
}

template<class T, class O>
void LaunchLookup(const LookupArgs &a, hipStream_t stream)
{
    hipLaunchKernelGGL((EmbeddingKernel<T, O>), dim3(std::min(a.count, kMostGroups)), dim3(256), 0, stream, a);
    CheckLaunch("EmbeddingKernel");
}

template<class T, class O>
void LaunchGrad(const GradArgs &a, hipStream_t stream)
{
    hipLaunchKernelGGL((EmbeddingGradKernel<T, O>), dim3((int)std::min<int64_t>((int64_t)a.vocabulary * DivUp(a.columns, 256), kMostGroups)), dim3(256), 0, stream, a);
    CheckLaunch("EmbeddingGradKernel");
}

struct Tokens
{
    const void *base;
    int32_t     count, wide;
};

Tokens TakeTokens(NVCVTensorHandle h)
{
    const DenseView v = RequireDense(h, "Tokens", NVCV_DATA_TYPE_NONE);
    if (v.dtype != NVCV_DATA_TYPE_S32 && v.dtype != NVCV_DATA_TYPE_S64)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tokens must be S32 or S64");
    }
    if (v.count > INT32_MAX)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Too many tokens");
    }
    return {v.base, (int32_t)v.count, v.dtype == NVCV_DATA_TYPE_S64};
}

void RequireScale(float scale)
{
    if (!std::isfinite(scale))
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Scale must be finite");
    }
}

class Embedding final : public IOperator
{
public:
    void submit(hipStream_t stream, NVCVTensorHandle htable, NVCVTensorHandle htokens, NVCVTensorHandle hout, float scale) const
    {
        const RowsView table = RequireRows(htable, "Table"), out = RequireRows(hout, "Output");
        const Tokens   tokens = TakeTokens(htokens);
        RequireScale(scale);
        if (out.rows != tokens.count || out.columns != table.columns)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Output must have a row per token (%d) with the table's elements (%d), not %d of %d",
                          tokens.count, table.columns, out.rows, out.columns);
        }
        if (out.elem != table.elem && table.elem != kRowF32)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Output must have the table's type, or the table's must be F32");
        }
        if (tokens.count == 0 || table.columns == 0)
        {
            return;
        }
        const LookupArgs a = {RowPlaces(table), RowPlaces(out), tokens.base, tokens.wide, tokens.count, table.rows, table.columns, scale};
        if (table.elem == kRowF16)
        {
            LaunchLookup<Half, Half>(a, stream);
        }
        else if (table.elem == kRowBf16)
        {
            LaunchLookup<Bf16, Bf16>(a, stream);
        }
        else if (out.elem == kRowF32)
        {
            LaunchLookup<float, float>(a, stream);
        }
        else if (out.elem == kRowF16)
        {
            LaunchLookup<float, Half>(a, stream);
        }
        else
        {
            LaunchLookup<float, Bf16>(a, stream);
        }
    }

    static void submitGrad(hipStream_t stream, NVCVTensorHandle hgrad, NVCVTensorHandle htokens, NVCVTensorHandle htable,
                           NVCVTensorHandle hworkspace, float scale, int64_t padding, bool accumulate)
    {
        const RowsView grad = RequireRows(hgrad, "Output's gradient"), table = RequireRows(htable, "Table's gradient");
        const Tokens   tokens = TakeTokens(htokens);
        RequireScale(scale);
        if (grad.rows != tokens.count || grad.columns != table.columns)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Output's gradient must have a row per token (%d) with the table's elements (%d), not %d of %d",
                          tokens.count, table.columns, grad.rows, grad.columns);
        }
        if (table.elem != grad.elem && table.elem != kRowF32)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Table's gradient must have the type of the output's gradient, or F32");
        }
        if (padding < -1)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Padding must be a token, or -1 for none, not %ld", (long)padding);
        }
        (void)RequireWorkspace(hworkspace, GradWorkspace(tokens.count, table.rows, table.columns));
        if (table.rows == 0 || table.columns == 0)
        {
            return;
        }
        const GradArgs a = {RowPlaces(grad), RowPlaces(table), tokens.base, tokens.wide, accumulate, tokens.count, table.rows, table.columns,
                            padding, scale};
        if (grad.elem == kRowF32)
        {
            LaunchGrad<float, float>(a, stream);
        }
        else if (grad.elem == kRowF16)
        {
            table.elem == kRowF32 ? LaunchGrad<Half, float>(a, stream) : LaunchGrad<Half, Half>(a, stream);
        }
        else
        {
            table.elem == kRowF32 ? LaunchGrad<Bf16, float>(a, stream) : LaunchGrad<Bf16, Bf16>(a, stream);
        }
    }
};

} // namespace
} // namespace cvamd

using namespace cvamd;

extern "C"
{
CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingCreate(NVCVOperatorHandle *handle)
{
    return CreateOperator<Embedding>(handle);
}

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle table,
                                                NVCVTensorHandle tokens, NVCVTensorHandle out, float scale)
{
    return Protect([&] { ToOperator<Embedding>(handle).submit(stream, table, tokens, out, scale); });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingGradWorkspace(int64_t tokens, int64_t vocabulary, int64_t columns, int64_t *bytes)
{
    return Protect(
        [&]
        {
            if (bytes == nullptr)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Pointer to output must not be NULL");
            }
            if (tokens < 0 || tokens > INT32_MAX || vocabulary < 0 || vocabulary > INT32_MAX || columns < 0 || columns > INT32_MAX)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tokens, rows of the table and row elements must be in [0, %d], not %ld, %ld and %ld",
                              INT32_MAX, (long)tokens, (long)vocabulary, (long)columns);
            }
            *bytes = GradWorkspace(tokens, vocabulary, columns);
        });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle gradOut,
                                                    NVCVTensorHandle tokens, NVCVTensorHandle gradTable,
                                                    NVCVTensorHandle workspace, float scale, int64_t padding,
                                                    int8_t accumulate)
{
    return Protect(
        [&]
        {
            (void)ToOperator<Embedding>(handle);
            Embedding::submitGrad(stream, gradOut, tokens, gradTable, workspace, scale, padding, accumulate != 0);
        });
}
}
