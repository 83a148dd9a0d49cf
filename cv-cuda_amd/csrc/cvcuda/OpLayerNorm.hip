// Layer norm of rows, and its gradient (formulas: cvcuda/LayerNorm.h).
//
// One workgroup per row: the mean, then the squares of what remains of each element without it (a sum of squares from
// which the squared mean is taken would lose the variance of rows that lie far from 0), then the row itself. The gradient's
// sums over rows are made by columns, in two steps whose order is fixed.
#include "RowOps.hpp"

#include <cvcuda/LayerNorm.h>

#include <algorithm>
#include <cmath>

namespace cvamd {

namespace {

struct NormArgs
{
    RowPlaces   in, out;
    const void *gamma, *beta; // nullptr: 1 and 0
    float      *mean, *rstd;  // nullptr: not wanted
    float       epsilon;
    int32_t     rows, columns;
};

struct GradArgs
{
    RowPlaces    grad, in, out;
    const void  *gamma;
    const float *mean, *rstd;
    float       *partial; // [parts][2][columns]
    void        *gradGamma, *gradBeta;
    int32_t      rows, columns, parts;
};

// Sum over a workgroup of 256, in every thread.
__device__ __forceinline__ float BlockSum(float v)
{
    __shared__ float part[4];
    v = WaveSum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
    {
        part[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

template<class T, class W>
__global__ __launch_bounds__(256) void LayerNormKernel(const NormArgs a)
{
    for (uint32_t r = blockIdx.x; r < (uint32_t)a.rows; r += gridDim.x)
    {
        const T  *x = reinterpret_cast<const T *>(a.in.at(r));
        T        *y = reinterpret_cast<T *>(a.out.at(r));
        const int D = a.columns;
        float     s = 0;
        for (int c = threadIdx.x; c < D; c += 256)
        {
            s += (float)x[c];
        }
        const float mean = BlockSum(s) / (float)D;
        s                = 0;
        for (int c = threadIdx.x; c < D; c += 256)
        {
            const float d = (float)x[c] - mean;
            s += d * d;
        }
        const float rstd = 1.f / sqrtf(BlockSum(s) / (float)D + a.epsilon);
        for (int c = threadIdx.x; c < D; c += 256)
        {
            const float g = a.gamma != nullptr ? (float)static_cast<const W *>(a.gamma)[c] : 1.f;
            const float b = a.beta != nullptr ? (float)static_cast<const W *>(a.beta)[c] : 0.f;
            y[c]          = FromFloat<T>(((float)x[c] - mean) * rstd * g + b);
        }
        if (threadIdx.x == 0 && a.mean != nullptr)
        {
            a.mean[r] = mean;
        }
        if (threadIdx.x == 0 && a.rstd != nullptr)
        {
            a.rstd[r] = rstd;
        }
    }
}

template<class T, class W>
__global__ __launch_bounds__(256) void LayerNormGradKernel(const GradArgs a)
{
    for (uint32_t r = blockIdx.x; r < (uint32_t)a.rows; r += gridDim.x)
    {
        const T    *dy = reinterpret_cast<const T *>(a.grad.at(r)), *x = reinterpret_cast<const T *>(a.in.at(r));
        T          *dx   = reinterpret_cast<T *>(a.out.at(r));
        const float mean = a.mean[r], rstd = a.rstd[r];
        const int   D = a.columns;
        float       s = 0, sh = 0;
        for (int c = threadIdx.x; c < D; c += 256)
        {
            const float w = (float)dy[c] * (a.gamma != nullptr ? (float)static_cast<const W *>(a.gamma)[c] : 1.f);
            s += w;
            sh += w * (((float)x[c] - mean) * rstd);
        }
        s  = BlockSum(s) / (float)D;
        sh = BlockSum(sh) / (float)D;
        for (int c = threadIdx.x; c < D; c += 256)
        {
            const float w = (float)dy[c] * (a.gamma != nullptr ? (float)static_cast<const W *>(a.gamma)[c] : 1.f);
            const float h = ((float)x[c] - mean) * rstd;
            dx[c]         = FromFloat<T>(rstd * (w - s - h * sh));
        }
    }
}

// A thread per column and part of the rows.
template<class T>
__global__ __launch_bounds__(256) void LayerNormPartsKernel(const GradArgs a)
{
    const int c = blockIdx.x * 256 + threadIdx.x, D = a.columns;
    if (c >= D)
    {
        return;
    }
    float g = 0, b = 0;
    for (uint32_t r = blockIdx.y; r < (uint32_t)a.rows; r += a.parts)
    {
        const float dy = (float)reinterpret_cast<const T *>(a.grad.at(r))[c];
        g += dy * (((float)reinterpret_cast<const T *>(a.in.at(r))[c] - a.mean[r]) * a.rstd[r]);
        b += dy;
    }
    a.partial[(size_t)blockIdx.y * 2 * D + c]     = g;
    a.partial[(size_t)blockIdx.y * 2 * D + D + c] = b;
}

template<class W>
__global__ __launch_bounds__(256) void LayerNormJoinKernel(const GradArgs a)
{
    const int c = blockIdx.x * 256 + threadIdx.x, D = a.columns;
    if (c >= D)
    {
        return;
    }
    float g = 0, b = 0;
    for (int p = 0; p < a.parts; ++p)
    {
        g += a.partial[(size_t)p * 2 * D + c];
        b += a.partial[(size_t)p * 2 * D + D + c];
    }
    if (a.gradGamma != nullptr)
    {
        static_cast<W *>(a.gradGamma)[c] = FromFloat<W>(g);
    }
    if (a.gradBeta != nullptr)
    {
        static_cast<W *>(a.gradBeta)[c] = FromFloat<W>(b);
    }
}

// Workgroups of a launch: a dimension of the grid holds fewer than 2^32 threads.
constexpr int kMostGroups = 1 << 20;

// ---- host ----------------------------------------------------------------------------------------------------------
int Parts(int64_t rows)
{
    return (int)std::min<int64_t>(rows, 256);
}

int64_t GradWorkspace(int64_t rows, int64_t columns)
{
    return (int64_t)Parts(rows) * 2 * columns * (int64_t)sizeof(float);
}

template<class T, class W>
void LaunchNorm(const NormArgs &a, hipStream_t stream)
{
    hipLaunchKernelGGL((LayerNormKernel<T, W>), dim3(std::min(a.rows, kMostGroups)), dim3(256), 0, stream, a);
    CheckLaunch("LayerNormKernel");
}

template<class T, class W>
void LaunchGrad(const GradArgs &a, hipStream_t stream)
{
    // gradIn may be written over gradOut or in: the sums over rows come first
    if (a.gradGamma != nullptr || a.gradBeta != nullptr)
    {
        const int tiles = DivUp(a.columns, 256);
        if (a.parts > 0)
        {
            hipLaunchKernelGGL((LayerNormPartsKernel<T>), dim3(tiles, a.parts), dim3(256), 0, stream, a);
            CheckLaunch("LayerNormPartsKernel");
        }
        hipLaunchKernelGGL((LayerNormJoinKernel<W>), dim3(tiles), dim3(256), 0, stream, a);
        CheckLaunch("LayerNormJoinKernel");
    }
    if (a.rows > 0)
    {
        hipLaunchKernelGGL((LayerNormGradKernel<T, W>), dim3(std::min(a.rows, kMostGroups)), dim3(256), 0, stream, a);
        CheckLaunch("LayerNormGradKernel");
    }
}

// f(element type's tag, weights' type's tag)
template<class F>
void Dispatch(RowElem elem, bool sameWeights, F &&f)
{
    if (elem == kRowF32)
    {
        f(float{}, float{});
    }
    else if (elem == kRowF16)
    {
        sameWeights ? f(Half{}, Half{}) : f(Half{}, float{});
    }
    else
    {
        sameWeights ? f(Bf16{}, Bf16{}) : f(Bf16{}, float{});
    }
}

// The vectors of D weights given (NULL ones left out): all F32 or all of the rows' type. Sets `same` in the latter case.
struct Weights
{
    RowElem elem;
    int64_t columns;
    RowElem have = kRowNone;

    void *take(NVCVTensorHandle h, const char *what)
    {
        if (h == nullptr)
        {
            return nullptr;
        }
        const DenseView v = RequireDense(h, what, NVCV_DATA_TYPE_NONE);
        const RowElem   e = RowElemOf(v.dtype);
        if (v.count != columns)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must hold %ld elements, not %ld", what, (long)columns, (long)v.count);
        }
        if ((e != kRowF32 && e != elem) || (have != kRowNone && have != e))
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Weights and their gradients must all be F32 or all of the rows' type: %s", what);
        }
        have = e;
        return v.base;
    }

    bool same() const
    {
        return have == elem;
    }
};

float *TakeStatistics(NVCVTensorHandle h, const char *what, int64_t rows)
{
    const DenseView v = RequireDense(h, what, NVCV_DATA_TYPE_F32);
    if (v.count != rows)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must hold an element per row (%ld), not %ld", what, (long)rows, (long)v.count);
    }
    return reinterpret_cast<float *>(v.base);
}

void RequireSame(const RowsView &a, const RowsView &b, const char *what)
{
    if (a.elem != b.elem || a.rows != b.rows || a.columns != b.columns)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have the input's type, rows and row elements", what);
    }
}

class LayerNorm final : public IOperator
{
public:
    void submit(hipStream_t stream, NVCVTensorHandle hin, NVCVTensorHandle hgamma, NVCVTensorHandle hbeta, NVCVTensorHandle hout,
                NVCVTensorHandle hmean, NVCVTensorHandle hrstd, float epsilon) const
    {
        const RowsView in = RequireRows(hin, "Input"), out = RequireRows(hout, "Output");
        RequireSame(in, out, "Output");
        Weights     w     = {in.elem, in.columns};
        const void *gamma = w.take(hgamma, "Gamma"), *beta = w.take(hbeta, "Beta");
        float      *mean  = hmean != nullptr ? TakeStatistics(hmean, "Mean", in.rows) : nullptr;
        float      *rstd  = hrstd != nullptr ? TakeStatistics(hrstd, "Rstd", in.rows) : nullptr;
        if (!(epsilon >= 0) || !std::isfinite(epsilon))
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Epsilon must be a finite number >= 0, not %g", (double)epsilon);
        }
        if (in.rows == 0 || in.columns == 0)
        {
            return;
        }
        const NormArgs a = {RowPlaces(in), RowPlaces(out), gamma, beta, mean, rstd, epsilon, in.rows, in.columns};
        Dispatch(in.elem, w.same(), [&](auto t, auto wt) { LaunchNorm<decltype(t), decltype(wt)>(a, stream); });
    }
};

class LayerNormGrad
{
public:
    static void submit(hipStream_t stream, NVCVTensorHandle hgrad, NVCVTensorHandle hin, NVCVTensorHandle hgamma, NVCVTensorHandle hmean,
                       NVCVTensorHandle hrstd, NVCVTensorHandle hout, NVCVTensorHandle hgradGamma, NVCVTensorHandle hgradBeta,
                       NVCVTensorHandle hworkspace)
    {
        const RowsView in = RequireRows(hin, "Input"), grad = RequireRows(hgrad, "Output's gradient"), out = RequireRows(hout, "Input's gradient");
        RequireSame(in, grad, "Output's gradient");
        RequireSame(in, out, "Input's gradient");
        Weights      w     = {in.elem, in.columns};
        const void  *gamma = w.take(hgamma, "Gamma");
        void        *gradGamma = w.take(hgradGamma, "Gamma's gradient"), *gradBeta = w.take(hgradBeta, "Beta's gradient");
        const float *mean = TakeStatistics(hmean, "Mean", in.rows), *rstd = TakeStatistics(hrstd, "Rstd", in.rows);
        const bool   sums = gradGamma != nullptr || gradBeta != nullptr;
        float       *partial = sums ? reinterpret_cast<float *>(RequireWorkspace(hworkspace, GradWorkspace(in.rows, in.columns))) : nullptr;
        if (in.columns == 0)
        {
            return;
        }
        const GradArgs a = {RowPlaces(grad), RowPlaces(in), RowPlaces(out), gamma, mean, rstd, partial, gradGamma, gradBeta,
                            in.rows, in.columns, Parts(in.rows)};
        Dispatch(in.elem, w.same(), [&](auto t, auto wt) { LaunchGrad<decltype(t), decltype(wt)>(a, stream); });
    }
};

} // namespace
} // namespace cvamd

using namespace cvamd;

extern "C"
{
CVCUDA_PUBLIC NVCVStatus cvcudaxLayerNormCreate(NVCVOperatorHandle *handle)
{
    return CreateOperator<LayerNorm>(handle);
}

CVCUDA_PUBLIC NVCVStatus cvcudaxLayerNormSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle in,
                                                NVCVTensorHandle gamma, NVCVTensorHandle beta, NVCVTensorHandle out,
                                                NVCVTensorHandle mean, NVCVTensorHandle rstd, float epsilon)
{
    return Protect([&] { ToOperator<LayerNorm>(handle).submit(stream, in, gamma, beta, out, mean, rstd, epsilon); });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxLayerNormGradWorkspace(int64_t rows, int64_t columns, int64_t *bytes)
{
    return Protect(
        [&]
        {
            if (bytes == nullptr)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Pointer to output must not be NULL");
            }
            if (rows < 0 || rows > INT32_MAX || columns < 0 || columns > INT32_MAX)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Rows and row elements must be in [0, %d], not %ld and %ld", INT32_MAX, (long)rows,
                              (long)columns);
            }
            *bytes = GradWorkspace(rows, columns);
        });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxLayerNormGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle gradOut,
                                                    NVCVTensorHandle in, NVCVTensorHandle gamma, NVCVTensorHandle mean,
                                                    NVCVTensorHandle rstd, NVCVTensorHandle gradIn,
                                                    NVCVTensorHandle gradGamma, NVCVTensorHandle gradBeta,
                                                    NVCVTensorHandle workspace)
{
    return Protect(
        [&]
        {
            (void)ToOperator<LayerNorm>(handle);
            LayerNormGrad::submit(stream, gradOut, in, gamma, mean, rstd, gradIn, gradGamma, gradBeta, workspace);
        });
}
}
