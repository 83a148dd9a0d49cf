// One step of AdamW over many tensors at once, states in 32 or in 8 bits (formulas: cvcuda/AdamW.h).
//
// The tensors of a call are packed into a launch: its arguments hold a table of them, a workgroup finds its tensor by the
// first tile of each, as image batches of mixed sizes are packed. Nothing is uploaded and nothing is kept.
#include "RowOps.hpp"

#include <cvcuda/AdamW.h>

#include <algorithm>
#include <cmath>

namespace cvamd {

namespace {

constexpr int kBlock = CVCUDAX_ADAMW_BLOCK; // elements that share a scale: a tile

struct Entry
{
    void       *param, *moment, *variance, *copy;
    const void *grad;
    float      *momentScale, *varianceScale;
    int64_t     count;
    uint8_t     paramElem, gradElem, copyElem;
};

// Tensors of a launch: with the coefficients they stay within 4 KiB of arguments.
constexpr int kMostEntries = 48;

struct StepArgs
{
    Entry        entry[kMostEntries];
    uint32_t     firstTile[kMostEntries];
    uint32_t     tiles;
    int32_t      entries;
    const float *gradScale;
    float        beta1, gradPart1, beta2, gradPart2, keep, step, rootScale, epsilon;
};

static_assert(sizeof(StepArgs) <= 4096, "arguments of a launch");

__device__ __forceinline__ float LoadAs(const void *p, int elem, int64_t i)
{
    return elem == kRowF32 ? static_cast<const float *>(p)[i] : elem == kRowF16 ? (float)static_cast<const Half *>(p)[i]
                                                                               : (float)static_cast<const Bf16 *>(p)[i];
}

__device__ __forceinline__ void StoreAs(void *p, int elem, int64_t i, float v)
{
    if (elem == kRowF32)
    {
        static_cast<float *>(p)[i] = v;
    }
    else if (elem == kRowF16)
    {
        static_cast<Half *>(p)[i] = FromFloat<Half>(v);
    }
    else
    {
        static_cast<Bf16 *>(p)[i] = FromFloat<Bf16>(v);
    }
}

__device__ __forceinline__ float MomentOf(int q, float scale)
{
    const float t = (float)q * (1.f / 127.f);
    return (t * fabsf(t)) * scale;
}

__device__ __forceinline__ float VarianceOf(uint32_t q, float scale)
{
    float t = (float)q * (1.f / 255.f);
    t       = t * t;
    return (t * t) * scale;
}

// The larger of two magnitudes; NaN where one is.
__device__ __forceinline__ float Larger(float a, float b)
{
    return a != a || a > b ? a : b;
}

// Of a workgroup of 256, in every thread; NaN unless it is finite.
__device__ __forceinline__ float BlockLargest(float v)
{
    __shared__ float part[4];
#pragma unroll
    for (int s = 32; s > 0; s >>= 1)
    {
        v = Larger(v, __shfl_xor(v, s));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
    {
        part[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = Larger(Larger(part[0], part[1]), Larger(part[2], part[3]));
    return v < __builtin_inff() ? v : __builtin_nanf("");
}

// A code for |value| / scale = share: NaN gives 0.
__device__ __forceinline__ int CodeOf(float root, float most)
{
    const float q = rintf(root * most);
    return q >= 0 ? (int)fminf(q, most) : 0;
}

__device__ __forceinline__ const Entry &EntryOf(const StepArgs &a, uint32_t tile, uint32_t &within)
{
    int e = 0;
    for (int k = 1; k < a.entries; ++k)
    {
        e = tile >= a.firstTile[k] ? k : e;
    }
    within = tile - a.firstTile[e];
    return a.entry[e];
}

// A workgroup per tile, an element per thread.
template<bool SHORT>
__global__ __launch_bounds__(kBlock) void AdamWKernel(const StepArgs a)
{
    for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        uint32_t      within;
        const Entry  &e    = EntryOf(a, tile, within);
        const int64_t i    = (int64_t)within * kBlock + threadIdx.x;
        const bool    live = i < e.count;
        float         p = 0, m = 0, v = 0;
        if (live)
        {
            float g = LoadAs(e.grad, e.gradElem, i);
            g       = a.gradScale != nullptr ? g * *a.gradScale : g;
            p       = LoadAs(e.param, e.paramElem, i);
            m       = SHORT ? MomentOf(static_cast<const int8_t *>(e.moment)[i], e.momentScale[within]) : static_cast<const float *>(e.moment)[i];
            v = SHORT ? VarianceOf(static_cast<const uint8_t *>(e.variance)[i], e.varianceScale[within]) : static_cast<const float *>(e.variance)[i];
            m = a.beta1 * m + g * a.gradPart1;
            v = a.beta2 * v + g * a.gradPart2 * g;
            p = p * a.keep - m / (sqrtf(v) * a.rootScale + a.epsilon) * a.step;
            StoreAs(e.param, e.paramElem, i, p);
            if (e.copy != nullptr)
            {
                StoreAs(e.copy, e.copyElem, i, p);
            }
            if (!SHORT)
            {
                static_cast<float *>(e.moment)[i]   = m;
                static_cast<float *>(e.variance)[i] = v;
            }
        }
        if (SHORT)
        {
            const float ms = BlockLargest(fabsf(m)), vs = BlockLargest(v);
            if (live)
            {
                const int q                          = CodeOf(sqrtf(ms > 0 ? fabsf(m) / ms : 0.f), 127.f);
                static_cast<int8_t *>(e.moment)[i]   = (int8_t)(m < 0 ? -q : q);
                static_cast<uint8_t *>(e.variance)[i] = (uint8_t)max(CodeOf(sqrtf(sqrtf(vs > 0 ? v / vs : 0.f)), 255.f), v > 0 ? 1 : 0);
            }
            if (threadIdx.x == 0)
            {
                e.momentScale[within]   = ms;
                e.varianceScale[within] = vs;
            }
        }
    }
}

struct UnpackEntry
{
    const void  *codes;
    const float *scales;
    float       *out;
    int64_t      count;
    bool         variance;
};

struct UnpackArgs
{
    UnpackEntry entry[kMostEntries];
    uint32_t    firstTile[kMostEntries];
    uint32_t    tiles;
    int32_t     entries;
};

static_assert(sizeof(UnpackArgs) <= 4096, "arguments of a launch");

__global__ __launch_bounds__(kBlock) void AdamWUnpackKernel(const UnpackArgs a)
{
    for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        int n = 0;
        for (int k = 1; k < a.entries; ++k)
        {
            n = tile >= a.firstTile[k] ? k : n;
        }
        const UnpackEntry &e      = a.entry[n];
        const uint32_t     within = tile - a.firstTile[n];
        const int64_t      i      = (int64_t)within * kBlock + threadIdx.x;
        if (i < e.count)
        {
            e.out[i] = e.variance ? VarianceOf(static_cast<const uint8_t *>(e.codes)[i], e.scales[within])
                                  : MomentOf(static_cast<const int8_t *>(e.codes)[i], e.scales[within]);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------
// Workgroups of a launch: a dimension of the grid holds fewer than 2^32 threads.
constexpr uint32_t kMostGroups = 1 << 20;

int64_t Tiles(int64_t count)
{
    return (count + kBlock - 1) / kBlock;
}

NVCVTensorHandle At(const NVCVTensorHandle *list, int i)
{
    return list != nullptr ? list[i] : nullptr;
}

DenseView Take(NVCVTensorHandle h, const char *what, int64_t count, NVCVDataType dt = NVCV_DATA_TYPE_NONE)
{
    const DenseView v = RequireDense(h, what, dt);
    if (v.count != count)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have %ld elements, not %ld", what, (long)count, (long)v.count);
    }
    return v;
}

uint8_t FloatElem(const DenseView &v, const char *what)
{
    const RowElem e = RowElemOf(v.dtype);
    if (e == kRowNone)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must hold F32, F16 or BF16 values", what);
    }
    return (uint8_t)e;
}

void RequireCount(int32_t count, bool lists)
{
    if (count < 0 || (count > 0 && !lists))
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Lists of tensors must not be NULL and their number must be >= 0, not %d", count);
    }
}

// Adds an entry of `tiles` tiles to a launch's table; false where it does not fit behind what is there.
template<class Args, class E>
bool Add(Args &a, const E &e, int64_t tiles)
{
    if (a.entries == kMostEntries || tiles > (int64_t)UINT32_MAX - a.tiles)
    {
        return false;
    }
    a.entry[a.entries]     = e;
    a.firstTile[a.entries] = a.tiles;
    a.tiles += (uint32_t)tiles;
    ++a.entries;
    return true;
}

class AdamW final : public IOperator
{
public:
    static void submit(hipStream_t stream, int32_t count, const NVCVTensorHandle *params, const NVCVTensorHandle *moments,
                       const NVCVTensorHandle *variances, const NVCVTensorHandle *grads, const NVCVTensorHandle *copies,
                       const NVCVTensorHandle *momentScales, const NVCVTensorHandle *varianceScales, NVCVTensorHandle gradScale,
                       const CVCUDAXAdamW *args)
    {
        RequireCount(count, params != nullptr && moments != nullptr && variances != nullptr && grads != nullptr);
        if (args == nullptr)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Pointer to the step's arguments must not be NULL");
        }
        const CVCUDAXAdamW &s = *args;
        if (!std::isfinite(s.lr) || !(s.beta1 >= 0 && s.beta1 < 1) || !(s.beta2 >= 0 && s.beta2 < 1) || !(s.epsilon >= 0)
            || !std::isfinite(s.epsilon) || !std::isfinite(s.weightDecay) || s.step < 1)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT,
                          "Step must be >= 1, betas in [0, 1), epsilon >= 0 and all finite: step %ld, lr %g, betas %g and %g, epsilon %g, "
                          "weight decay %g",
                          (long)s.step, s.lr, s.beta1, s.beta2, s.epsilon, s.weightDecay);
        }
        if ((momentScales == nullptr) != (varianceScales == nullptr))
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Scales must be given for both states or for none");
        }
        const bool small = momentScales != nullptr;
        StepArgs   a     = {};
        if (gradScale != nullptr)
        {
            a.gradScale = reinterpret_cast<const float *>(Take(gradScale, "Gradients' scale", 1, NVCV_DATA_TYPE_F32).base);
        }
        a.beta1     = (float)s.beta1;
        a.gradPart1 = (float)(1 - s.beta1);
        a.beta2     = (float)s.beta2;
        a.gradPart2 = (float)(1 - s.beta2);
        a.keep      = (float)(1 - s.lr * s.weightDecay);
        a.step      = (float)(s.lr / (1 - std::pow(s.beta1, (double)s.step)));
        a.rootScale = (float)(1 / std::sqrt(1 - std::pow(s.beta2, (double)s.step)));
        a.epsilon   = (float)s.epsilon;
        // all of them are looked at before the first is changed
        for (int pass = 0; pass < 2; ++pass)
        {
            for (int i = 0; i < count; ++i)
            {
                const Entry   e     = EntryFor(i, params, moments, variances, grads, copies, momentScales, varianceScales);
                const int64_t tiles = Tiles(e.count);
                if (tiles > UINT32_MAX)
                {
                    throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tensor %d has too many elements", i);
                }
                if (pass == 1 && tiles > 0 && !Add(a, e, tiles))
                {
                    launch(a, small, stream);
                    Add(a, e, tiles);
                }
            }
        }
        launch(a, small, stream);
    }

    static void unpack(hipStream_t stream, int32_t count, const NVCVTensorHandle *codes, const NVCVTensorHandle *scales,
                       const NVCVTensorHandle *out)
    {
        RequireCount(count, codes != nullptr && scales != nullptr && out != nullptr);
        UnpackArgs a = {};
        for (int pass = 0; pass < 2; ++pass)
        {
            for (int i = 0; i < count; ++i)
            {
                const DenseView c = RequireDense(codes[i], "Codes", NVCV_DATA_TYPE_NONE);
                if (c.dtype != NVCV_DATA_TYPE_S8 && c.dtype != NVCV_DATA_TYPE_U8)
                {
                    throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Codes must be S8 or U8");
                }
                const int64_t     tiles = Tiles(c.count);
                const UnpackEntry e     = {c.base, reinterpret_cast<const float *>(Take(scales[i], "Scales", tiles, NVCV_DATA_TYPE_F32).base),
                                           reinterpret_cast<float *>(Take(out[i], "Output", c.count, NVCV_DATA_TYPE_F32).base), c.count,
                                           c.dtype == NVCV_DATA_TYPE_U8};
                if (tiles > UINT32_MAX)
                {
                    throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tensor %d has too many elements", i);
                }
                if (pass == 1 && tiles > 0 && !Add(a, e, tiles))
                {
                    launch(a, stream);
                    Add(a, e, tiles);
                }
            }
        }
        launch(a, stream);
    }

private:
    static Entry EntryFor(int i, const NVCVTensorHandle *params, const NVCVTensorHandle *moments, const NVCVTensorHandle *variances,
                          const NVCVTensorHandle *grads, const NVCVTensorHandle *copies, const NVCVTensorHandle *momentScales,
                          const NVCVTensorHandle *varianceScales)
    {
        const bool      small = momentScales != nullptr;
        const DenseView p     = RequireDense(params[i], "Parameter", NVCV_DATA_TYPE_NONE);
        const DenseView g     = Take(grads[i], "Gradient", p.count);
        Entry           e     = {};
        e.count               = p.count;
        e.param               = p.base;
        e.paramElem           = FloatElem(p, "Parameter");
        e.grad                = g.base;
        e.gradElem            = FloatElem(g, "Gradient");
        e.moment              = Take(moments[i], "Moment", p.count, small ? NVCV_DATA_TYPE_S8 : NVCV_DATA_TYPE_F32).base;
        e.variance            = Take(variances[i], "Variance", p.count, small ? NVCV_DATA_TYPE_U8 : NVCV_DATA_TYPE_F32).base;
        if (small)
        {
            e.momentScale   = reinterpret_cast<float *>(Take(momentScales[i], "Moment's scales", Tiles(p.count), NVCV_DATA_TYPE_F32).base);
            e.varianceScale = reinterpret_cast<float *>(Take(varianceScales[i], "Variance's scales", Tiles(p.count), NVCV_DATA_TYPE_F32).base);
        }
        if (NVCVTensorHandle h = At(copies, i))
        {
            const DenseView c = Take(h, "Copy", p.count);
            e.copy            = c.base;
            e.copyElem        = FloatElem(c, "Copy");
            if (e.copyElem == kRowF32)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Copy must be F16 or BF16");
            }
        }
        return e;
    }

    static void launch(StepArgs &a, bool small, hipStream_t stream)
    {
        if (a.tiles > 0)
        {
            const dim3 grid(std::min(a.tiles, kMostGroups));
            if (small)
            {
                hipLaunchKernelGGL(AdamWKernel<true>, grid, dim3(kBlock), 0, stream, a);
            }
            else
            {
                hipLaunchKernelGGL(AdamWKernel<false>, grid, dim3(kBlock), 0, stream, a);
            }
            CheckLaunch("AdamWKernel");
        }
        a.tiles   = 0;
        a.entries = 0;
    }

    static void launch(UnpackArgs &a, hipStream_t stream)
    {
        if (a.tiles > 0)
        {
            hipLaunchKernelGGL(AdamWUnpackKernel, dim3(std::min(a.tiles, kMostGroups)), dim3(kBlock), 0, stream, a);
            CheckLaunch("AdamWUnpackKernel");
        }
        a.tiles   = 0;
        a.entries = 0;
    }
};

} // namespace
} // namespace cvamd

using namespace cvamd;

extern "C"
{
CVCUDA_PUBLIC NVCVStatus cvcudaxAdamWCreate(NVCVOperatorHandle *handle)
{
    return CreateOperator<AdamW>(handle);
}

CVCUDA_PUBLIC NVCVStatus cvcudaxAdamWSubmit(NVCVOperatorHandle handle, hipStream_t stream, int32_t count,
                                            const NVCVTensorHandle *params, const NVCVTensorHandle *moments,
                                            const NVCVTensorHandle *variances, const NVCVTensorHandle *grads,
                                            const NVCVTensorHandle *copies, const NVCVTensorHandle *momentScales,
                                            const NVCVTensorHandle *varianceScales, NVCVTensorHandle gradScale,
                                            const CVCUDAXAdamW *args)
{
    return Protect(
        [&]
        {
            (void)ToOperator<AdamW>(handle);
            AdamW::submit(stream, count, params, moments, variances, grads, copies, momentScales, varianceScales, gradScale, args);
        });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxAdamWUnpackSubmit(NVCVOperatorHandle handle, hipStream_t stream, int32_t count,
                                                  const NVCVTensorHandle *codes, const NVCVTensorHandle *scales,
                                                  const NVCVTensorHandle *out)
{
    return Protect(
        [&]
        {
            (void)ToOperator<AdamW>(handle);
            AdamW::unpack(stream, count, codes, scales, out);
        });
}
}
