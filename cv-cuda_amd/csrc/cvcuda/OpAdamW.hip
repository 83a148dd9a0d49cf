// One step of AdamW over many tensors at once, states in 32 or in 8 bits (formulas: cvcuda/AdamW.h).
//
// The tensors of a call are packed into a launch: its arguments hold a table of them, a workgroup finds its tensor by the
// first tile of each, as image batches of mixed sizes are packed. Nothing is uploaded and nothing is kept.
#include "RowOps.hpp"

#include <cvcuda/AdamW.h>

#include <algorithm>
#include <cmath>
#include <vector>

namespace cvamd {

namespace {

constexpr int kBlock = CVCUDAX_ADAMW_BLOCK; // elements that share a scale: four for each lane of a wave
constexpr int kRun   = 4;                   // elements that follow one another in a lane

// Runs of a lane that are on their way before the first is used, of 8-bit states and of codes to unpack: 120 M elements take 640 us
// so, 690 with two of each, 813 with one. Of 32-bit states one is enough, four arrays of 16 bytes: 210 M elements 1070 us, 1100
// with two, 1120 with four.
constexpr int kSmallRuns = 2, kUnpackRuns = 4;

// Elements of a workgroup of four waves.
constexpr int kStepTile = 4 * kBlock, kSmallTile = 4 * kSmallRuns * kBlock, kUnpackTile = 4 * kUnpackRuns * kBlock;

static_assert(kBlock == 64 * kRun, "a wave's runs make a block");

struct Entry
{
    void       *param, *moment, *variance, *copy;
    const void *grad;
    float      *momentScale, *varianceScale;
    int64_t     count;
    int32_t     copyElem;
};

// Tensors of a launch: with the coefficients they stay within 4 KiB of arguments.
constexpr int kMostEntries = 48;

struct StepArgs
{
    Entry        entry[kMostEntries];
    uint32_t     firstTile[kMostEntries]; // behind the last entry: no tile's number
    uint32_t     tiles;
    int32_t      entries;
    const float *gradScale;
    float        beta1, gradPart1, beta2, gradPart2, keep, step, rootScale, epsilon;
};

static_assert(sizeof(StepArgs) <= 4096, "arguments of a launch");

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

// A code as the formula gives it: NaN gives 0.
__device__ __forceinline__ int CodeOf(float root, float most)
{
    const float q = rintf(root * most);
    return q >= 0 ? (int)fminf(q, most) : 0;
}

// Codes of magnitudes of a block with the largest `scale`. The formula's division and square roots are rounded to the nearest:
// forty instructions and more for each. The hardware's approximations are within 2^-23 of them each, so that a code can differ
// only where its root is within 6 * 2^-23 * 255 = 1.9e-4 of the middle between two: those are made again by the formula,
// and so is a block whose scale has no reciprocal among the normal numbers.
template<bool VARIANCE>
__device__ __forceinline__ float Code(float magnitude, float scale, float reciprocal, bool ordinary)
{
    constexpr float most = VARIANCE ? 255.f : 127.f;
    float           root = __builtin_amdgcn_sqrtf(magnitude * reciprocal);
    root                 = (VARIANCE ? __builtin_amdgcn_sqrtf(root) : root) * most;
    float code           = rintf(root);
    if (!ordinary || fabsf(root - code) > 0.5f - 2.5e-4f || (VARIANCE && root < 0.5f))
    {
        root = sqrtf(scale > 0 ? magnitude / scale : 0.f);
        code = (float)CodeOf(VARIANCE ? sqrtf(root) : root, most);
        code = VARIANCE && magnitude > 0 ? fmaxf(code, 1.f) : code;
    }
    return code;
}

struct Moments
{
    float m, v;
};

// One element: the moments after the step, and p.
__device__ __forceinline__ Moments Step(const StepArgs &a, float &p, float m, float v, float g, float gradScale)
{
    g = g * gradScale;
    m = a.beta1 * m + g * a.gradPart1;
    v = a.beta2 * v + g * a.gradPart2 * g;
    p = p * a.keep - m / (sqrtf(v) * a.rootScale + a.epsilon) * a.step;
    return {m, v};
}

template<class T>
__device__ __forceinline__ Run<T, kRun> RunAt(const void *base, int64_t i)
{
    return *reinterpret_cast<const Run<T, kRun> *>(static_cast<const T *>(base) + i);
}

template<class T>
__device__ __forceinline__ void PutRun(void *base, int64_t i, const float (&v)[kRun])
{
    Run<T, kRun> r;
#pragma unroll
    for (int k = 0; k < kRun; ++k)
    {
        r.v[k] = FromFloat<T>(v[k]);
    }
    *reinterpret_cast<Run<T, kRun> *>(static_cast<T *>(base) + i) = r;
}

// The same of floats, as one streaming store.
__device__ __forceinline__ void StreamRun(void *base, int64_t i, const float (&v)[kRun])
{
    uint32_t w[kRun];
    __builtin_memcpy(w, v, sizeof(w));
    StoreDwordsNT<kRun>(reinterpret_cast<uint8_t *>(static_cast<float *>(base) + i), w);
}

__device__ __forceinline__ void PutCopy(const Entry &e, int64_t i, const float (&v)[kRun])
{
    if (e.copy != nullptr) // (of the whole tensor)
    {
        e.copyElem == kRowF16 ? PutRun<Half>(e.copy, i, v) : PutRun<Bf16>(e.copy, i, v);
    }
}

__device__ __forceinline__ void PutCopyOne(const Entry &e, int64_t i, float v)
{
    if (e.copy != nullptr)
    {
        e.copyElem == kRowF16 ? (void)(static_cast<Half *>(e.copy)[i] = FromFloat<Half>(v)) : (void)(static_cast<Bf16 *>(e.copy)[i] = FromFloat<Bf16>(v));
    }
}

// The entry of a tile. All first tiles are compared at once: a search would wait for each of its loads.
template<class Args>
__device__ __forceinline__ int EntryOf(const Args &a, uint32_t tile)
{
    int e = 0;
#pragma unroll
    for (int k = 1; k < kMostEntries; ++k)
    {
        e += tile >= a.firstTile[k] ? 1 : 0;
    }
    return e;
}

// States of 32 bits. 24 bytes of an element and its gradient's, 40 instructions: bound by memory (134 M elements with BF16 gradients
// 654 us, 5.3 TB/s; 772 thousand F32 ones 6.2 us).
template<class P, class G>
__global__ __launch_bounds__(256) void AdamWKernel(const StepArgs a)
{
    const float gradScale = a.gradScale != nullptr ? *a.gradScale : 1.f;
    for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        const int     n     = EntryOf(a, tile);
        const Entry  &e     = a.entry[n];
        const int64_t first = (int64_t)(tile - a.firstTile[n]) * kStepTile;
        float        *ms = static_cast<float *>(e.moment), *vs = static_cast<float *>(e.variance);
        if (first + kStepTile <= e.count)
        {
            const int64_t    i = first + threadIdx.x * kRun;
            const auto       p = RunAt<P>(e.param, i);
            const auto       g = RunAt<G>(e.grad, i);
            Run<float, kRun> m = RunAt<float>(ms, i), v = RunAt<float>(vs, i);
            float            pn[kRun];
#pragma unroll
            for (int k = 0; k < kRun; ++k)
            {
                pn[k]           = (float)p.v[k];
                const Moments s = Step(a, pn[k], m.v[k], v.v[k], (float)g.v[k], gradScale);
                m.v[k]          = s.m;
                v.v[k]          = s.v;
            }
            PutRun<P>(e.param, i, pn);
            PutRun<float>(ms, i, m.v);
            PutRun<float>(vs, i, v.v);
            PutCopy(e, i, pn);
            continue;
        }
        for (int64_t i = first + threadIdx.x; i < e.count; i += 256)
        {
            float         p = (float)static_cast<const P *>(e.param)[i];
            const Moments s = Step(a, p, ms[i], vs[i], (float)static_cast<const G *>(e.grad)[i], gradScale);
            static_cast<P *>(e.param)[i] = FromFloat<P>(p);
            ms[i]                        = s.m;
            vs[i]                        = s.v;
            PutCopyOne(e, i, p);
        }
    }
}

// What a block's codes are made with.
struct BlockScale
{
    float scale, reciprocal;
    bool  ordinary;

    // of the largest magnitude's bits
    __device__ __forceinline__ explicit BlockScale(uint32_t largest)
    {
        scale      = largest < 0x7F800000u ? __uint_as_float(largest) : __builtin_nanf("");
        reciprocal = __builtin_amdgcn_rcpf(scale);
        ordinary   = scale > 1e-30f && scale < 1e30f;
    }
};

// States of 8 bits: a wave takes whole blocks, whose largest magnitudes are found across its lanes. Bound by its arithmetic: 110
// instructions and six approximations of an element, 410 us for 134 M elements, which move their 14 bytes in 370 (measured: 430).
template<class P, class G>
__global__ __launch_bounds__(256) void AdamWSmallKernel(const StepArgs a)
{
    const float    gradScale = a.gradScale != nullptr ? *a.gradScale : 1.f;
    const uint32_t lane      = threadIdx.x & 63;
    for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        const int     n     = EntryOf(a, tile);
        const Entry  &e     = a.entry[n];
        const int64_t block = (int64_t)(tile - a.firstTile[n]) * (kSmallTile / kBlock) + WaveOfGroup() * kSmallRuns, first = block * kBlock;
        int8_t       *mq = static_cast<int8_t *>(e.moment);
        uint8_t      *vq = static_cast<uint8_t *>(e.variance);
        const bool    whole = first + kSmallRuns * kBlock <= e.count;
        Run<P, kRun>       p[kSmallRuns] = {};
        Run<G, kRun>       g[kSmallRuns] = {};
        Run<int8_t, kRun>  m[kSmallRuns] = {};
        Run<uint8_t, kRun> v[kSmallRuns] = {};
        float              ms[kSmallRuns] = {}, vs[kSmallRuns] = {};
        if (whole)
        {
#pragma unroll
            for (int r = 0; r < kSmallRuns; ++r)
            {
                const int64_t i = first + r * kBlock + lane * kRun;
                p[r]            = RunAt<P>(e.param, i);
                g[r]            = RunAt<G>(e.grad, i);
                m[r]            = RunAt<int8_t>(mq, i);
                v[r]            = RunAt<uint8_t>(vq, i);
                ms[r]           = e.momentScale[block + r];
                vs[r]           = e.varianceScale[block + r];
            }
        }
        else
        {
#pragma unroll
            for (int r = 0; r < kSmallRuns; ++r)
            {
                if (first + r * kBlock < e.count)
                {
                    ms[r] = e.momentScale[block + r];
                    vs[r] = e.varianceScale[block + r];
                }
#pragma unroll
                for (int k = 0; k < kRun; ++k)
                {
                    const int64_t i = first + r * kBlock + lane * kRun + k;
                    if (i < e.count)
                    {
                        p[r].v[k] = static_cast<const P *>(e.param)[i];
                        g[r].v[k] = static_cast<const G *>(e.grad)[i];
                        m[r].v[k] = mq[i];
                        v[r].v[k] = vq[i];
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kSmallRuns; ++r)
        {
            const int64_t i = first + r * kBlock + lane * kRun;
            if (first + r * kBlock >= e.count)
            {
                break;
            }
            float    pn[kRun], mn[kRun], vn[kRun];
            uint32_t mMost = 0, vMost = 0;
#pragma unroll
            for (int k = 0; k < kRun; ++k)
            {
                pn[k]           = (float)p[r].v[k];
                const Moments s = Step(a, pn[k], MomentOf(m[r].v[k], ms[r]), VarianceOf(v[r].v[k], vs[r]), (float)g[r].v[k], gradScale);
                const bool    in = whole || i + k < e.count; // (past the end nothing counts)
                mn[k]            = in ? s.m : 0.f;
                vn[k]            = in ? s.v : 0.f;
                mMost            = max(mMost, __float_as_uint(fabsf(mn[k])));
                vMost            = max(vMost, __float_as_uint(fabsf(vn[k])));
            }
            const BlockScale   mScale(WaveLargest(mMost)), vScale(WaveLargest(vMost));
            uint32_t           mBytes = 0, vBytes = 0;
            Run<int8_t, kRun>  mCode;
            Run<uint8_t, kRun> vCode;
#pragma unroll
            for (int k = 0; k < kRun; ++k)
            {
                const float q = Code<false>(fabsf(mn[k]), mScale.scale, mScale.reciprocal, mScale.ordinary);
                mBytes |= ((uint32_t)(int)copysignf(q, mn[k]) & 255) << 8 * k;
                vBytes = __builtin_amdgcn_cvt_pk_u8_f32(Code<true>(vn[k], vScale.scale, vScale.reciprocal, vScale.ordinary), k, vBytes);
            }
            __builtin_memcpy(&mCode, &mBytes, sizeof(mCode));
            __builtin_memcpy(&vCode, &vBytes, sizeof(vCode));
            if (lane == 0)
            {
                e.momentScale[block + r]   = mScale.scale;
                e.varianceScale[block + r] = vScale.scale;
            }
            if (whole)
            {
                PutRun<P>(e.param, i, pn);
                *reinterpret_cast<Run<int8_t, kRun> *>(mq + i)  = mCode;
                *reinterpret_cast<Run<uint8_t, kRun> *>(vq + i) = vCode;
                PutCopy(e, i, pn);
                continue;
            }
#pragma unroll
            for (int k = 0; k < kRun; ++k)
            {
                if (i + k < e.count)
                {
                    static_cast<P *>(e.param)[i + k] = FromFloat<P>(pn[k]);
                    mq[i + k]                        = mCode.v[k];
                    vq[i + k]                        = vCode.v[k];
                    PutCopyOne(e, i + k, pn[k]);
                }
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

// 5 bytes of an element, four of them written: 134 M elements 96 us, 7.0 TB/s, the rate of a fill.
__global__ __launch_bounds__(256) void AdamWUnpackKernel(const UnpackArgs a)
{
    for (uint32_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x)
    {
        const int          n     = EntryOf(a, tile);
        const UnpackEntry &e     = a.entry[n];
        const int64_t      first = (int64_t)(tile - a.firstTile[n]) * kUnpackTile;
        if (first + kUnpackTile <= e.count)
        {
            Run<uint8_t, kRun> q[kUnpackRuns];
            float              scale[kUnpackRuns];
#pragma unroll
            for (int r = 0; r < kUnpackRuns; ++r)
            {
                const int64_t i = first + (r * 256 + threadIdx.x) * kRun;
                q[r]            = RunAt<uint8_t>(e.codes, i);
                scale[r]        = e.scales[i / kBlock];
            }
#pragma unroll
            for (int r = 0; r < kUnpackRuns; ++r)
            {
                float v[kRun];
#pragma unroll
                for (int k = 0; k < kRun; ++k)
                {
                    v[k] = e.variance ? VarianceOf(q[r].v[k], scale[r]) : MomentOf((int8_t)q[r].v[k], scale[r]);
                }
                StreamRun(e.out, first + (r * 256 + threadIdx.x) * kRun, v);
            }
            continue;
        }
        for (int64_t i = first + threadIdx.x; i < e.count; i += 256)
        {
            e.out[i] = e.variance ? VarianceOf(static_cast<const uint8_t *>(e.codes)[i], e.scales[i / kBlock])
                                  : MomentOf(static_cast<const int8_t *>(e.codes)[i], e.scales[i / kBlock]);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------
// Workgroups of a launch: a dimension of the grid holds fewer than 2^32 threads.
constexpr uint32_t kMostGroups = 1 << 20;

int64_t Tiles(int64_t count, int tile)
{
    return (count + tile - 1) / tile;
}

int64_t Blocks(int64_t count)
{
    return (count + kBlock - 1) / kBlock;
}

template<class Args>
void Clear(Args &a)
{
    a.tiles   = 0;
    a.entries = 0;
    std::fill_n(a.firstTile, kMostEntries, UINT32_MAX);
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

RowElem FloatElem(const DenseView &v, const char *what)
{
    const RowElem e = RowElemOf(v.dtype);
    if (e == kRowNone)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must hold F32, F16 or BF16 values", what);
    }
    return e;
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
    if (a.entries == kMostEntries || tiles >= (int64_t)UINT32_MAX - a.tiles)
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
        // all of them are looked at before the first is changed; those of one pair of types go into a launch
        const int          tile = small ? kSmallTile : kStepTile;
        std::vector<Given> given(count);
        bool               there[kRowNone][kRowNone] = {};
        for (int i = 0; i < count; ++i)
        {
            given[i] = EntryFor(i, params, moments, variances, grads, copies, momentScales, varianceScales);
            if (Tiles(given[i].entry.count, tile) >= UINT32_MAX)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tensor %d has too many elements", i);
            }
            there[given[i].param][given[i].grad] = true;
        }
        for (int pair = 0; pair < kRowNone * kRowNone; ++pair)
        {
            const auto param = (RowElem)(pair / kRowNone), grad = (RowElem)(pair % kRowNone);
            if (!there[param][grad])
            {
                continue;
            }
            Clear(a);
            for (const Given &g : given)
            {
                const int64_t tiles = Tiles(g.entry.count, tile);
                if (g.param == param && g.grad == grad && tiles > 0 && !Add(a, g.entry, tiles))
                {
                    launch(a, param, grad, small, stream);
                    Add(a, g.entry, tiles);
                }
            }
            launch(a, param, grad, small, stream);
        }
    }

    static void unpack(hipStream_t stream, int32_t count, const NVCVTensorHandle *codes, const NVCVTensorHandle *scales,
                       const NVCVTensorHandle *out)
    {
        RequireCount(count, codes != nullptr && scales != nullptr && out != nullptr);
        UnpackArgs a = {};
        Clear(a);
        for (int pass = 0; pass < 2; ++pass)
        {
            for (int i = 0; i < count; ++i)
            {
                const DenseView c = RequireDense(codes[i], "Codes", NVCV_DATA_TYPE_NONE);
                if (c.dtype != NVCV_DATA_TYPE_S8 && c.dtype != NVCV_DATA_TYPE_U8)
                {
                    throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Codes must be S8 or U8");
                }
                const int64_t     tiles = Tiles(c.count, kUnpackTile);
                const UnpackEntry e     = {c.base, reinterpret_cast<const float *>(Take(scales[i], "Scales", Blocks(c.count), NVCV_DATA_TYPE_F32).base),
                                           reinterpret_cast<float *>(Take(out[i], "Output", c.count, NVCV_DATA_TYPE_F32).base), c.count,
                                           c.dtype == NVCV_DATA_TYPE_U8};
                if (tiles >= UINT32_MAX)
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
    struct Given
    {
        Entry   entry;
        RowElem param, grad;
    };

    static Given EntryFor(int i, const NVCVTensorHandle *params, const NVCVTensorHandle *moments, const NVCVTensorHandle *variances,
                          const NVCVTensorHandle *grads, const NVCVTensorHandle *copies, const NVCVTensorHandle *momentScales,
                          const NVCVTensorHandle *varianceScales)
    {
        const bool      small = momentScales != nullptr;
        const DenseView p     = RequireDense(params[i], "Parameter", NVCV_DATA_TYPE_NONE);
        const DenseView g     = Take(grads[i], "Gradient", p.count);
        Given           given = {{}, FloatElem(p, "Parameter"), FloatElem(g, "Gradient")};
        Entry          &e     = given.entry;
        e.count               = p.count;
        e.param               = p.base;
        e.grad                = g.base;
        e.moment              = Take(moments[i], "Moment", p.count, small ? NVCV_DATA_TYPE_S8 : NVCV_DATA_TYPE_F32).base;
        e.variance            = Take(variances[i], "Variance", p.count, small ? NVCV_DATA_TYPE_U8 : NVCV_DATA_TYPE_F32).base;
        if (small)
        {
            e.momentScale   = reinterpret_cast<float *>(Take(momentScales[i], "Moment's scales", Blocks(p.count), NVCV_DATA_TYPE_F32).base);
            e.varianceScale = reinterpret_cast<float *>(Take(varianceScales[i], "Variance's scales", Blocks(p.count), NVCV_DATA_TYPE_F32).base);
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
        return given;
    }

    template<class P, class G>
    static void launch(const StepArgs &a, bool small, hipStream_t stream)
    {
        const dim3 grid(std::min(a.tiles, kMostGroups));
        if (small)
        {
            hipLaunchKernelGGL((AdamWSmallKernel<P, G>), grid, dim3(256), 0, stream, a);
        }
        else
        {
            hipLaunchKernelGGL((AdamWKernel<P, G>), grid, dim3(256), 0, stream, a);
        }
        CheckLaunch("AdamWKernel");
    }

    template<class P>
    static void launch(const StepArgs &a, RowElem grad, bool small, hipStream_t stream)
    {
        grad == kRowF32   ? launch<P, float>(a, small, stream)
        : grad == kRowF16 ? launch<P, Half>(a, small, stream)
                          : launch<P, Bf16>(a, small, stream);
    }

    static void launch(StepArgs &a, RowElem param, RowElem grad, bool small, hipStream_t stream)
    {
        if (a.tiles > 0)
        {
            param == kRowF32   ? launch<float>(a, grad, small, stream)
            : param == kRowF16 ? launch<Half>(a, grad, small, stream)
                               : launch<Bf16>(a, grad, small, stream);
        }
        Clear(a);
    }

    static void launch(UnpackArgs &a, hipStream_t stream)
    {
        if (a.tiles > 0)
        {
            hipLaunchKernelGGL(AdamWUnpackKernel, dim3(std::min(a.tiles, kMostGroups)), dim3(256), 0, stream, a);
            CheckLaunch("AdamWUnpackKernel");
        }
        Clear(a);
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
