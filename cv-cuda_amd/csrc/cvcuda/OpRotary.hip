// Rotary positions (formulas: cvcuda/Rotary.h). Bound by memory: each element is read and written once (16384 tokens of 40 heads of 128 BF16
// elements, 336 MB: 55.6 us, 6.0 TB/s).
//
// A frequency is held as the fraction of a whole turn that one position makes, in units of 2^-64 turns. A position times it, modulo
// 2^64, is the angle without its whole turns, exactly, however far the position; the eighth of a turn nearest to it is taken off as well,
// and what is left, at most 1/8 turn, is small enough for the sine's and cosine's Taylor polynomials.
#include "HeadOps.hpp"

#include <cvcuda/Rotary.h>

#include <algorithm>
#include <cmath>

namespace cvamd {

namespace {

constexpr int kMostPairs = 128, kRotaryThreads = 256;

struct RotaryArgs
{
    const uint8_t *in;
    uint8_t       *out;
    const void    *positions;
    int64_t        inToken, inHead, outToken, outHead;
    double         step; // the logarithm to the base 2 of what a frequency is of the one before
    double         factor, original, low, high;
    float          magnitude;
    int32_t        tokens, heads, dims, pairs;
    int32_t        copied;         // elements of a row behind the pairs' (0 in place)
    int32_t        turned;         // runs of N pairs of a head
    DivBy          units, ofHeads; // runs of a head: those, then of N copied elements; heads of a token
    bool           wide, inverse;  // wide: positions of 64 bits
};

// The frequency of pair i (cvcuda/Rotary.h) in turns of 2^-64 each.
__device__ __forceinline__ uint64_t TurnsOf(const RotaryArgs &a, int i)
{
    constexpr double kTurn = 0.15915494309189535; // 1 / (2 pi)
    double           turns = exp2(a.step * (double)i) * kTurn;
    if (a.original > 0)
    {
        const double g = fmin(fmax((a.original * turns - a.low) / (a.high - a.low), 0.), 1.);
        turns *= g + (1. - g) / a.factor;
    }
    else
    {
        turns /= a.factor;
    }
    turns -= floor(turns);
    return (uint64_t)(turns * 18446744073709549568.); // (the largest double below 2^64: a fraction next to 1 stays in range)
}

// Cosine and sine of an angle of `hi` * 2^-32 turns.
__device__ __forceinline__ void CosSin(uint32_t hi, float &c, float &s)
{
    const uint32_t quarter = hi + 0x20000000u;                        // the nearest quarter turn in its upper two bits
    const float    x       = (float)(int32_t)(hi - (quarter & 0xC0000000u)) * 1.46291807926715968e-9f; // 2 pi * 2^-32: at most pi / 4
    const float    q       = x * x;
    // terms up to x^9 and x^10: the next ones are below 2^-28
    const float sine = __builtin_fmaf(
        __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(2.7557319e-6f, q, -1.9841270e-4f), q, 8.3333333e-3f), q, -1.6666667e-1f), q * x, x);
    const float cosine = __builtin_fmaf(
        __builtin_fmaf(
            __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(-2.7557319e-7f, q, 2.4801587e-5f), q, -1.3888889e-3f), q, 4.1666667e-2f), q, -0.5f),
        q, 1.f);
    const bool odd = (quarter & 0x40000000u) != 0;
    c              = odd ? sine : cosine;
    s              = odd ? cosine : sine;
    // quarters 1 and 2: the cosine changes its sign, 2 and 3: the sine
    c = __uint_as_float(__float_as_uint(c) ^ ((quarter + 0x40000000u) & 0x80000000u));
    s = __uint_as_float(__float_as_uint(s) ^ (quarter & 0x80000000u));
}

// A lane turns N pairs, or copies N elements behind them, of a token's head; at the end of the pairs and of the row there may be fewer. Lanes
// that follow one another have a head's runs. A lane that turned several heads by its angles measured slower: 16384 tokens of 40 heads
// of 128 BF16 took 59.0 us, with two heads to a lane 59.6, with four 63.6.
template<class T, int N, bool INTERLEAVED, bool PAST>
__global__ __launch_bounds__(kRotaryThreads) void RotaryKernel(const RotaryArgs a)
{
    __shared__ uint64_t s_turns[kMostPairs + N];
    if (threadIdx.x < (uint32_t)(kMostPairs + N))
    {
        s_turns[threadIdx.x] = threadIdx.x < (uint32_t)a.pairs ? TurnsOf(a, (int)threadIdx.x) : 0;
    }
    __syncthreads();
    const uint32_t item = blockIdx.x * kRotaryThreads + threadIdx.x, row = a.units.Quotient(item), unit = item - row * a.units.d;
    const uint32_t token = a.ofHeads.Quotient(row), head = row - token * a.ofHeads.d;
    if (token >= (uint32_t)a.tokens)
    {
        return;
    }
    const T *in  = reinterpret_cast<const T *>(a.in + (int64_t)token * a.inToken + (int64_t)head * a.inHead);
    T       *out = reinterpret_cast<T *>(a.out + (int64_t)token * a.outToken + (int64_t)head * a.outHead);
    if ((int)unit >= a.turned)
    {
        const int at = a.dims + ((int)unit - a.turned) * N, count = a.dims + a.copied - at;
        if (count >= N)
        {
            StoreRun<PAST>(out + at, LoadRun<PAST, T, N>(in + at));
            return;
        }
        for (int i = 0; i < count; ++i)
        {
            out[at + i] = in[at + i];
        }
        return;
    }
    const int      pair = (int)unit * N, count = a.pairs - pair;
    const uint64_t position = a.wide ? static_cast<const uint64_t *>(a.positions)[token]
                                     : (uint64_t)(int64_t)static_cast<const int32_t *>(a.positions)[token];
    float c[N], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
        CosSin((uint32_t)((position * s_turns[pair + i]) >> 32), c[i], s[i]);
        c[i] *= a.magnitude;
        s[i] *= a.inverse ? -a.magnitude : a.magnitude;
    }
    const T *from = in + (INTERLEAVED ? 2 * pair : pair);
    T       *to   = out + (INTERLEAVED ? 2 * pair : pair);
    if (count < N)
    {
        const int step = INTERLEAVED ? 2 : 1, other = INTERLEAVED ? 1 : a.pairs;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            if (i < count)
            {
                const float x = (float)from[i * step], y = (float)from[i * step + other];
                to[i * step]         = FromFloat<T>(x * c[i] - y * s[i]);
                to[i * step + other] = FromFloat<T>(x * s[i] + y * c[i]);
            }
        }
    }
    else if constexpr (INTERLEAVED)
    {
        const Run<T, 2 * N> r = LoadRun<PAST, T, 2 * N>(from);
        Run<T, 2 * N>       made;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const float x = (float)r.v[2 * i], y = (float)r.v[2 * i + 1];
            made.v[2 * i]     = FromFloat<T>(x * c[i] - y * s[i]);
            made.v[2 * i + 1] = FromFloat<T>(x * s[i] + y * c[i]);
        }
        StoreRun<PAST>(to, made);
    }
    else
    {
        const Run<T, N> r = LoadRun<PAST, T, N>(from), t = LoadRun<PAST, T, N>(from + a.pairs);
        Run<T, N>       toX, toY;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const float x = (float)r.v[i], y = (float)t.v[i];
            toX.v[i] = FromFloat<T>(x * c[i] - y * s[i]);
            toY.v[i] = FromFloat<T>(x * s[i] + y * c[i]);
        }
        StoreRun<PAST>(to, toX);
        StoreRun<PAST>(to + a.pairs, toY);
    }
}

template<class T, int N, bool PAST>
void Launch(const RotaryArgs &all, bool interleaved, hipStream_t stream)
{
    const int64_t ofToken = (int64_t)all.units.d * all.ofHeads.d, most = std::max<int64_t>(1, INT32_MAX / ofToken);
    for (int64_t first = 0; first < all.tokens; first += most)
    {
        RotaryArgs a = all;
        a.tokens     = (int32_t)std::min(most, all.tokens - first);
        a.in += first * a.inToken;
        a.out += first * a.outToken;
        a.positions           = static_cast<const uint8_t *>(a.positions) + first * (a.wide ? 8 : 4);
        const uint32_t blocks = (uint32_t)((a.tokens * ofToken + kRotaryThreads - 1) / kRotaryThreads);
        if (!interleaved)
        {
            RotaryKernel<T, N, false, PAST><<<blocks, kRotaryThreads, 0, stream>>>(a);
        }
        else
        {
            RotaryKernel<T, N / 2, true, PAST><<<blocks, kRotaryThreads, 0, stream>>>(a);
        }
        CheckLaunch("rotary");
    }
}

template<class T>
void Choose(RotaryArgs &a, bool interleaved, hipStream_t stream)
{
    // runs of 16 bytes, or of 8 where a row's pairs are whole ones of those alone
    const int wide = interleaved ? kRunOf<T> / 2 : kRunOf<T>, n = a.pairs % wide != 0 && a.pairs % (wide / 2) == 0 ? wide / 2 : wide;
    a.turned  = DivUp(a.pairs, n);
    a.units   = DivBy((uint32_t)(a.turned + DivUp(a.copied, n)));
    a.ofHeads = DivBy((uint32_t)a.heads);
    if ((int64_t)a.units.d * a.ofHeads.d > INT32_MAX)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Input has too many elements in a token");
    }
    const bool past = MovesPastCaches(2 * (int64_t)a.tokens * a.heads * (a.dims + a.copied) * (int64_t)sizeof(T));
    n != wide ? Launch<T, kRunOf<T> / 2, false>(a, interleaved, stream)
    : past    ? Launch<T, kRunOf<T>, true>(a, interleaved, stream)
              : Launch<T, kRunOf<T>, false>(a, interleaved, stream);
}

class Rotary final : public IOperator
{
public:
    static void submit(hipStream_t stream, NVCVTensorHandle hin, NVCVTensorHandle hpositions, NVCVTensorHandle hout, const CVCUDAXRotary *args)
    {
        const HeadsView in = RequireHeads(hin, "Input", 0), out = RequireHeads(hout, "Output", 0);
        RequireSameHeads(in, out, "Output");
        const DenseView positions = RequireDense(hpositions, "Positions", NVCV_DATA_TYPE_NONE);
        if (positions.dtype != NVCV_DATA_TYPE_S32 && positions.dtype != NVCV_DATA_TYPE_S64)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Positions must hold S32 or S64 values");
        }
        if (positions.count != in.tokens)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Positions must have one element for each of %d tokens, not %ld", in.tokens, (long)positions.count);
        }
        if (args == nullptr)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Pointer to arguments must not be NULL");
        }
        if (args->dims < 2 || args->dims % 2 != 0 || args->dims > 2 * kMostPairs || args->dims > in.dims)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Dims must be even, in [2, %d] and at most a head's %d, not %d", 2 * kMostPairs, in.dims, args->dims);
        }
        auto positive = [](double v, const char *what)
        {
            if (!(v > 0) || !std::isfinite(v))
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must be finite and positive, not %g", what, v);
            }
        };
        positive(args->base, "Base");
        positive(args->factor, "Factor");
        positive(args->magnitude, "Magnitude");
        positive((float)args->magnitude, "Magnitude");
        if (!(args->original >= 0) || !std::isfinite(args->original))
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Original must be finite and not negative, not %g", args->original);
        }
        if (args->original > 0 && (!(args->low >= 0) || !(args->high > args->low) || !std::isfinite(args->high)))
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Low and high must be finite, 0 <= low < high, not %g and %g", args->low, args->high);
        }
        if (in.tokens == 0 || in.heads == 0)
        {
            return;
        }
        const bool inPlace = in.base == out.base && (in.tokens == 1 || in.tokenStride == out.tokenStride) && in.headStride == out.headStride;
        RotaryArgs a = {in.base, out.base, positions.base, in.tokenStride, in.headStride, out.tokenStride, out.headStride,
                        std::log2(args->base) * -2. / args->dims, args->factor, args->original, args->low, args->high, (float)args->magnitude,
                        in.tokens, in.heads, args->dims, args->dims / 2, inPlace ? 0 : in.dims - args->dims, 0, DivBy(1), DivBy(1),
                        positions.dtype == NVCV_DATA_TYPE_S64, args->inverse != 0};
        const bool interleaved = args->interleaved != 0;
        switch (in.elem)
        {
        case kRowF32: Choose<float>(a, interleaved, stream); break;
        case kRowF16: Choose<Half>(a, interleaved, stream); break;
        default: Choose<Bf16>(a, interleaved, stream); break;
        }
    }
};

} // namespace
} // namespace cvamd

using namespace cvamd;

extern "C"
{
CVCUDA_PUBLIC NVCVStatus cvcudaxRotaryCreate(NVCVOperatorHandle *handle)
{
    return CreateOperator<Rotary>(handle);
}

CVCUDA_PUBLIC NVCVStatus cvcudaxRotarySubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle in,
                                             NVCVTensorHandle positions, NVCVTensorHandle out, const CVCUDAXRotary *args)
{
    return Protect(
        [&]
        {
            (void)ToOperator<Rotary>(handle);
            Rotary::submit(stream, in, positions, out, args);
        });
}
}
