// Layer norm of rows, and its gradient (formulas: cvcuda/LayerNorm.h). Bound by memory: a row is read once and held in
// registers by one, four or more waves, runs of 16 bytes of it in each lane.
//
// The variance is the mean of the squares of what remains of each element without the mean: the difference of the mean
// square and the squared mean would lose it in rows that lie far from 0. The gradient's sums over rows stay in the registers of
// workgroups that go through the rows in turn; each leaves its own in the workspace, a second launch adds them up: always in
// the same order.
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
    int32_t     rows, columns, firstRow;
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

// The runs of a lane in a row that WAVES waves hold: run k is N elements from `first(k)` on. It is loaded from `from(k)` on, which
// lies before that where the row ends within or before the run, so that no load stands under a condition; of what is loaded
// the elements from skip(k) on are its own. Stores are of whole runs too: twice the same values where runs overlap.
template<int N, int WAVES>
struct RowRuns
{
    int columns, lane0;

    __device__ __forceinline__ explicit RowRuns(int of)
        : columns(of)
        , lane0((int)((WAVES == 1 ? 0 : WaveOfGroup() * 64) + (threadIdx.x & 63)) * N)
    {
    }

    __device__ __forceinline__ int first(int k) const
    {
        return k * WAVES * 64 * N + lane0;
    }

    __device__ __forceinline__ int from(int k) const
    {
        return min(first(k), columns - N);
    }

    __device__ __forceinline__ int skip(int k) const
    {
        return first(k) - from(k);
    }

    // all lanes' runs lie within the row
    __device__ __forceinline__ bool whole(int k) const
    {
        return (k + 1) * WAVES * 64 * N <= columns;
    }

    template<class T>
    __device__ __forceinline__ Run<T, N> get(const void *row, int k) const
    {
        return *reinterpret_cast<const Run<T, N> *>(static_cast<const T *>(row) + from(k));
    }

    template<class T>
    __device__ __forceinline__ void put(void *row, int k, const float (&v)[N]) const
    {
        if (first(k) < columns)
        {
            Run<T, N> r;
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                r.v[i] = FromFloat<T>(v[i]);
            }
            *reinterpret_cast<Run<T, N> *>(static_cast<T *>(row) + from(k)) = r;
        }
    }
};

// Sum over the WAVES waves of a row, in all of them. `part`: room for a sum of each, not read by anyone at the time.
template<int WAVES>
__device__ __forceinline__ float RowSum(float v, float (&part)[WAVES])
{
    v = WaveSum(v);
    if constexpr (WAVES > 1)
    {
        part[WaveOfGroup()] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
        {
            v += part[w];
        }
    }
    return v;
}

// Waves of the widest workgroup. The gradient's lanes also hold two sums for each element: with sixteen waves, 128 registers
// to a lane, they would not fit.
constexpr int kNormWidest = 16, kGradWidest = 8;

constexpr int GroupWaves(int waves)
{
    return waves == 1 ? 4 : waves; // narrow rows: four to a workgroup
}

// Workgroups of sixteen waves go through the rows in turn, each with the next row on its way: they are alone on their CU or nearly
// so, and each sum would find all of its waves waiting (4000 rows of 8192 BF16 38 us, 52 with a workgroup to each row; with eight
// waves 26 and 24, with four and 65536 rows of 4096 209 and 191). Not with 32 elements in a lane: two rows of them do not fit
// in the registers (2000 rows of 24576 F32 144 us and 95).
constexpr bool Turns(int waves, int elements)
{
    return waves == kNormWidest && elements <= 16;
}

// E: elements in a lane. 65536 rows of 4096 BF16 190 us, 5.6 TB/s; 12544 rows of 768 F16 11 us, 3.6 TB/s (half of that is the first
// loads' and the last stores' time), one row 2.6.
template<class T, class W, int WAVES, int E>
__global__ __launch_bounds__(64 * GroupWaves(WAVES)) void LayerNormKernel(const NormArgs a)
{
    constexpr int    N = std::min(E, kRunOf<T>), K = E / N;
    constexpr bool   kTurns        = Turns(WAVES, E);
    constexpr bool   kWeightsFirst = E <= 16; // on their way beside the row; more of them would take registers from other rows
    __shared__ float s_sum[WAVES], s_squares[WAVES];
    const RowRuns<N, WAVES> runs(a.columns);
    uint32_t                row = a.firstRow + (WAVES == 1 ? blockIdx.x * 4 + WaveOfGroup() : blockIdx.x);
    if (row >= (uint32_t)a.rows)
    {
        return;
    }
    Run<T, N> x[K];
    Run<W, N> gamma[K], beta[K];
    auto      load = [&](Run<T, N>(&to)[K], uint32_t r)
    {
        const uint8_t *from = a.in.at(r);
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            to[k] = runs.template get<T>(from, k);
        }
    };
    load(x, row);
    auto loadWeights = [&]
    {
        if (a.gamma != nullptr)
        {
#pragma unroll
            for (int k = 0; k < K; ++k)
            {
                gamma[k] = runs.template get<W>(a.gamma, k);
            }
        }
        if (a.beta != nullptr)
        {
#pragma unroll
            for (int k = 0; k < K; ++k)
            {
                beta[k] = runs.template get<W>(a.beta, k);
            }
        }
    };
    if (kWeightsFirst)
    {
        loadWeights();
    }
    for (;;)
    {
        float s = 0;
        Run<T, N> next[K];
        if (kTurns && gridDim.x < (uint32_t)a.rows - row)
        {
            load(next, row + gridDim.x);
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            const int skip = runs.whole(k) ? 0 : runs.skip(k);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                s += i >= skip ? (float)x[k].v[i] : 0.f;
            }
        }
        const float mean = RowSum<WAVES>(s, s_sum) / (float)a.columns;
        s                = 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            const int skip = runs.whole(k) ? 0 : runs.skip(k);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                const float d = i >= skip ? (float)x[k].v[i] - mean : 0.f;
                s += d * d;
            }
        }
        const float rstd = 1.f / sqrtf(RowSum<WAVES>(s, s_squares) / (float)a.columns + a.epsilon);
        uint8_t    *to   = a.out.at(row);
        if (!kWeightsFirst)
        {
            loadWeights();
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            float y[N];
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                y[i] = ((float)x[k].v[i] - mean) * rstd;
            }
            if (a.gamma != nullptr)
            {
#pragma unroll
                for (int i = 0; i < N; ++i)
                {
                    y[i] *= (float)gamma[k].v[i];
                }
            }
            if (a.beta != nullptr)
            {
#pragma unroll
                for (int i = 0; i < N; ++i)
                {
                    y[i] += (float)beta[k].v[i];
                }
            }
            runs.template put<T>(to, k, y);
        }
        if (runs.lane0 == 0)
        {
            if (a.mean != nullptr)
            {
                a.mean[row] = mean;
            }
            if (a.rstd != nullptr)
            {
                a.rstd[row] = rstd;
            }
        }
        if (!kTurns || gridDim.x >= (uint32_t)a.rows - row)
        {
            break;
        }
        row += gridDim.x;
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            x[k] = next[k];
        }
    }
}

// The rows' gradient, and the sums over the rows that a workgroup goes through: every parts-th (in narrow rows each of its
// waves takes one). The next row and its statistics are on their way while the sums of one are awaited (8949 rows of 3328 F16 43
// us, 49 where the statistics were not), unless two rows are too much for the registers (4000 rows of 12288 F32 124 us and 214).
// 65536 rows of 4096 BF16 283 us, 5.7 TB/s; 12544 rows of 768 F16 15.6 us, 3.7 TB/s.
template<class T, class W, int WAVES, int E, bool SUMS>
__device__ __forceinline__ void GradRows(const GradArgs &a)
{
    constexpr int    N = std::min(E, kRunOf<T>), K = E / N, kRows = WAVES == 1 ? 4 : 1;
    constexpr bool   kAhead = E * sizeof(T) <= 64;
    __shared__ float s_sum[2][2][WAVES]; // of one row and the next
    const RowRuns<N, WAVES> runs(a.columns);
    const uint32_t          step = (uint32_t)a.parts * kRows;
    uint32_t                row  = blockIdx.x * kRows + (WAVES == 1 ? WaveOfGroup() : 0);
    float                   gamma[K][N], toGamma[K][N] = {}, toBeta[K][N] = {};
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            gamma[k][i] = 1;
        }
    }
    if (a.gamma != nullptr)
    {
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            const Run<W, N> g = runs.template get<W>(a.gamma, k);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                gamma[k][i] = (float)g.v[i];
            }
        }
    }
    Run<T, N> x[K], dy[K];
    float     mean, rstd;
    auto      load = [&](uint32_t r)
    {
        mean = a.mean[r];
        rstd = a.rstd[r];
        const uint8_t *px = a.in.at(r), *pdy = a.grad.at(r);
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            x[k]  = runs.template get<T>(px, k);
            dy[k] = runs.template get<T>(pdy, k);
        }
    };
    if (row < (uint32_t)a.rows)
    {
        load(row);
    }
    for (int turn = 0; row < (uint32_t)a.rows; row += step, turn ^= 1)
    {
        const float scale = rstd;
        float       w[K][N], h[K][N], s = 0, sh = 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            const int skip = runs.whole(k) ? 0 : runs.skip(k);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                const float d = (float)dy[k].v[i];
                h[k][i]       = ((float)x[k].v[i] - mean) * rstd;
                w[k][i]       = d * gamma[k][i];
                if constexpr (SUMS)
                {
                    toGamma[k][i] += d * h[k][i];
                    toBeta[k][i] += d;
                }
                s += i >= skip ? w[k][i] : 0.f;
                sh += i >= skip ? w[k][i] * h[k][i] : 0.f;
            }
        }
        const uint32_t next = row + step;
        if (kAhead && next < (uint32_t)a.rows)
        {
            load(next);
        }
        s  = WaveSum(s);
        sh = WaveSum(sh);
        if constexpr (WAVES > 1)
        {
            s_sum[turn][0][WaveOfGroup()] = s;
            s_sum[turn][1][WaveOfGroup()] = sh;
            __syncthreads();
            s = sh = 0;
#pragma unroll
            for (int i = 0; i < WAVES; ++i)
            {
                s += s_sum[turn][0][i];
                sh += s_sum[turn][1][i];
            }
        }
        s /= (float)a.columns;
        sh /= (float)a.columns;
        uint8_t *to = a.out.at(row);
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                w[k][i] = scale * (w[k][i] - s - h[k][i] * sh);
            }
            runs.template put<T>(to, k, w[k]);
        }
        if (!kAhead && next < (uint32_t)a.rows)
        {
            load(next);
        }
    }
    if (!SUMS || a.partial == nullptr)
    {
        return;
    }
    if constexpr (WAVES == 1)
    {
        // the workgroup's four waves hold the same columns
        __shared__ float s_part[4][64][N];
        const uint32_t   wave = WaveOfGroup(), lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < 2 * K; ++j)
        {
            float(&v)[N] = j < K ? toGamma[j] : toBeta[j - K];
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                s_part[wave][lane][i] = v[i];
            }
            __syncthreads();
            if (wave == (uint32_t)j % 4)
            {
#pragma unroll
                for (int i = 0; i < N; ++i)
                {
                    v[i] = s_part[0][lane][i] + s_part[1][lane][i] + s_part[2][lane][i] + s_part[3][lane][i];
                }
                runs.template put<float>(a.partial + ((size_t)blockIdx.x * 2 + j / K) * a.columns, j % K, v);
            }
            __syncthreads();
        }
    }
    else
    {
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            runs.template put<float>(a.partial + (size_t)blockIdx.x * 2 * a.columns, k, toGamma[k]);
            runs.template put<float>(a.partial + ((size_t)blockIdx.x * 2 + 1) * a.columns, k, toBeta[k]);
        }
    }
}

template<class T, class W, int WAVES, int E>
__global__ __launch_bounds__(64 * GroupWaves(WAVES)) void LayerNormGradKernel(const GradArgs a)
{
    GradRows<T, W, WAVES, E, true>(a);
}

// Rows too wide for registers, or of fewer than four columns: a workgroup goes over the row more than once, by runs of N (one for
// narrow rows). 1000 rows of 50000 BF16 86 us, their gradient 144
// (element by element 310 and 493): what the second time reads is in the cache.
constexpr int kAnyThreads = 1024;

// Sum over a workgroup of kAnyThreads, in every thread.
__device__ __forceinline__ float BlockSum(float v)
{
    __shared__ float part[kAnyThreads / 64];
    __syncthreads();
    return RowSum(v, part);
}

// The run from `first` on of D columns; it is loaded from `from` on, the first `skip` of what is loaded are not its own.
template<int N>
struct AnyRun
{
    int from, skip;

    __device__ __forceinline__ AnyRun(int first, int D)
        : from(min(first, D - N))
        , skip(first - from)
    {
    }

    template<class T>
    __device__ __forceinline__ Run<T, N> get(const void *row) const
    {
        return *reinterpret_cast<const Run<T, N> *>(static_cast<const T *>(row) + from);
    }

    // the weights of its columns: 1 or 0 where there are none
    template<class W>
    __device__ __forceinline__ void weights(float (&v)[N], const void *w, float none) const
    {
        if (w == nullptr)
        {
            for (float &x : v)
            {
                x = none;
            }
            return;
        }
        const Run<W, N> r = get<W>(w);
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            v[i] = (float)r.v[i];
        }
    }

    // (its own alone: others' may be read from the same memory still)
    template<class T>
    __device__ __forceinline__ void put(void *row, const float (&v)[N]) const
    {
        T        *to = static_cast<T *>(row) + from;
        Run<T, N> r;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            r.v[i] = FromFloat<T>(v[i]);
        }
        if (skip == 0)
        {
            *reinterpret_cast<Run<T, N> *>(to) = r;
            return;
        }
#pragma unroll
        for (int i = 1; i < N; ++i)
        {
            if (i >= skip)
            {
                to[i] = r.v[i];
            }
        }
    }
};

template<class T, class W, int N>
__global__ __launch_bounds__(kAnyThreads) void LayerNormAnyKernel(const NormArgs a)
{
    const int D = a.columns;
    for (uint32_t row = blockIdx.x; row < (uint32_t)a.rows; row += gridDim.x)
    {
        const uint8_t *x = a.in.at(row);
        uint8_t       *y = a.out.at(row);
        float          s = 0;
        for (int c = threadIdx.x * N; c < D; c += kAnyThreads * N)
        {
            const AnyRun<N> run(c, D);
            const Run<T, N> v = run.template get<T>(x);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                s += i >= run.skip ? (float)v.v[i] : 0.f;
            }
        }
        const float mean = BlockSum(s) / (float)D;
        s                = 0;
        for (int c = threadIdx.x * N; c < D; c += kAnyThreads * N)
        {
            const AnyRun<N> run(c, D);
            const Run<T, N> v = run.template get<T>(x);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                const float d = i >= run.skip ? (float)v.v[i] - mean : 0.f;
                s += d * d;
            }
        }
        const float rstd = 1.f / sqrtf(BlockSum(s) / (float)D + a.epsilon);
        for (int c = threadIdx.x * N; c < D; c += kAnyThreads * N)
        {
            const AnyRun<N> run(c, D);
            const Run<T, N> v = run.template get<T>(x);
            float           g[N], b[N], out[N];
            run.template weights<W>(g, a.gamma, 1);
            run.template weights<W>(b, a.beta, 0);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                out[i] = ((float)v.v[i] - mean) * rstd * g[i] + b[i];
            }
            run.template put<T>(y, out);
        }
        if (threadIdx.x == 0 && a.mean != nullptr)
        {
            a.mean[row] = mean;
        }
        if (threadIdx.x == 0 && a.rstd != nullptr)
        {
            a.rstd[row] = rstd;
        }
    }
}

template<class T, class W, int N>
__global__ __launch_bounds__(kAnyThreads) void LayerNormGradAnyKernel(const GradArgs a)
{
    const int D = a.columns;
    for (uint32_t row = blockIdx.x; row < (uint32_t)a.rows; row += gridDim.x)
    {
        const uint8_t *dy = a.grad.at(row), *x = a.in.at(row);
        uint8_t       *dx   = a.out.at(row);
        const float    mean = a.mean[row], rstd = a.rstd[row];
        float          s = 0, sh = 0;
        for (int c = threadIdx.x * N; c < D; c += kAnyThreads * N)
        {
            const AnyRun<N> run(c, D);
            const Run<T, N> v = run.template get<T>(x), d = run.template get<T>(dy);
            float           g[N];
            run.template weights<W>(g, a.gamma, 1);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                const float w = (float)d.v[i] * g[i];
                s += i >= run.skip ? w : 0.f;
                sh += i >= run.skip ? w * (((float)v.v[i] - mean) * rstd) : 0.f;
            }
        }
        s  = BlockSum(s) / (float)D;
        sh = BlockSum(sh) / (float)D;
        for (int c = threadIdx.x * N; c < D; c += kAnyThreads * N)
        {
            const AnyRun<N> run(c, D);
            const Run<T, N> v = run.template get<T>(x), d = run.template get<T>(dy);
            float           g[N], out[N];
            run.template weights<W>(g, a.gamma, 1);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                const float w = (float)d.v[i] * g[i], h = ((float)v.v[i] - mean) * rstd;
                out[i]        = rstd * (w - s - h * sh);
            }
            run.template put<T>(dx, out);
        }
    }
}

// The same rows' sums: a thread for each run of columns and part of the rows.
constexpr int kPartsThreads = 256;

template<class T, int N>
__global__ __launch_bounds__(kPartsThreads) void LayerNormPartsAnyKernel(const GradArgs a)
{
    const int64_t c = ((int64_t)blockIdx.x * kPartsThreads + threadIdx.x) * N;
    const int     D = a.columns;
    if (c >= D)
    {
        return;
    }
    const AnyRun<N> run((int)c, D);
    float           g[N] = {}, b[N] = {};
#pragma unroll 4
    for (uint32_t r = blockIdx.y; r < (uint32_t)a.rows; r += a.parts)
    {
        const float     mean = a.mean[r], rstd = a.rstd[r];
        const Run<T, N> v = run.template get<T>(a.in.at(r)), d = run.template get<T>(a.grad.at(r));
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            g[i] += (float)d.v[i] * (((float)v.v[i] - mean) * rstd);
            b[i] += (float)d.v[i];
        }
    }
    run.template put<float>(a.partial + (size_t)blockIdx.y * 2 * D, g);
    run.template put<float>(a.partial + ((size_t)blockIdx.y * 2 + 1) * D, b);
}

// The sums over few rows, of as many columns as a workgroup holds for 32 rows at once, in runs of four.
constexpr int kFewSlots = 32, kFewRun = 4;

constexpr int FewColumns(int threads)
{
    return threads / kFewSlots * kFewRun;
}

template<class T, class W, int THREADS>
__device__ __forceinline__ void SumColumns(const GradArgs &a, uint32_t tile)
{
    constexpr int    N = kFewRun, kColumns = FewColumns(THREADS), kLanes = kColumns / N, kAhead = 8; // rows of a lane on their way
    __shared__ float s_gamma[kFewSlots][kColumns], s_beta[kFewSlots][kColumns];
    const int        slot = threadIdx.x / kLanes, first = (int)tile * kColumns + (threadIdx.x % kLanes) * N;
    const AnyRun<N>  run(first, a.columns);
    float            g[N] = {}, b[N] = {};
    for (int r0 = slot; r0 < a.rows; r0 += kFewSlots * kAhead)
    {
        Run<T, N> x[kAhead], dy[kAhead];
        float     mean[kAhead], rstd[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
        {
            const uint32_t r = min(r0 + j * kFewSlots, a.rows - 1);
            x[j]             = run.template get<T>(a.in.at(r));
            dy[j]            = run.template get<T>(a.grad.at(r));
            mean[j]          = a.mean[r];
            rstd[j]          = a.rstd[r];
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
        {
            const bool there = r0 + j * kFewSlots < a.rows;
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                const float d = (float)dy[j].v[i];
                g[i] += there ? d * (((float)x[j].v[i] - mean[j]) * rstd[j]) : 0.f;
                b[i] += there ? d : 0.f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
        if (i >= run.skip)
        {
            const int at     = run.from + i - (int)tile * kColumns;
            s_gamma[slot][at] = g[i];
            s_beta[slot][at]  = b[i];
        }
    }
    __syncthreads();
    const int c = threadIdx.x % kColumns, column = (int)tile * kColumns + c, which = threadIdx.x / kColumns;
    W        *to = static_cast<W *>(which == 0 ? a.gradGamma : a.gradBeta);
    if (which < 2 && column < a.columns && to != nullptr)
    {
        float s = 0;
#pragma unroll
        for (int k = 0; k < kFewSlots; ++k)
        {
            s += which == 0 ? s_gamma[k][c] : s_beta[k][c];
        }
        to[column] = FromFloat<W>(s);
    }
}

// Few rows: all of the gradient in one launch, the sums from the rows themselves by workgroups behind those of the rows. 256 rows of
// 768 BF16 4.2 us (in two launches 7.5, and a call 4 more), 512 rows of 4096 7.2 (13.9), 1024 of 768 9.0 (9.2).
template<class T, class W, int WAVES, int E>
__global__ __launch_bounds__(64 * GroupWaves(WAVES)) void LayerNormGradFewKernel(const GradArgs a)
{
    if (blockIdx.x < (uint32_t)a.parts)
    {
        GradRows<T, W, WAVES, E, false>(a);
    }
    else
    {
        SumColumns<T, W, 64 * GroupWaves(WAVES)>(a, blockIdx.x - a.parts);
    }
}

// Adds up the parts' sums: 16 columns to a workgroup, whose 64 rows of 16 lanes take every 64th part each (512 parts of 4096
// columns 7.5 us, of 768 3.9, most of them one wait after another).
constexpr int kJoinColumns = 16;

template<class W>
__global__ __launch_bounds__(1024) void LayerNormJoinKernel(const GradArgs a)
{
    __shared__ float s_part[64][kJoinColumns + 1];
    const int64_t    all = 2 * (int64_t)a.columns;
    const int        l = threadIdx.x % kJoinColumns, r = threadIdx.x / kJoinColumns;
    for (int64_t first = (int64_t)blockIdx.x * kJoinColumns; first < all; first += (int64_t)gridDim.x * kJoinColumns)
    {
        const int64_t c = min(first + l, all - 1);
        float         s = 0;
#pragma unroll 8
        for (int p = r; p < a.parts; p += 64)
        {
            s += a.partial[(size_t)p * all + c];
        }
        s_part[r][l] = s;
        __syncthreads();
#pragma unroll
        for (int n = 32; n > 0; n >>= 1)
        {
            if (r < n)
            {
                s_part[r][l] += s_part[r + n][l];
            }
            __syncthreads();
        }
        if (r == 0 && first + l < all)
        {
            void *to = c < a.columns ? a.gradGamma : a.gradBeta;
            if (to != nullptr)
            {
                static_cast<W *>(to)[c < a.columns ? c : c - a.columns] = FromFloat<W>(s_part[0][l]);
            }
        }
        __syncthreads();
    }
}

// Workgroups of a launch: a dimension of the grid holds fewer than 2^32 threads.
constexpr int kMostGroups = 1 << 20;

// ---- host ----------------------------------------------------------------------------------------------------------
// What a kernel of rows is built for: waves to a row and elements to a lane. 0 waves: the kernels for any width.
struct RowShape
{
    int waves, elements;
};

constexpr int kNarrowest = 4; // columns, of a lane where they are few

// The fewest waves whose lanes hold the row with 16 elements each, 32 where the widest workgroup needs them. Eight where they
// suffice: 40000 rows of 8192 BF16 258 us, 391 with sixteen of which half their runs lie behind the row. Lanes of four where a
// wave has enough: 60000 rows of 200 F32 17 us, 19 with runs of eight, the gradient 28 and 31.
RowShape ShapeOf(int64_t columns, int widest)
{
    if (columns < kNarrowest || columns > widest * 64 * 32)
    {
        return {0, 0};
    }
    const int waves = columns <= 64 * 16 ? 1 : columns <= 4 * 64 * 16 ? 4 : columns <= 8 * 64 * 16 ? 8 : widest;
    return {waves, columns <= 64 * 4 ? 4 : columns <= waves * 64 * 8 ? 8 : columns <= waves * 64 * 16 ? 16 : 32};
}

// Rows whose gradient is one launch: the sums over 2048 of 768 would take 18 us, with a second launch 10. At any width that a workgroup
// holds: whole calls of 1024 rows of 8192 BF16 are 19 us, 21 with a second launch, of 16384 32 and 40, and the fewer rows the more (512 of
// 16384 19 and 30, up to 4096 columns 15.5 and 17). Only the widest F32 rows, read a second time, are even: 1024 of 8192 27 and 26, of 12288 44
// and 44, of 16384 60 and 58; 512 of 16384 30 and 33.
constexpr int kFewRows = 1024;

bool Few(int64_t rows, int64_t columns)
{
    return rows > 0 && rows <= kFewRows && ShapeOf(columns, kGradWidest).waves != 0;
}

// Workgroups that share the rows of a gradient. Each has the next row under way, so two waves on a SIMD are enough where a lane
// has 16 elements or more, and fewer sums are left to add up: 65536 rows of 4096 BF16 293 us with 512 workgroups of four waves,
// 317 with 768, 343 with 1024, 352 with 384; 4000 rows of 8192 56 with 256 of eight, 64 with 512. Lanes of 8 or 4 elements want as
// many as fit, six: 60000 rows of 512 40 us with 1536, 52 with 512.
constexpr int64_t kMostParts = 1536;

// Rows that no workgroup holds have a launch of their own for the sums, of tiles of 1024 columns or more and parts: a million columns
// in all parts together are 500 workgroups or more, and what they leave is 8 MiB, little beside the rows themselves. 6144 rows of 40000 BF16
// 598 us, 585 with two million, 741 with half of one, 1153 with a part to four rows; 2000 rows of 20000 F32 201, 208, 204 and 238. Rows of
// fewer than four columns have one tile, and so the most parts (100000 rows of 3 F32 270 us).
constexpr int64_t kWideSums = 1 << 20;

int PartsOf(int64_t rows, int64_t columns)
{
    const RowShape s    = ShapeOf(columns, kGradWidest);
    const int64_t  most = s.waves == 0      ? std::min(kMostParts, std::max<int64_t>(1, kWideSums / std::max<int64_t>(columns, 1)))
                          : s.elements <= 8 ? kMostParts
                                            : 2048 / std::max(s.waves, 4);
    return (int)std::min((rows + 3) / 4, most);
}

// A gradient of one launch has no use for a workspace, and asks for the least: callers bring one, and learn that it is missing, at any
// number of rows. What is touched is larger.
int64_t GradWorkspace(int64_t rows, int64_t columns)
{
    constexpr int64_t kUntouched = CVCUDAX_LAYER_NORM_UNTOUCHED_WORKSPACE;
    if (Few(rows, columns))
    {
        return kUntouched;
    }
    const int64_t bytes = (int64_t)PartsOf(rows, columns) * 2 * columns * (int64_t)sizeof(float);
    return bytes > 0 ? std::max(bytes, 2 * kUntouched) : 0;
}

template<class T, class W, int WAVES, int E>
void LaunchNormAs(const NormArgs &a, hipStream_t stream)
{
    const int64_t groups = WAVES == 1 ? ((int64_t)a.rows + 3) / 4 : a.rows;
    if (Turns(WAVES, E))
    {
        hipLaunchKernelGGL((LayerNormKernel<T, W, WAVES, E>), dim3((uint32_t)std::min<int64_t>(groups, 256)), dim3(64 * WAVES), 0, stream, a);
        CheckLaunch("LayerNormKernel");
        return;
    }
    // (rows beyond what a launch may hold go into further ones)
    constexpr int64_t kMost = ((int64_t)1 << 32) / (64 * GroupWaves(WAVES)) - 1;
    for (int64_t first = 0; first < groups; first += kMost)
    {
        NormArgs b = a;
        b.firstRow = (int32_t)(first * (WAVES == 1 ? 4 : 1));
        hipLaunchKernelGGL((LayerNormKernel<T, W, WAVES, E>), dim3((uint32_t)std::min(groups - first, kMost)), dim3(64 * GroupWaves(WAVES)), 0, stream, b);
        CheckLaunch("LayerNormKernel");
    }
}

template<class T, class W>
void LaunchNorm(const NormArgs &a, hipStream_t stream)
{
    const RowShape s = ShapeOf(a.columns, kNormWidest);
    if (s.waves == 0)
    {
        const auto kernel = a.columns < kNarrowest ? LayerNormAnyKernel<T, W, 1> : LayerNormAnyKernel<T, W, kRunOf<T>>;
        hipLaunchKernelGGL(kernel, dim3(std::min(a.rows, kMostGroups)), dim3(kAnyThreads), 0, stream, a);
        CheckLaunch("LayerNormAnyKernel");
    }
    else if (s.waves == 1)
    {
        s.elements == 4   ? LaunchNormAs<T, W, 1, 4>(a, stream)
        : s.elements == 8 ? LaunchNormAs<T, W, 1, 8>(a, stream)
                          : LaunchNormAs<T, W, 1, 16>(a, stream);
    }
    else if (s.waves == 4)
    {
        s.elements == 8 ? LaunchNormAs<T, W, 4, 8>(a, stream) : LaunchNormAs<T, W, 4, 16>(a, stream);
    }
    else if (s.waves == 8)
    {
        LaunchNormAs<T, W, 8, 16>(a, stream);
    }
    else
    {
        s.elements <= 16 ? LaunchNormAs<T, W, kNormWidest, 16>(a, stream) : LaunchNormAs<T, W, kNormWidest, 32>(a, stream);
    }
}

template<class T, class W, int WAVES, int E>
void LaunchGradAs(const GradArgs &a, hipStream_t stream)
{
    if (Few(a.rows, a.columns))
    {
        // gradIn may be written over gradOut or in: the sums over rows come first there
        const bool     sums = a.gradGamma != nullptr || a.gradBeta != nullptr, over = a.out.base == a.grad.base || a.out.base == a.in.base;
        const uint32_t tiles = sums ? DivUp(a.columns, FewColumns(64 * GroupWaves(WAVES))) : 0, rows = DivUp(a.rows, WAVES == 1 ? 4 : 1);
        auto           launch = [&](uint32_t rowGroups, uint32_t columnGroups)
        {
            GradArgs b = a;
            b.parts    = (int32_t)rowGroups;
            hipLaunchKernelGGL((LayerNormGradFewKernel<T, W, WAVES, E>), dim3(rowGroups + columnGroups), dim3(64 * GroupWaves(WAVES)), 0, stream, b);
            CheckLaunch("LayerNormGradFewKernel");
        };
        if (over && sums)
        {
            launch(0, tiles);
            launch(rows, 0);
        }
        else
        {
            launch(rows, tiles);
        }
        return;
    }
    hipLaunchKernelGGL((LayerNormGradKernel<T, W, WAVES, E>), dim3(a.parts), dim3(64 * GroupWaves(WAVES)), 0, stream, a);
    CheckLaunch("LayerNormGradKernel");
}

template<class T, class W>
void LaunchGrad(const GradArgs &a, hipStream_t stream)
{
    const RowShape s    = ShapeOf(a.columns, kGradWidest);
    const bool     sums = a.gradGamma != nullptr || a.gradBeta != nullptr;
    if (a.rows == 0)
    {
    }
    else if (s.waves == 0)
    {
        // gradIn may be written over gradOut or in: the sums over rows come first
        const bool narrow = a.columns < kNarrowest;
        if (sums)
        {
            const auto kernel = narrow ? LayerNormPartsAnyKernel<T, 1> : LayerNormPartsAnyKernel<T, kRunOf<T>>;
            hipLaunchKernelGGL(kernel, dim3(DivUp(a.columns, kPartsThreads * (narrow ? 1 : kRunOf<T>)), a.parts), dim3(kPartsThreads), 0, stream, a);
            CheckLaunch("LayerNormPartsAnyKernel");
        }
        const auto kernel = narrow ? LayerNormGradAnyKernel<T, W, 1> : LayerNormGradAnyKernel<T, W, kRunOf<T>>;
        hipLaunchKernelGGL(kernel, dim3(std::min(a.rows, kMostGroups)), dim3(kAnyThreads), 0, stream, a);
        CheckLaunch("LayerNormGradAnyKernel");
    }
    else if (s.waves == 1)
    {
        s.elements == 4   ? LaunchGradAs<T, W, 1, 4>(a, stream)
        : s.elements == 8 ? LaunchGradAs<T, W, 1, 8>(a, stream)
                          : LaunchGradAs<T, W, 1, 16>(a, stream);
    }
    else if (s.waves == 4)
    {
        s.elements == 8 ? LaunchGradAs<T, W, 4, 8>(a, stream) : LaunchGradAs<T, W, 4, 16>(a, stream);
    }
    else
    {
        s.elements <= 16 ? LaunchGradAs<T, W, kGradWidest, 16>(a, stream) : LaunchGradAs<T, W, kGradWidest, 32>(a, stream);
    }
    if (sums && !Few(a.rows, a.columns))
    {
        const int64_t groups = (2 * (int64_t)a.columns + kJoinColumns - 1) / kJoinColumns;
        hipLaunchKernelGGL((LayerNormJoinKernel<W>), dim3((uint32_t)std::min<int64_t>(groups, kMostGroups)), dim3(1024), 0, stream, a);
        CheckLaunch("LayerNormJoinKernel");
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
        const NormArgs a = {RowPlaces(in), RowPlaces(out), gamma, beta, mean, rstd, epsilon, in.rows, in.columns, 0};
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
        uint8_t     *room    = sums ? RequireWorkspace(hworkspace, GradWorkspace(in.rows, in.columns)) : nullptr;
        float       *partial = Few(in.rows, in.columns) ? nullptr : reinterpret_cast<float *>(room);
        if (in.columns == 0)
        {
            return;
        }
        const GradArgs a = {RowPlaces(grad), RowPlaces(in), RowPlaces(out), gamma, mean, rstd, partial, gradGamma, gradBeta,
                            in.rows, in.columns, PartsOf(in.rows, in.columns)};
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
