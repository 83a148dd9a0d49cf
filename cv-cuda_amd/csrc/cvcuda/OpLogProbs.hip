// Log probabilities of tokens with entropy and top alternatives, and their gradient (formulas: cvcuda/LogProbs.h). Bound by memory: the
// logits are read once.
//
// One pass over a row: each wave has a logit a that it takes exponentials relative to, and the sums r of e = exp(z - z_a) and t of
// e * (z - z_a) of all its logits but a. a is the largest of its first ones, and then the largest of those that lie more than kSlack above a, the
// sums being rescaled: few do. The waves' are joined relative to the largest a. Log probabilities are then (x - a) * scale - log(1 + r), the entropy is
// log(1 + r) - t / (1 + r). Of a row with one logit far above the others that one is a: r is what the others leave of it, in all its digits,
// and nothing of the size of logits, or of 1, is there to cancel. (A largest logit that isn't a lies at most kSlack above it, so that a has
// a share of 1 / (1 + e^kSlack) at least beside it.)
//
// The top tokens come from what the pass has anyway: a number that K of the lanes' largest logits, by 64 groups, reach is one that K
// logits of the row reach, so that the lanes which reach it, few in most rows, look through theirs again for those that do (4096 rows of
// 128000 BF16 with the top 5 188 us, 5.6 TB/s). Where too many do, or the row has NaN, the whole row is gone over K times.
#include "RowOps.hpp"

#include <cvcuda/LogProbs.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace cvamd {

namespace {

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2   = 0.6931471805599453f;
constexpr float kFar   = -1e30f; // below any difference whose exponential isn't 0; a sum of 2^31 of it is finite
constexpr float kSlack = 2.f; // (4096 rows of 128000 BF16 189.5 us; with 20 187.7, and what is within that of a likely token's logit lies in its digits)

__device__ __forceinline__ float Exp(float x)
{
    return __builtin_amdgcn_exp2f(x * kLog2E);
}
constexpr int   kGroups = 64, kCandidates = 512, kFewMore = 5;
static_assert(CVCUDAX_LOG_PROBS_MOST_TOP <= kGroups, "as many groups as top tokens");

struct LogProbsArgs
{
    RowPlaces   logits;
    const void *tokens;
    float      *out, *entropy, *lse, *topValues; // all but out: nullptr where not wanted
    int32_t    *topTokens;
    float       scale, slack; // slack: kSlack / scale
    int32_t     rows, columns, top, firstRow;
    bool        wide; // tokens of 64 bits
};

__device__ __forceinline__ int64_t TokenAt(const void *tokens, bool wide, uint32_t row)
{
    return wide ? static_cast<const int64_t *>(tokens)[row] : static_cast<const int32_t *>(tokens)[row];
}

// Whole numbers in the order of the logits: NaN above all, -0 as +0.
__device__ __forceinline__ uint32_t OrderOf(float x)
{
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0xFFFFFFFFu : (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float ValueOf(uint32_t order)
{
    return order == 0xFFFFFFFFu ? NAN : __uint_as_float((order & 0x80000000u) != 0 ? order & 0x7FFFFFFFu : ~order);
}

// A logit and its column: larger logits first, of equal ones the lower columns.
__device__ __forceinline__ uint64_t KeyOf(float x, int column)
{
    return ((uint64_t)OrderOf(x) << 32) | (0xFFFFFFFFu - (uint32_t)column);
}

__device__ __forceinline__ int ColumnOf(uint64_t key)
{
    return (int)(0xFFFFFFFFu - (uint32_t)key);
}

// Run r of a row: N logits from N * r on, at the row's end the last N of it, of which those from `skip` on are its own.
template<class T, int N, bool PAST>
struct Logits
{
    Run<T, N> run;
    int       from, skip;

    __device__ __forceinline__ void get(const T *row, int columns, int r)
    {
        from = min(r * N, columns - N);
        skip = r * N - from;
        run  = LoadRun<PAST, T, N>(row + from);
    }
};

struct TopRoom
{
    uint32_t group[kGroups];
    uint64_t key[kCandidates];
    uint32_t count;
};

// The largest of the lanes' keys, in all of them. `part`: room that nobody reads or writes at the time, nor after the next barrier.
template<int WAVES>
__device__ __forceinline__ uint64_t LargestKey(uint64_t v, uint64_t (&part)[WAVES])
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
    {
        const uint64_t o = ((uint64_t)__shfl_xor((uint32_t)(v >> 32), d) << 32) | __shfl_xor((uint32_t)v, d);
        v                = o > v ? o : v;
    }
    if constexpr (WAVES > 1)
    {
        __syncthreads();
        part[WaveOfGroup()] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
        {
            v = part[w] > v ? part[w] : v;
        }
    }
    return v;
}

// What the row's log probabilities are taken relative to: that of x is scale * x - scale * at - logSum.
struct Total
{
    float scale, base, rounding, logSum; // base: scale * at, rounded; rounding: what it is short of that
    bool  nothing;                       // all logits are -infinity

    __device__ __forceinline__ float of(float x) const
    {
        return nothing ? -INFINITY : (__builtin_fmaf(x, scale, -base) - rounding) - logSum;
    }
};

// Entry `rank` of a row's top tokens.
__device__ __forceinline__ void PutTop(const LogProbsArgs &a, uint32_t row, int rank, uint64_t key, const Total &total)
{
    const int64_t at = (int64_t)row * a.top + rank;
    a.topTokens[at]  = ColumnOf(key);
    a.topValues[at]  = total.of(ValueOf((uint32_t)(key >> 32)));
}

// The largest of three numbers, in one instruction: fmaxf makes a copy of each that may be a NaN first (three more instructions for two
// logits; 4096 rows of 128000 BF16 255 us, 249 with this).
__device__ __forceinline__ float Largest(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// The largest of N logits and of `top`. (A NaN among them is left out.)
template<int N>
__device__ __forceinline__ float LargestOf(float top, const float (&v)[N])
{
#pragma unroll
    for (int i = 0; i < N; i += 2)
    {
        top = Largest(top, v[i], v[std::min(i + 1, N - 1)]);
    }
    return top;
}

// The sums r of e and t of e * (z - z_a) over some logits but `at`, the logit a (-infinity: all were).
struct Sums
{
    float at, r, t;
};

// A wave's lanes on their way through the row.
struct Running
{
    float at, base, limit; // the same in all lanes: scale * at, rounded, and the logit above which the sums are rescaled
    float r, t, top;       // the lane's, relative to `base`; its largest logit

    __device__ __forceinline__ explicit Running()
        : at(-INFINITY)
        , base(-INFINITY)
        , limit(-INFINITY)
        , r(0)
        , t(0)
        , top(-INFINITY)
    {
    }

    // Sums from now on relative to `to`, the largest of the lanes' `top` and one of their next logits v: the first lane that has it
    // takes it out of them.
    template<int N>
    __device__ __forceinline__ void begin(float to, float (&v)[N], float scale, float slack)
    {
        const uint64_t some = __ballot(top == to);
        bool           mine = some != 0 && (int)(threadIdx.x & 63) == (int)__builtin_ctzll(some);
        base  = to * scale;
        at    = base == -INFINITY ? base : to;
        limit = at == -INFINITY ? at : at + slack;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const bool its = mine && v[i] == to;
            v[i]           = its ? -INFINITY : v[i];
            mine           = mine && !its;
        }
    }

    // The lanes' next N logits (-infinity where one has none).
    template<int N>
    __device__ __forceinline__ void next(float (&v)[N], float scale, float slack)
    {
        top = LargestOf(top, v);
        if (__any(top > limit))
        {
            const float to = ValueOf(WaveLargest(OrderOf(top)));
            if (at != -INFINITY)
            {
                // the logit `at` is one of the first lane's from here on
                const float its = rounding(scale), e = (threadIdx.x & 63) == 0 ? Exp(its) : 0.f;
                const float less = fmaxf(base - to * scale, kFar), share = Exp(less);
                r += e;
                t = share * __builtin_fmaf(r, less, __builtin_fmaf(e, its, t));
                r = share * r;
            }
            begin(to, v, scale, slack);
        }
        add(v, scale);
    }

    template<int N>
    __device__ __forceinline__ void add(const float (&v)[N], float scale)
    {
        const float from = base == -INFINITY ? 0.f : base; // (all were -infinity so far)
        float       e[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const float d = __builtin_fmaf(v[i], scale, -from);
            e[i]          = Exp(d);
            t             = __builtin_fmaf(e[i], fmaxf(d, kFar), t); // (e is 0 where d is -infinity)
        }
#pragma unroll
        for (int w = N / 2; w > 0; w /= 2)
        {
#pragma unroll
            for (int i = 0; i < w; ++i)
            {
                e[i] += e[i + w];
            }
        }
        r += e[0];
    }

    // What scale * at is above `base`.
    __device__ __forceinline__ float rounding(float scale) const
    {
        return base == -INFINITY ? 0.f : __builtin_fmaf(at, scale, -base);
    }

    // The wave's, relative to `at` itself.
    __device__ __forceinline__ Sums sums(float scale) const
    {
        Sums        s    = {at, WaveSum(r), WaveSum(t)};
        const float less = -rounding(scale);
        if (less != 0)
        {
            const float share = Exp(less);
            s.t = share * __builtin_fmaf(s.r, less, s.t);
            s.r = share * s.r;
        }
        return s;
    }
};

// log(1 + r), to its own last bits: 1 + r is u and what was lost when that was rounded, whose share of u is what the logarithm lacks.
__device__ __forceinline__ float Log1(float r)
{
    const float u = 1.f + r;
    return __builtin_fmaf(__builtin_amdgcn_logf(u), kLn2, (r - (u - 1.f)) * __builtin_amdgcn_rcpf(u));
}

// The sums that a wave's lanes have as one.
__device__ __forceinline__ Sums Joined(const Sums &s, float scale)
{
    const float    at   = ValueOf(WaveLargest(OrderOf(s.at)));
    const uint64_t some = __ballot(s.at == at);
    const bool     its  = some != 0 && (int)(threadIdx.x & 63) == (int)__builtin_ctzll(some);
    const float    less = s.at == at ? 0.f : fmaxf((s.at - at) * scale, kFar), share = Exp(less), all = s.r + (its || s.at == -INFINITY ? 0.f : 1.f);
    return {at, WaveSum(share * all), WaveSum(share * __builtin_fmaf(all, less, s.t))};
}

// N: logits of a run (1 where rows are narrower than 16 bytes). One workgroup to a row. HELD: the row fits the registers of runs on their
// way, and is looked through again there.
template<class T, int N, int WAVES, int AHEAD, bool HELD, bool PAST>
__global__ __launch_bounds__(64 * WAVES) void LogProbsKernel(const LogProbsArgs a)
{
    constexpr int       kLanes = 64 * WAVES;
    __shared__ Sums     s_sums[WAVES];
    __shared__ uint64_t s_key[WAVES];
    __shared__ TopRoom  s_top;
    const uint32_t row  = a.firstRow + blockIdx.x;
    const T       *in   = reinterpret_cast<const T *>(a.logits.at(row));
    const int      runs = (a.columns + N - 1) / N, whole = a.columns / N;
    Running        run;
    Logits<T, N, PAST>   x[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
    {
        x[k].get(in, a.columns, min((int)threadIdx.x + k * kLanes, runs - 1));
    }
    // the token's own logit, on its way beside them
    const int64_t token = TokenAt(a.tokens, a.wide, row);
    const bool    there = token >= 0 && token < a.columns;
    const float   its   = (float)in[there ? token : 0];
    // runs of the wave's lanes from `at` on
    const int lane = (int)(threadIdx.x & 63);
    auto      take = [&](const Logits<T, N, PAST> &l, int at)
    {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            v[i] = (float)l.run.v[i];
        }
        if (at + 64 > whole) // (the row's last run, where it is not a whole one, or none)
        {
            asm volatile(""); // (or the compiler makes what follows for every run, and chooses afterwards)
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                v[i] = at + lane < whole || (i >= l.skip && at + lane < runs) ? v[i] : -INFINITY;
            }
        }
        run.next(v, a.scale, a.slack);
    };
    for (int at = (int)WaveOfGroup() * 64; at < runs; at += AHEAD * kLanes)
    {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
        {
            if (at + k * kLanes < runs)
            {
                take(x[k], at + k * kLanes);
            }
            if (!HELD)
            {
                x[k].get(in, a.columns, min(at + lane + (k + AHEAD) * kLanes, runs - 1));
            }
        }
    }
    Sums sums = run.sums(a.scale);
    if constexpr (WAVES > 1)
    {
        if ((threadIdx.x & 63) == 0)
        {
            s_sums[WaveOfGroup()] = sums;
        }
    }
    if (a.top > 0)
    {
        // groups of WAVES lanes that follow one another
        float g = run.top;
#pragma unroll
        for (int d = 1; d < WAVES; d *= 2)
        {
            g = fmaxf(g, __shfl_xor(g, d));
        }
        if (threadIdx.x % WAVES == 0)
        {
            s_top.group[threadIdx.x / WAVES] = OrderOf(g);
        }
        if (threadIdx.x == 0)
        {
            s_top.count = 0;
        }
    }
    __syncthreads();
    bool sound = sums.r == sums.r; // (the row has neither NaN nor +infinity)
    if constexpr (WAVES > 1)
    {
        const Sums none = {-INFINITY, 0, 0};
        sums            = lane < WAVES ? s_sums[lane] : none;
        sound           = !__any(sums.r != sums.r);
    }
    // (by the first wave, and by all where all need it)
    Total total;
    auto  join = [&]()
    {
        const Sums  all  = WAVES > 1 ? Joined(sums, a.scale) : sums;
        const float base = all.at * a.scale;
        total            = {a.scale, base, __builtin_fmaf(all.at, a.scale, -base), Log1(all.r), all.at == -INFINITY && all.r == 0};
        return all;
    };
    if (threadIdx.x < 64)
    {
        const Sums all = join();
        if (threadIdx.x == 0)
        {
            a.out[row] = there ? total.of(its) : 0.f;
            if (a.entropy != nullptr)
            {
                a.entropy[row] = total.nothing ? 0.f : total.logSum - all.t / (1.f + all.r);
            }
            if (a.lse != nullptr)
            {
                a.lse[row] = total.nothing ? -INFINITY : __builtin_fmaf(all.at, a.scale, total.logSum);
            }
        }
    }
    if (a.top == 0)
    {
        return;
    }
    // A logit that K groups' largest ones reach, and not many more: between the smallest and the largest of them, by halves.
    const uint32_t mine = s_top.group[threadIdx.x & 63];
    uint32_t       low = ~WaveLargest(~mine), high = sound ? WaveLargest(mine) + 1 : low;
    while (high - low > 1)
    {
        const uint32_t middle = low + (high - low) / 2;
        const int      reach  = __popcll(__ballot(mine >= middle));
        reach >= a.top ? low = middle : high = middle;
        if (reach >= a.top && reach < a.top + kFewMore)
        {
            break;
        }
    }
    const float least = ValueOf(low);
    auto        look  = [&](const Logits<T, N, PAST> &l)
    {
        float v[N], largest = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            v[i] = (float)l.run.v[i];
        }
#pragma unroll
        for (int i = 0; i < N; i += 2)
        {
            largest = Largest(largest, v[i], v[std::min(i + 1, N - 1)]);
        }
        if (largest >= least)
        {
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                if (i >= l.skip && v[i] >= least)
                {
                    const uint32_t at = atomicAdd(&s_top.count, 1u);
                    if (at < kCandidates)
                    {
                        s_top.key[at] = KeyOf(v[i], l.from + i);
                    }
                }
            }
        }
    };
    if (run.top >= least && sound)
    {
        if constexpr (HELD)
        {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
            {
                if ((int)threadIdx.x + k * kLanes < runs)
                {
                    look(x[k]);
                }
            }
        }
        else
        {
            for (int r = (int)threadIdx.x; r < runs; r += AHEAD * kLanes)
            {
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                {
                    x[k].get(in, a.columns, min(r + k * kLanes, runs - 1));
                }
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                {
                    if (r + k * kLanes < runs)
                    {
                        look(x[k]);
                    }
                }
            }
        }
    }
    __syncthreads();
    const int count = (int)s_top.count;
    if (sound && count >= a.top && count <= 64)
    {
        if (threadIdx.x < 64)
        {
            const uint64_t key   = (int)threadIdx.x < count ? s_top.key[threadIdx.x] : 0;
            int            above = 0;
            for (int j = 0; j < count; ++j)
            {
                const uint64_t other = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), j) << 32) |
                                       (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)key, j);
                above += other > key ? 1 : 0;
            }
            if ((int)threadIdx.x < count && above < a.top)
            {
                PutTop(a, row, above, key, total);
            }
        }
        return;
    }
    if (sound && count >= a.top && count <= kCandidates)
    {
        if (threadIdx.x >= 64)
        {
            join();
        }
        for (int i = (int)threadIdx.x; i < count; i += kLanes)
        {
            const uint64_t key   = s_top.key[i];
            int            above = 0;
            for (int j = 0; j < count; ++j)
            {
                above += s_top.key[j] > key ? 1 : 0;
            }
            if (above < a.top)
            {
                PutTop(a, row, above, key, total);
            }
        }
        return;
    }
    uint64_t before = ~0ull;
    for (int k = 0; k < a.top; ++k)
    {
        uint64_t best = 0;
        for (int r = (int)threadIdx.x; r < runs; r += kLanes)
        {
            Logits<T, N, PAST> l;
            l.get(in, a.columns, r);
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                const uint64_t key = KeyOf((float)l.run.v[i], l.from + i);
                best               = key < before && key > best ? key : best;
            }
        }
        before = LargestKey<WAVES>(best, s_key);
        if (threadIdx.x == 0)
        {
            PutTop(a, row, k, before, total);
        }
    }
}

struct LogProbsGradArgs
{
    RowPlaces    logits, out;
    const void  *tokens;
    const float *lse, *entropy, *grad, *gradEntropy; // gradEntropy: nullptr for none
    float        scale;
    int32_t      rows, columns;
    DivBy        parts; // workgroups of a row
    bool         wide;
};

constexpr int kGradThreads = 256;

// A run of a row to a lane (4096 rows of 128000 BF16 320 us, 6.6 TB/s; with two runs 332).
template<class T, int N, bool ENTROPY, bool PAST>
__global__ __launch_bounds__(kGradThreads) void LogProbsGradKernel(const LogProbsGradArgs a, uint32_t firstBlock)
{
    const uint32_t block = firstBlock + blockIdx.x, row = a.parts.Quotient(block), part = block - row * a.parts.d;
    const T       *in    = reinterpret_cast<const T *>(a.logits.at(row));
    T             *out   = reinterpret_cast<T *>(a.out.at(row));
    const int      runs = (a.columns + N - 1) / N, r = (int)(part * kGradThreads + threadIdx.x);
    Logits<T, N, PAST>   x;
    x.get(in, a.columns, min(r, runs - 1));
    const int64_t token   = TokenAt(a.tokens, a.wide, row);
    const bool    there   = token >= 0 && token < a.columns;
    const float   lse     = a.lse[row], g = there ? a.grad[row] : 0.f, h = ENTROPY ? a.gradEntropy[row] : 0.f;
    const float   entropy = ENTROPY ? a.entropy[row] : 0.f;
    const bool    nothing = lse == -INFINITY;
    if (r >= runs)
    {
        return;
    }
    Run<T, N> made;
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
        const float logp = a.scale * (float)x.run.v[i] - lse, p = __builtin_amdgcn_exp2f(logp * kLog2E);
        float       v = -g * p;
        if (ENTROPY)
        {
            v -= p == 0 ? 0.f : h * p * (logp + entropy);
        }
        v += there && x.from + i == (int)token ? g : 0.f;
        made.v[i] = FromFloat<T>(nothing ? 0.f : a.scale * v);
    }
    if (x.skip == 0)
    {
        StoreRun<PAST>(out + x.from, made);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            if (i >= x.skip)
            {
                out[x.from + i] = made.v[i];
            }
        }
    }
}

// runs of a lane on their way (4096 rows of 128000 BF16, eight waves: with two 264 us, four 249, six 250, eight 262)
constexpr int kAhead = 4;

template<class T, int N, int WAVES, bool PAST>
void LaunchRows(LogProbsArgs a, hipStream_t stream)
{
    constexpr int most = INT32_MAX / (64 * WAVES);
    const bool    held = a.columns <= kAhead * 64 * WAVES * N;
    for (int64_t first = 0; first < a.rows; first += most)
    {
        const uint32_t blocks = (uint32_t)std::min<int64_t>(most, a.rows - first);
        a.firstRow            = (int32_t)first;
        if (held)
        {
            LogProbsKernel<T, N, WAVES, kAhead, true, PAST><<<blocks, 64 * WAVES, 0, stream>>>(a);
        }
        else
        {
            LogProbsKernel<T, N, WAVES, kAhead, false, PAST><<<blocks, 64 * WAVES, 0, stream>>>(a);
        }
        CheckLaunch("log probabilities");
    }
}

template<class T, int N, bool PAST>
void LaunchLogProbs(const LogProbsArgs &a, hipStream_t stream)
{
    if constexpr (N == 1)
    {
        LaunchRows<T, N, 1, PAST>(a, stream);
    }
    else
    {
        // Where rows fill the card, waves of 8 runs to a lane and more, so that joining lanes is little beside them: 20000 rows of 4000
        // BF16 with the top 20 59 us with one wave, 82 with two; 2600 of 32000 45 with eight, 92 with sixteen; 1300 of 64000 46 and 49, 660 of
        // 128000 48 and 44. Where there are fewer, more waves, until there are 4096: 64 rows of 2000 8.3 us with one, 6.5 with four; of 16000
        // 10.3 with four, 8.5 with eight; of 64000 15.1 with eight, 12.7 with sixteen. A row of more than
        // 32 runs has more than 32 groups of lanes with logits in all of them: with fewer than top tokens the whole row would be gone over.
        const int runs = (a.columns + N - 1) / N;
        const int many = runs <= 512 ? 1 : runs <= 1024 ? 2 : runs <= 2048 ? 4 : runs <= 8192 ? 8 : 16;
        const int few  = runs <= 64 ? 1 : runs <= 128 ? 2 : runs <= 512 ? 4 : runs <= 2048 ? 8 : 16;
        switch (std::max(many, std::min(few, 4096 / a.rows)))
        {
        case 0:
        case 1: LaunchRows<T, N, 1, PAST>(a, stream); break;
        case 2:
        case 3: LaunchRows<T, N, 2, PAST>(a, stream); break;
        case 4:
        case 5:
        case 6:
        case 7: LaunchRows<T, N, 4, PAST>(a, stream); break;
        case 16: LaunchRows<T, N, 16, PAST>(a, stream); break;
        default: LaunchRows<T, N, 8, PAST>(a, stream); break;
        }
    }
}

template<class T, int N, bool ENTROPY, bool PAST>
void LaunchLogProbsGrad(const LogProbsGradArgs &a, hipStream_t stream)
{
    const int64_t blocks = (int64_t)a.rows * a.parts.d, most = INT32_MAX / kGradThreads;
    if (blocks > INT32_MAX)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Logits have too many elements");
    }
    for (int64_t first = 0; first < blocks; first += most)
    {
        LogProbsGradKernel<T, N, ENTROPY, PAST><<<(uint32_t)std::min(most, blocks - first), kGradThreads, 0, stream>>>(a, (uint32_t)first);
        CheckLaunch("log probabilities' gradient");
    }
}

template<class F>
void Dispatch(RowElem elem, F &&f)
{
    elem == kRowF32 ? f(float{}) : elem == kRowF16 ? f(Half{}) : f(Bf16{});
}

RowsView TakeLogits(NVCVTensorHandle h, const char *what)
{
    const RowsView v = RequireRows(h, what);
    if (v.columns < 1 && v.rows > 0)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have rows of at least one element", what);
    }
    return v;
}

// A tensor of `count` elements; nullptr where there is none and it may be left out.
float *TakeFloats(NVCVTensorHandle h, const char *what, int64_t count, bool optional)
{
    if (h == nullptr && optional)
    {
        return nullptr;
    }
    const DenseView v = RequireDense(h, what, NVCV_DATA_TYPE_F32);
    if (v.count != count)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "%s must have %ld elements, not %ld", what, (long)count, (long)v.count);
    }
    return reinterpret_cast<float *>(v.base);
}

DenseView TakeTokens(NVCVTensorHandle h, int64_t count)
{
    const DenseView v = RequireDense(h, "Tokens", NVCV_DATA_TYPE_NONE);
    if (v.dtype != NVCV_DATA_TYPE_S32 && v.dtype != NVCV_DATA_TYPE_S64)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tokens must hold S32 or S64 values");
    }
    if (v.count != count)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tokens must have one element for each of %ld rows, not %ld", (long)count, (long)v.count);
    }
    return v;
}

void RequireScale(float scale)
{
    if (!(scale > 0) || !std::isfinite(scale))
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Scale must be finite and positive, not %g", (double)scale);
    }
}

class LogProbs final : public IOperator
{
public:
    static void submit(hipStream_t stream, NVCVTensorHandle hlogits, NVCVTensorHandle htokens, NVCVTensorHandle hout, NVCVTensorHandle hentropy,
                       NVCVTensorHandle hlse, NVCVTensorHandle htopValues, NVCVTensorHandle htopTokens, float scale)
    {
        const RowsView  logits = TakeLogits(hlogits, "Logits");
        const DenseView tokens = TakeTokens(htokens, logits.rows);
        float          *out = TakeFloats(hout, "Output", logits.rows, false), *entropy = TakeFloats(hentropy, "Entropy", logits.rows, true);
        float          *lse = TakeFloats(hlse, "Lse", logits.rows, true), *topValues = nullptr;
        int32_t        *topTokens = nullptr;
        int64_t         top       = 0;
        RequireScale(scale);
        if ((htopValues == nullptr) != (htopTokens == nullptr))
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Top values and top tokens go together");
        }
        if (htopTokens != nullptr && logits.rows > 0)
        {
            const DenseView v = RequireDense(htopTokens, "Top tokens", NVCV_DATA_TYPE_S32);
            top               = v.count / logits.rows;
            if (top < 1 || top > CVCUDAX_LOG_PROBS_MOST_TOP || top > logits.columns || v.count % logits.rows != 0)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Top tokens must have 1 to %d elements for each of %d rows of %d logits, not %ld in all",
                              CVCUDAX_LOG_PROBS_MOST_TOP, logits.rows, logits.columns, (long)v.count);
            }
            topTokens = reinterpret_cast<int32_t *>(v.base);
            topValues = TakeFloats(htopValues, "Top values", v.count, false);
        }
        if (logits.rows == 0)
        {
            return;
        }
        const LogProbsArgs a = {RowPlaces(logits), tokens.base, out, entropy, lse, topValues, topTokens, scale, kSlack / scale, logits.rows, logits.columns,
                                (int32_t)top, 0, tokens.dtype == NVCV_DATA_TYPE_S64};
        Dispatch(logits.elem,
                 [&](auto t)
                 {
                     using T = decltype(t);
                     logits.columns < kRunOf<T>                                                         ? LaunchLogProbs<T, 1, false>(a, stream)
                     : MovesPastCaches((int64_t)logits.rows * logits.columns * (int64_t)sizeof(T)) ? LaunchLogProbs<T, kRunOf<T>, true>(a, stream)
                                                                                                        : LaunchLogProbs<T, kRunOf<T>, false>(a, stream);
                 });
    }

    static void submitGrad(hipStream_t stream, NVCVTensorHandle hlogits, NVCVTensorHandle htokens, NVCVTensorHandle hlse, NVCVTensorHandle hentropy,
                           NVCVTensorHandle hgrad, NVCVTensorHandle hgradEntropy, NVCVTensorHandle hout, float scale)
    {
        const RowsView logits = TakeLogits(hlogits, "Logits"), out = TakeLogits(hout, "Logits' gradient");
        if (out.elem != logits.elem || out.rows != logits.rows || out.columns != logits.columns)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Logits' gradient must have the type and shape of the logits");
        }
        const DenseView tokens = TakeTokens(htokens, logits.rows);
        const float    *lse = TakeFloats(hlse, "Lse", logits.rows, false), *grad = TakeFloats(hgrad, "Output's gradient", logits.rows, false);
        const float    *gradEntropy = TakeFloats(hgradEntropy, "Entropy's gradient", logits.rows, true);
        const float    *entropy     = TakeFloats(hentropy, "Entropy", logits.rows, gradEntropy == nullptr);
        RequireScale(scale);
        if (logits.rows == 0)
        {
            return;
        }
        Dispatch(logits.elem,
                 [&](auto t)
                 {
                     using T              = decltype(t);
                     const auto run       = [&](auto n, auto past)
                     {
                         constexpr int          N     = decltype(n)::value;
                         constexpr bool         PAST  = decltype(past)::value;
                         const int64_t          parts = ((int64_t)logits.columns + N * kGradThreads - 1) / (N * kGradThreads);
                         const LogProbsGradArgs a     = {RowPlaces(logits), RowPlaces(out), tokens.base, lse, entropy, grad, gradEntropy, scale,
                                                         logits.rows, logits.columns, DivBy((uint32_t)parts), tokens.dtype == NVCV_DATA_TYPE_S64};
                         gradEntropy != nullptr ? LaunchLogProbsGrad<T, N, true, PAST>(a, stream) : LaunchLogProbsGrad<T, N, false, PAST>(a, stream);
                     };
                     const std::integral_constant<int, kRunOf<T>> whole;
                     logits.columns < kRunOf<T> ? run(std::integral_constant<int, 1>(), std::false_type())
                     : MovesPastCaches(2 * (int64_t)logits.rows * logits.columns * (int64_t)sizeof(T)) ? run(whole, std::true_type())
                                                                                                       : run(whole, std::false_type());
                 });
    }
};

} // namespace
} // namespace cvamd

using namespace cvamd;

extern "C"
{
CVCUDA_PUBLIC NVCVStatus cvcudaxLogProbsCreate(NVCVOperatorHandle *handle)
{
    return CreateOperator<LogProbs>(handle);
}

CVCUDA_PUBLIC NVCVStatus cvcudaxLogProbsSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle logits,
                                               NVCVTensorHandle tokens, NVCVTensorHandle out, NVCVTensorHandle entropy,
                                               NVCVTensorHandle lse, NVCVTensorHandle topValues, NVCVTensorHandle topTokens,
                                               float scale)
{
    return Protect(
        [&]
        {
            (void)ToOperator<LogProbs>(handle);
            LogProbs::submit(stream, logits, tokens, out, entropy, lse, topValues, topTokens, scale);
        });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxLogProbsGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle logits,
                                                   NVCVTensorHandle tokens, NVCVTensorHandle lse, NVCVTensorHandle entropy,
                                                   NVCVTensorHandle gradOut, NVCVTensorHandle gradEntropy,
                                                   NVCVTensorHandle gradLogits, float scale)
{
    return Protect(
        [&]
        {
            (void)ToOperator<LogProbs>(handle);
            LogProbs::submitGrad(stream, logits, tokens, lse, entropy, gradOut, gradEntropy, gradLogits, scale);
        });
}
}
