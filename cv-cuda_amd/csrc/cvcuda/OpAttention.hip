// Attention over packed sequences (formulas: cvcuda/Attention.h; tiles and products: AttentionTiles.hpp).
//
// One pass over the keys, with the running maximum and sum of a softmax: a tile's scores live in registers from one product to the next. The
// rows that a key head serves (all heads of its group, token by token) are one matrix, so that its keys and values are read once for
// them, whatever the group.
//
// Measured: long prompts (8 sequences of up to 4096 tokens, 32 heads on 8 key heads of 128 BF16 elements, causal) 272 us, 967 TFLOP/s, where a
// product of two 8192 x 8192 matrices by the library has 1253: exponentials take as long as the products, and overlap those of other waves
// only. Single tokens (16 before caches of up to 8192, the same heads: 362 MB) 70 us, of them 65 of reading at 5.6 TB/s.
#include "AttentionTiles.hpp"

#include <cvcuda/Attention.h>

#include <algorithm>
#include <cmath>

namespace cvamd {

namespace {

struct AttentionArgs
{
    const uint8_t     *q, *k, *v;
    uint8_t           *out;
    int64_t            qToken, qHead, kToken, kHead, vToken, vHead, outToken, outHead;
    AttentionSequences sequences;
    float             *lse;                  // nullptr: not wanted
    float             *partial, *partialLse; // [splits][heads][rows][dims], [splits][heads][rows]: where keys are split
    GroupRows          rows;                 // of a key head
    DivBy              keyHeads;
    int32_t            heads, dims, splits, chunkKeys;
    uint32_t           tiles;
    float              scale; // to the base 2
    bool               causal;

    // in lse
    __device__ __forceinline__ int64_t number(const AttentionRow &row) const
    {
        return (int64_t)row.head * sequences.rows + row.token;
    }
};

// A lane's row on its way through the keys: a score to the base 2, near the largest so far, that exponentials are taken relative to, the sum of its
// own keys' exponentials (the other half wave has the other keys') and the weighted values.
template<class T, int DP>
struct Running
{
    float top = -INFINITY, sum = 0;
    Acc16 out[DP / 32] = {};

    // KEYS / 32 products of scores; values: tile of KEYS rows in LDS.
    template<int KEYS>
    __device__ __forceinline__ void add(Acc16 (&scores)[KEYS / 32], const uint8_t *values, float scale)
    {
        float largest = -INFINITY;
#pragma unroll
        for (int k = 0; k < KEYS / 32; ++k)
        {
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                largest = fmaxf(largest, scores[k][i]); // (a NaN is left out here, and reaches the sums below)
            }
        }
        largest = BothMax(largest) * scale;
        // Sums are rescaled when the largest score has grown by more than kSlack: among 32 rows some largest score grows in nearly every
        // tile, by little (long prompts 303 us with every growth, 290).
        if (__any(largest > top + kSlack))
        {
            largest          = fmaxf(top, largest);
            const float less = largest > top ? __builtin_amdgcn_exp2f(top - largest) : 1.f; // (0 for the first)
            sum *= less;
#pragma unroll
            for (int p = 0; p < DP / 32; ++p)
            {
                out[p] *= less;
            }
            top = largest;
        }
        const float shift = kExpShift<T> - (top == -INFINITY ? 0.f : top);
#pragma unroll
        for (int k = 0; k < KEYS / 32; ++k)
        {
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                scores[k][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(scores[k][i], scale, shift));
                sum += scores[k][i];
            }
#pragma unroll
            for (int half = 0; half < 2; ++half)
            {
                const Vec8<T> shares = RoundedHalf<T>(scores[k], half);
#pragma unroll
                for (int p = 0; p < DP / 32; ++p)
                {
                    Multiply(out[p], ColumnsOperand<T, DP>(values, 32 * k + 16 * half, p), shares);
                }
            }
        }
    }
};

// Scores of 32 * N keys, keys that a row does not see as -infinity.
template<class T, int DP, int N>
__device__ __forceinline__ void Scores(Acc16 (&scores)[N], const uint8_t *keys, const Vec8<T> (&q)[DP / 16], int firstKey, int limit, bool hide)
{
#pragma unroll
    for (int k = 0; k < N; ++k)
    {
        scores[k] = {};
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
        {
            Multiply(scores[k], RowsOperand<T, DP>(keys, 32 * k, s), q[s]);
        }
    }
    if (hide)
    {
        KeepBranch();
#pragma unroll
        for (int k = 0; k < N; ++k)
        {
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                scores[k][i] = firstKey + 32 * k + RowOf(i) <= limit ? scores[k][i] : -INFINITY;
            }
        }
    }
}

// Numbers 32 * part on of a row's weighted values from keys firstKey to behindKey, `step` of them after the other, made from memory, those
// that the row doesn't see left out.
template<class T, int DP>
__device__ __forceinline__ Acc16 SeenPart(const AttentionArgs &a, const Vec8<T> (&q)[DP / 16], const uint8_t *k, const uint8_t *v, int firstKey,
                                          int behindKey, int step, int keys, int limit, float top, int part)
{
    const float shift = kExpShift<T> - (top == -INFINITY ? 0.f : top);
    Acc16       out   = {};
    const int   lane  = (int)Again(threadIdx.x) & 63;
    for (int key = firstKey; key < behindKey; key += step)
    {
        Acc16 scores = {};
        MultiplyRows<T, DP>(scores, k + min(key + (lane & 31), keys - 1) * a.kToken, a.dims, [&](int s) { return q[s]; });
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            scores[i] = key + RowOf(i, lane) <= limit ? __builtin_amdgcn_exp2f(__builtin_fmaf(scores[i], a.scale, shift)) : 0.f;
        }
        MultiplySeen<T>(out, scores, part, a.dims, keys - key, !__any(key + 31 > limit),
                        [&](int n) { return v + (key + n) * a.vToken; }, [&](int n) { return key + n <= limit; });
    }
    return out;
}

// What a row has at the end: lse to the base 2.
template<class T>
__device__ __forceinline__ float LseOf(float top, float sum)
{
    return sum == 0 ? -INFINITY : top + (__builtin_amdgcn_logf(sum) - kExpShift<T>);
}

// ---- prompts: 128 rows to a workgroup, 32 to a wave ------------------------------------------------------------------
constexpr int kManyRows = 128, kManyThreads = 256;

// Keys of a tile, and waves to a SIMD. With heads of 128 elements three waves with tiles of 32 keys hide more of each other's waits than
// two with 64 do (long prompts 290 us, 276); with 64 elements four waves have registers for 64 keys.
template<int DP>
constexpr int kManyKeys = DP > 64 ? 32 : 64;
template<int DP>
constexpr int kManyWaves = DP > 64 ? 3 : 4;

// (CAUSAL: calls of the other kind hide nothing, and their kernels need fewer registers without what that takes: pairs 21.6 us, with one kernel for
// both 21.9, their gradient 69.4 and 73.)
template<class T, int DP, bool CAUSAL>
__global__ __launch_bounds__(kManyThreads, kManyWaves<DP>) void AttentionKernel(const AttentionArgs a)
{
    constexpr int kKeys = kManyKeys<DP>;
    __shared__ __attribute__((aligned(256))) uint8_t s_k0[kKeys * DP * 2], s_k1[kKeys * DP * 2];
    __shared__ __attribute__((aligned(256))) uint8_t s_v0[kKeys * DP * 2], s_v1[kKeys * DP * 2];
    const uint32_t     t       = a.keyHeads.Quotient(blockIdx.x);
    const int          keyHead = (int)(blockIdx.x - t * a.keyHeads.d);
    const SequenceTile s       = FindTile(a.sequences, t, a.tiles, kManyRows, a.rows.size(), false, CAUSAL);
    if (s.tile < 0)
    {
        return;
    }
    const uint32_t wave = WaveOfGroup();
    const int  first = s.tile * kManyRows, ownFirst = first + (int)wave * 32, all = s.rows * a.rows.size();
    const AttentionRow row(a.rows, CAUSAL, s, keyHead, ownFirst + (int)(threadIdx.x & 31));
    // keys of the tile, of the wave and those that all of the wave's rows see; this workgroup's part of the tile's
    auto       limitAt  = [&](int r) { return LimitOf(CAUSAL, s, a.rows.token(min(r, all - 1))); };
    const int  tileKeys = max(limitAt(first + kManyRows - 1) + 1, 0), waveKeys = ownFirst < all ? limitAt(ownFirst + 31) + 1 : 0;
    const int  seenKeys = limitAt(ownFirst) + 1;
    const int  parts    = (tileKeys + kKeys - 1) / kKeys;
    const int  from = (int)((int64_t)parts * blockIdx.y / a.splits), to = (int)((int64_t)parts * (blockIdx.y + 1) / a.splits);
    const uint8_t *k = a.k + s.firstKey * a.kToken + keyHead * a.kHead, *v = a.v + s.firstKey * a.vToken + keyHead * a.vHead;

    using Copy = TileCopy<kKeys, DP, kManyThreads / 64>;
    auto load  = [&](int part, uint8_t *toK, uint8_t *toV)
    {
        const int key = part * kKeys;
        Copy::rows(wave, toK, k + key * a.kToken, (uint32_t)a.kToken, s.keys - key, a.dims);
        Copy::rows(wave, toV, v + key * a.vToken, (uint32_t)a.vToken, s.keys - key, a.dims);
    };
    if (from < to)
    {
        load(from, s_k0, s_v0);
    }
    Vec8<T> q[DP / 16];
    LoadColumn<T, DP>(q, a.q + row.token * a.qToken + row.head * a.qHead, a.dims);
    Running<T, DP> run;
    auto           take = [&](int part, const uint8_t *fromK, const uint8_t *fromV, uint8_t *nextK, uint8_t *nextV)
    {
        const int key = part * kKeys;
        CopiesAndBarrier(); // (all have done the part before: its place may be written over)
        if (part + 1 < to)
        {
            load(part + 1, nextK, nextV);
        }
        if (key < waveKeys)
        {
            Acc16 scores[kKeys / 32];
            Scores<T, DP>(scores, fromK, q, key, row.limit, key + kKeys > seenKeys);
            run.template add<kKeys>(scores, fromV, a.scale);
        }
    };
    // (by turns of their own, so that the compiler sees that what is read is not what is on its way)
    for (int part = from; part < to; part += 2)
    {
        take(part, s_k0, s_v0, s_k1, s_v1);
        if (part + 1 < to)
        {
            take(part + 1, s_k1, s_v1, s_k0, s_v0);
        }
    }
    const float   sum = BothSum(run.sum), factor = sum == 0 ? 0.f : 1.f / sum;
    const float   lse = LseOf<T>(run.top, sum);
    // 32 numbers of the results, from 32 * part on
    auto store = [&](int part, const Acc16 &made, const AttentionRow &its)
    {
        if (a.splits == 1)
        {
            StoreColumnPart<T>(made, part, factor, a.out + its.token * a.outToken + its.head * a.outHead, its.there, a.dims);
        }
        else
        {
            const int64_t at = (int64_t)blockIdx.y * a.heads * a.sequences.rows + a.number(its);
            StorePiecePart(made, part, factor, a.partial + at * a.dims, its.there, a.dims);
        }
    };
    const AttentionRow its(a.rows, CAUSAL, s, keyHead, ownFirst + (int)(Again(threadIdx.x) & 31));
    if (its.there && (threadIdx.x & 32) == 0)
    {
        const int64_t number = a.number(its);
        if (a.splits > 1)
        {
            a.partialLse[(int64_t)blockIdx.y * a.heads * a.sequences.rows + number] = lse;
        }
        else if (a.lse != nullptr)
        {
            a.lse[number] = lse * kLn2;
        }
    }
    auto hidden = [&](int n) { return v + (max(seenKeys, 0) + n) * a.vToken; };
    if (CAUSAL && AnyNotFinite(run.out) &&
        RowsNotFinite<T>(a.dims, min((waveKeys + kKeys - 1) / kKeys * kKeys, s.keys) - max(seenKeys, 0), hidden))
    {
        const AttentionRow again(a.rows, CAUSAL, s, keyHead, ownFirst + (int)(Again(threadIdx.x) & 31));
        LoadColumn<T, DP>(q, a.q + again.token * a.qToken + again.head * a.qHead, a.dims, Again(threadIdx.x));
        for (int part = 0; part * 32 < a.dims; ++part)
        {
            store(part, SeenPart<T, DP>(a, q, k, v, from * kKeys, min(to * kKeys, waveKeys), 32, s.keys, again.limit, run.top, part), again);
        }
        return;
    }
#pragma unroll
    for (int p = 0; p < DP / 32; ++p)
    {
        store(p, run.out[p], its);
    }
}

// ---- few rows to a sequence (single tokens): 32 rows to a workgroup, of whose waves each takes every fourth 32 keys -------------
// Bound by the reads of keys and values: 16 caches of up to 8192 keys, 362 MB, in 65 us, and 5.6 to join the pieces (75 where the caches are to keep them). (Eight waves are slower:
// 700 keys 13.1 us, 11.6 with four.)
constexpr int kFewRows = 32, kFewKeys = 32, kFewWaves = 4, kFewThreads = 64 * kFewWaves;

template<class T, int DP, bool PAST>
__global__ __launch_bounds__(kFewThreads, DP > 64 ? 2 : 4) void AttentionFewKernel(const AttentionArgs a)
{
    // each wave's keys and values, later its weighted values in 32 bits
    __shared__ __attribute__((aligned(256))) uint8_t s_tile[kFewWaves][2 * kFewKeys * DP * 2];
    __shared__ float                                 s_top[kFewWaves][kFewRows], s_sum[kFewWaves][kFewRows];
    // (a sequence's key heads next to each other on one XCD: what they read lies side by side. 88 us with one of eight heads to each XCD, 85)
    const int          keyHead = (int)(blockIdx.x / a.tiles);
    const uint32_t     t       = blockIdx.x - (uint32_t)keyHead * a.tiles;
    const SequenceTile s       = FindTile(a.sequences, t, a.tiles, kFewRows, a.rows.size(), false, false);
    if (s.tile < 0)
    {
        return;
    }
    const uint32_t lane = threadIdx.x & 63, wave = WaveOfGroup();
    const int      first = s.tile * kFewRows, all = s.rows * a.rows.size();
    const AttentionRow row(a.rows, a.causal, s, keyHead, first + (int)(lane & 31));
    auto           limitAt  = [&](int r) { return LimitOf(a.causal, s, a.rows.token(min(r, all - 1))); };
    const int      tileKeys = max(limitAt(first + kFewRows - 1) + 1, 0), seenKeys = limitAt(first) + 1;
    const int      parts    = (tileKeys + kFewKeys - 1) / kFewKeys;
    // its keys in as many pieces as have chunkKeys of them, all of about one length; the call's other pieces are empty
    const int      pieces = min((max(tileKeys, 1) - 1) / a.chunkKeys + 1, a.splits), piece = (int)blockIdx.y;
    const int      from = piece < pieces ? (int)((int64_t)parts * piece / pieces) + (int)wave : 0;
    const int      to   = piece < pieces ? (int)((int64_t)parts * (piece + 1) / pieces) : 0;
    const uint8_t *k = a.k + s.firstKey * a.kToken + keyHead * a.kHead, *v = a.v + s.firstKey * a.vToken + keyHead * a.vHead;
    uint8_t       *keys = s_tile[wave], *values = keys + kFewKeys * DP * 2;

    TileLoad<kFewKeys, DP> nextK, nextV;
    auto load = [&](int part)
    {
        const int key = part * kFewKeys;
        nextK.template get<PAST>(k + key * a.kToken, (uint32_t)a.kToken, s.keys - key, a.dims);
        nextV.template get<PAST>(v + key * a.vToken, (uint32_t)a.vToken, s.keys - key, a.dims);
    };
    if (from < to)
    {
        load(from);
    }
    Vec8<T> q[DP / 16];
    LoadColumn<T, DP>(q, a.q + row.token * a.qToken + row.head * a.qHead, a.dims);
    Running<T, DP> run;
    for (int part = from; part < to; part += kFewWaves)
    {
        const int key = part * kFewKeys;
        // (a wave's reads and writes of LDS take place in their order; the compiler is kept from changing it)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        nextK.put(keys);
        nextV.put(values);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (part + kFewWaves < to)
        {
            load(part + kFewWaves);
        }
        Acc16 scores[1];
        Scores<T, DP>(scores, keys, q, key, row.limit, key + kFewKeys > seenKeys);
        run.template add<kFewKeys>(scores, values, a.scale);
    }
    // the waves' results joined: thread l has row l % 32, an eighth of its elements
    const float sum = BothSum(run.sum);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float *own = reinterpret_cast<float *>(s_tile[wave]); // [DP][32]
    auto   put = [&](const Acc16 &made, int part)
    {
#pragma unroll
        for (int i = 0; i < 16; ++i)
        {
            own[(32 * part + RowOf(i)) * kFewRows + (lane & 31)] = made[i];
        }
    };
    auto hidden = [&](int n) { return v + (max(seenKeys, 0) + n) * a.vToken; };
    if (a.causal && AnyNotFinite(run.out) && RowsNotFinite<T>(a.dims, min(parts * kFewKeys, s.keys) - max(seenKeys, 0), hidden))
    {
        const AttentionRow again(a.rows, a.causal, s, keyHead, first + (int)(Again(threadIdx.x) & 31));
        LoadColumn<T, DP>(q, a.q + again.token * a.qToken + again.head * a.qHead, a.dims, Again(threadIdx.x));
        for (int part = 0; part * 32 < a.dims; ++part)
        {
            put(SeenPart<T, DP>(a, q, k, v, from * kFewKeys, to * kFewKeys, kFewWaves * kFewKeys, s.keys, again.limit, run.top, part), part);
        }
    }
    else
    {
#pragma unroll
        for (int p = 0; p < DP / 32; ++p)
        {
            put(run.out[p], p);
        }
    }
    if (lane < 32)
    {
        s_top[wave][lane] = run.top;
        s_sum[wave][lane] = sum;
    }
    __syncthreads();
    const uint32_t r = threadIdx.x % kFewRows, d0 = threadIdx.x / kFewRows * (DP / 8);
    float          top = -INFINITY, total = 0, weight[kFewWaves];
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w)
    {
        top = fmaxf(top, s_top[w][r]);
    }
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w)
    {
        weight[w] = s_top[w][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_top[w][r] - top);
        total += weight[w] * s_sum[w][r];
    }
    const float factor = total == 0 ? 0.f : 1.f / total, lse = LseOf<T>(top, total);
    const AttentionRow its(a.rows, a.causal, s, keyHead, first + (int)r);
    const int64_t number = a.number(its), at = (int64_t)blockIdx.y * a.heads * a.sequences.rows + number;
    if (!its.there)
    {
        return;
    }
#pragma unroll
    for (int d = 0; d < DP / 8; d += 8)
    {
        float v8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            v8[i] = 0;
#pragma unroll
            for (int w = 0; w < kFewWaves; ++w)
            {
                v8[i] += weight[w] * reinterpret_cast<const float *>(s_tile[w])[(d0 + d + i) * kFewRows + r];
            }
            v8[i] *= factor;
        }
        const int to8 = (int)d0 + d;
        if (to8 < a.dims)
        {
            if (a.splits == 1)
            {
                Run<T, 8> made;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                {
                    made.v[i] = FromFloat<T>(v8[i]);
                }
                *reinterpret_cast<Run<T, 8> *>(a.out + its.token * a.outToken + its.head * a.outHead + to8 * 2) = made;
            }
            else
            {
                float4 *partial = reinterpret_cast<float4 *>(a.partial + at * a.dims + to8);
                partial[0]      = make_float4(v8[0], v8[1], v8[2], v8[3]);
                partial[1]      = make_float4(v8[4], v8[5], v8[6], v8[7]);
            }
        }
    }
    if (d0 == 0)
    {
        if (a.splits > 1)
        {
            a.partialLse[at] = lse;
        }
        else if (a.lse != nullptr)
        {
            a.lse[number] = lse * kLn2;
        }
    }
}

// The parts of the keys joined: a tile of rows to blockIdx.y's workgroups, 16 lanes to a row, 8 elements to a lane. Tiles are found as they were made:
// rows of no sequence have no parts, and with offsets that go back they may lie anywhere.
constexpr int kJoinThreads = 256, kJoinRows = kJoinThreads / 16, kMostSplits = 64;

template<class T>
__global__ __launch_bounds__(kJoinThreads) void AttentionJoinKernel(const AttentionArgs a, int size)
{
    const int          keyHead = (int)(blockIdx.x / a.tiles);
    const SequenceTile s       = FindTile(a.sequences, blockIdx.x - (uint32_t)keyHead * a.tiles, a.tiles, size, a.rows.size(), false, false);
    if (s.tile < 0)
    {
        return;
    }
    const AttentionRow row(a.rows, false, s, keyHead, s.tile * size + (int)(blockIdx.y * kJoinRows + threadIdx.x / 16));
    if (!row.there)
    {
        return;
    }
    const int64_t rows = (int64_t)a.heads * a.sequences.rows, number = a.number(row);
    const int     d    = (int)(threadIdx.x % 16) * 8;
    // lane l of the row has the lse of its pieces l, l + 16 ...
    float lse[kMostSplits / 16], top = -INFINITY, total = 0, out[8] = {};
#pragma unroll
    for (int i = 0; i < kMostSplits / 16; ++i)
    {
        const int p = (int)(threadIdx.x % 16) + 16 * i;
        lse[i]      = p < a.splits ? a.partialLse[p * rows + number] : -INFINITY;
        top         = fmaxf(top, lse[i]);
    }
#pragma unroll
    for (int n = 1; n < 16; n *= 2)
    {
        top = fmaxf(top, __shfl_xor(top, n));
    }
#pragma unroll
    for (int i = 0; i < kMostSplits / 16; ++i)
    {
        const float weight = lse[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lse[i] - top);
        for (int l = 0; l < 16 && 16 * i + l < a.splits; l += 4)
        {
            // (pieces that are empty hold anything)
            float4 part[4][2];
#pragma unroll
            for (int n = 0; n < 4; ++n)
            {
                const float4 *from = reinterpret_cast<const float4 *>(a.partial + (min(16 * i + l + n, a.splits - 1) * rows + number) * a.dims + min(d, a.dims - 8));
                part[n][0] = from[0], part[n][1] = from[1];
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
            {
                const float w = __shfl(weight, l + n, 16);
                if (w != 0)
                {
                    const float v[8] = {part[n][0].x, part[n][0].y, part[n][0].z, part[n][0].w, part[n][1].x, part[n][1].y, part[n][1].z, part[n][1].w};
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                    {
                        out[k] += w * v[k];
                    }
                    total += w;
                }
            }
        }
    }
    if (d >= a.dims)
    {
        return;
    }
    const float factor = total == 0 ? 0.f : 1.f / total;
    Run<T, 8>   made;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        made.v[i] = FromFloat<T>(out[i] * factor);
    }
    *reinterpret_cast<Run<T, 8> *>(a.out + row.token * a.outToken + row.head * a.outHead + d * 2) = made;
    if (d == 0 && a.lse != nullptr)
    {
        a.lse[number] = total == 0 ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
    }
}

// How a call is made, by its sizes alone: the sequences' lengths are on the device.
struct Plan
{
    bool     few;
    int32_t  splits, chunkKeys; // pieces of a sequence's keys at most, and keys of one where there are few rows
    uint32_t tiles;             // at most, of a key head

    Plan(int64_t rows, int64_t keys, int64_t sequences, int64_t heads, int64_t keyHeads)
    {
        const int64_t matrix = rows * (heads / keyHeads), most = std::max<int64_t>(sequences, 1);
        // (4 sequences of 16 rows of a key head that see 1500 keys 14.8 us here, 15.8 where there are many; of 32 rows 21.5 and 16.3; 64 sequences
        // of 48 rows 120 and 73)
        few                = matrix <= 16 * most;
        const int64_t size = few ? kFewRows : kManyRows, whole = (matrix + size - 1) / size;
        tiles              = (uint32_t)(whole + std::min(sequences, rows));
        const int64_t groups = std::max<int64_t>(std::max(whole, std::min(sequences, rows)) * keyHeads, 1), each = keys / most;
        if (few)
        {
            // Pieces of one length whatever the sequences' lengths, so that no workgroup has much more to do than the others, and as many as
            // the card holds at once where all caches are full (single tokens 83 us, with twice as many 85, with four times 101), of 512
            // keys at least (8000 keys 21 us, with 256 at least 29). Up to 1024 keys are not worth the second launch that joins pieces.
            const int64_t chunk = std::max<int64_t>(groups * each / 512, 512);
            splits    = each <= 1024 ? 1 : (int32_t)std::max<int64_t>(std::min<int64_t>((2 * each + chunk - 1) / chunk, kMostSplits), 1);
            chunkKeys = (int32_t)std::min<int64_t>(chunk, INT32_MAX / 2);
        }
        else
        {
            // as many workgroups as fill the card's CUs twice, each with 256 keys at least (128 rows of 8 heads before 2048 keys 17 us, whole 52;
            // before 600 16 and 19)
            splits    = (int32_t)std::max<int64_t>(std::min<int64_t>({512 / groups, each / 256, kMostSplits}), 1);
            chunkKeys = 0;
        }
    }

    int64_t partials(int64_t rows, int64_t heads) const
    {
        return splits > 1 ? splits * rows * heads : 0;
    }

    int64_t bytes(int64_t rows, int64_t heads, int64_t dims) const
    {
        return partials(rows, heads) * (dims + 1) * (int64_t)sizeof(float);
    }
};

template<class T, int DP>
void Launch(const AttentionArgs &a, bool few, hipStream_t stream)
{
    const dim3 grid(a.tiles * a.keyHeads.d, (uint32_t)a.splits);
    if (few && MovesPastCaches(2 * (int64_t)a.sequences.keys * a.keyHeads.d * a.dims * (int64_t)sizeof(T)))
    {
        AttentionFewKernel<T, DP, true><<<grid, kFewThreads, 0, stream>>>(a);
    }
    else if (few)
    {
        AttentionFewKernel<T, DP, false><<<grid, kFewThreads, 0, stream>>>(a);
    }
    else if (a.causal)
    {
        AttentionKernel<T, DP, true><<<grid, kManyThreads, 0, stream>>>(a);
    }
    else
    {
        AttentionKernel<T, DP, false><<<grid, kManyThreads, 0, stream>>>(a);
    }
    CheckLaunch("attention");
    if (a.splits > 1)
    {
        const int size = few ? kFewRows : kManyRows;
        AttentionJoinKernel<T><<<dim3(grid.x, (uint32_t)(size / kJoinRows)), kJoinThreads, 0, stream>>>(a, size);
        CheckLaunch("attention's parts");
    }
}

struct Attention
{
    static void submit(hipStream_t stream, NVCVTensorHandle hq, NVCVTensorHandle hk, NVCVTensorHandle hv, NVCVTensorHandle hoffsets,
                       NVCVTensorHandle hkeyOffsets, NVCVTensorHandle hkeyLengths, NVCVTensorHandle hout, NVCVTensorHandle hlse,
                       NVCVTensorHandle hworkspace, float scale, bool causal)
    {
        const AttentionInputs in  = TakeAttention(hq, hk, hv, hoffsets, hkeyOffsets, hkeyLengths, hlse, true, scale);
        const HeadsView       out = TakeHeadsLike(hout, in.q, "Output");
        const Plan            plan(in.q.tokens, in.k.tokens, in.sequences.count, in.q.heads, in.k.heads);
        uint8_t              *room = RequireWorkspace(hworkspace, plan.bytes(in.q.tokens, in.q.heads, in.q.dims));
        if (in.q.tokens == 0 || in.sequences.count == 0)
        {
            return;
        }
        float              *partial = reinterpret_cast<float *>(room);
        const AttentionArgs a = {in.q.base, in.k.base, in.v.base, out.base, in.q.tokenStride, in.q.headStride, in.k.tokenStride, in.k.headStride,
                                 in.v.tokenStride, in.v.headStride, out.tokenStride, out.headStride, in.sequences, in.lse, partial,
                                 partial + plan.partials(in.q.tokens, in.q.heads) * in.q.dims, {DivBy((uint32_t)(in.q.heads / in.k.heads))},
                                 DivBy((uint32_t)in.k.heads), in.q.heads, in.q.dims, plan.splits, plan.chunkKeys, plan.tiles, scale * kLog2E, causal};
        auto                launch = [&](auto t)
        {
            using T = decltype(t);
            in.q.dims <= 64 ? Launch<T, 64>(a, plan.few, stream) : Launch<T, 128>(a, plan.few, stream);
        };
        in.q.elem == kRowF16 ? launch(Half{}) : launch(Bf16{});
    }
};

} // namespace
} // namespace cvamd

using namespace cvamd;

extern "C"
{
CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionCreate(NVCVOperatorHandle *handle)
{
    return CreateOperator<AttentionOperator>(handle);
}

CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionWorkspace(int64_t rows, int64_t keys, int64_t sequences, int32_t heads,
                                                   int32_t keyHeads, int32_t dims, int64_t *bytes)
{
    return Protect(
        [&]
        {
            if (bytes == nullptr)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Pointer to output must not be NULL");
            }
            RequireAttentionSizes(rows, keys, sequences, heads, keyHeads, dims);
            *bytes = Plan(rows, keys, sequences, heads, keyHeads).bytes(rows, heads, dims);
        });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle q,
                                                NVCVTensorHandle k, NVCVTensorHandle v, NVCVTensorHandle offsets,
                                                NVCVTensorHandle keyOffsets, NVCVTensorHandle keyLengths,
                                                NVCVTensorHandle out, NVCVTensorHandle lse, NVCVTensorHandle workspace,
                                                float scale, int8_t causal)
{
    return Protect(
        [&]
        {
            (void)ToOperator<AttentionOperator>(handle);
            Attention::submit(stream, q, k, v, offsets, keyOffsets, keyLengths, out, lse, workspace, scale, causal != 0);
        });
}
}
