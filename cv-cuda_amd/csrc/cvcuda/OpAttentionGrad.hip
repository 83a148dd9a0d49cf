// The gradient of attention (formulas: cvcuda/Attention.h; tiles and products: AttentionTiles.hpp).
//
// The shares p are made again from the scores and lse. Two kernels: one goes over the keys for 128 rows of queries and sums their gradient, one
// goes over the rows for 128 keys and sums the gradients of keys and values. So the products of scores and of gradOut . v are made
// twice (seven products of a pair where five would do), but every sum stays in the registers of one wave and is made in one
// order: there is nothing to add up by atomics in memory, and no gradient in 32 bits to write and read.
//
// Measured: long sequences (8 of up to 2048 tokens, 32 heads on 8 key heads of 128 BF16 elements, causal) 612 us, seven products at 0.67 of the
// 1253 TFLOP/s of a library's product of two 8192 x 8192 matrices: what bounds it are the phases of products, exponentials and reads of LDS between
// two barriers. Short ones (64 of up to 273 tokens, 12 heads of 64 F16 elements, not causal) 69.7 us, waits of workgroups of four or five tiles.
#include "AttentionTiles.hpp"

#include <cvcuda/Attention.h>

#include <algorithm>
#include <cmath>

namespace cvamd {

namespace {

struct AttentionGradArgs
{
    const uint8_t     *q, *k, *v, *out, *grad;
    uint8_t           *gradQ, *gradK, *gradV;
    int64_t            qToken, qHead, kToken, kHead, vToken, vHead, outToken, outHead, gradToken, gradHead;
    int64_t            gradQToken, gradQHead, gradKToken, gradKHead, gradVToken, gradVHead;
    AttentionSequences sequences;
    const float       *lse;
    float             *base, *delta; // [rows][heads]: ShareBase and gradOut . out
    float             *pieces;       // [pieces][tokens][heads][dims], of keys once more for values: where a kernel's work is split
    GroupRows          rows; // of a key head
    DivBy              keyHeads;
    int32_t            heads, dims;
    uint32_t           tiles, keyTiles;
    int32_t            splits, keySplits; // pieces, at most, of the keys that a row's gradient is summed over, and of the rows for a key's
    float              scale;
    bool               causal;

    // in base and delta
    __device__ __forceinline__ int64_t number(const AttentionRow &row) const
    {
        return (int64_t)row.token * heads + row.head;
    }
};

// Shares, at most 1, are kept in F16 times 2^15: a share of 2^-29 has all of its bits then.
template<class T>
constexpr float kShareShift = std::is_same<T, Half>::value ? 15.f : 0.f;

// What a row's scores are taken relative to: lse to the base 2, less the shift; a row without a key has no share.
template<class T>
__device__ __forceinline__ float ShareBase(float lse)
{
    return lse == -INFINITY ? INFINITY : __builtin_fmaf(lse, kLog2E, -kShareShift<T>);
}

// The larger of a and the magnitudes of b and c.
__device__ __forceinline__ float LargestMagnitude(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// What a column's gradients t of shares are multiplied with before they are rounded to T. In F16 small ones would be lost (its smallest number is
// 2^-24) and large ones are not bounded, so it is a power of two that follows the largest that the column, a row's or a key's, has met: at first one
// that no small t is lost with, and lowered, with the sums so far, where a t passes 2^15, so that the largest is at 2^11 to 2^12 again. What is 2^-25 of
// the largest keeps all of its bits. (Taken from the largest rows of gradOut and v, by a kernel that reads both before, it cost short sequences
// 13 us.)
template<class T>
struct GradScale
{
    static constexpr bool kNeeded = std::is_same<T, Half>::value;

    float factor = kNeeded ? 0x1p60f : 1.f;

    // The products t of a tile, times `factor`, and what goes with them: delta, and the sums so far.
    template<class F>
    __device__ __forceinline__ void fit(Acc16 &t, F &&lower)
    {
        if constexpr (kNeeded)
        {
            float most = 0;
#pragma unroll
            for (int i = 0; i < 16; i += 2)
            {
                most = LargestMagnitude(most, t[i], t[i + 1]);
            }
            if (__any(most > 0x1p15f))
            {
                most                    = BothMax(most); // (the column's other half)
                const uint32_t exponent = __float_as_uint(most) >> 23; // (127: 1 to 2; 255: not finite)
                const float    less     = most > 0x1p15f ? __uint_as_float((127u - min(exponent - (127u + 11u), 100u)) << 23) : 1.f;
                factor *= less;
                t *= less;
                lower(less);
            }
        }
    }
};

// Tiles: rows and keys of a workgroup of the first kernel and its steps, keys and rows of the second's.
constexpr int kGradRows = 128, kGradKeys = 64, kOfKeys = 128, kOfRows = 64;

// Of how many pieces a sum over `all` keys or rows is made, and where piece `n` begins among its tiles: pieces differ by one tile at most.
constexpr int kPiece = 256;

__device__ __forceinline__ int PiecesOf(int all, int most)
{
    return min((max(all, 1) - 1) / kPiece + 1, most);
}

__device__ __forceinline__ int PieceBegin(int tiles, int n, int pieces)
{
    return (int)((int64_t)tiles * n / pieces);
}

// The keys that a tile's rows see, and the first row, of a key head's, that sees one of a tile's keys.
__device__ __forceinline__ int KeysOfTile(const AttentionGradArgs &a, const SequenceTile &s)
{
    const int last = min((s.tile + 1) * kGradRows, s.rows * a.rows.size()) - 1;
    return max(LimitOf(a.causal, s, a.rows.token(last)) + 1, 0);
}

__device__ __forceinline__ int FirstRowOfTile(const AttentionGradArgs &a, const SequenceTile &s)
{
    return a.causal ? min(max(s.tile * kOfKeys - (s.keys - s.rows), 0), s.rows) * a.rows.size() : 0;
}

// ---- the queries' gradient: 128 rows to a workgroup, 32 to a wave --------------------------------------------------------
constexpr int kGradThreads = 256;

template<class T, int DP, bool CAUSAL>
__global__ __launch_bounds__(kGradThreads, 2) void AttentionGradQKernel(const AttentionGradArgs a)
{
    __shared__ __attribute__((aligned(256))) uint8_t s_k0[kGradKeys * DP * 2], s_k1[kGradKeys * DP * 2];
    __shared__ __attribute__((aligned(256))) uint8_t s_v0[kGradKeys * DP * 2], s_v1[kGradKeys * DP * 2];
    const uint32_t     t       = a.keyHeads.Quotient(blockIdx.x);
    const int          keyHead = (int)(blockIdx.x - t * a.keyHeads.d);
    const SequenceTile s       = FindTile(a.sequences, t, a.tiles, kGradRows, a.rows.size(), false, CAUSAL);
    if (s.tile < 0)
    {
        return;
    }
    const uint32_t wave = WaveOfGroup();
    const int      first = s.tile * kGradRows, ownFirst = first + (int)wave * 32, all = s.rows * a.rows.size();
    const AttentionRow row(a.rows, CAUSAL, s, keyHead, ownFirst + (int)(threadIdx.x & 31));
    auto               limitAt  = [&](int r) { return LimitOf(CAUSAL, s, a.rows.token(min(r, all - 1))); };
    const int          tileKeys = KeysOfTile(a, s), waveKeys = ownFirst < all ? limitAt(ownFirst + 31) + 1 : 0;
    const int          seenKeys = limitAt(ownFirst) + 1, parts = (tileKeys + kGradKeys - 1) / kGradKeys;
    const int          pieces = PiecesOf(tileKeys, a.splits), piece = (int)blockIdx.y;
    const int          from = PieceBegin(parts, piece, pieces), to = PieceBegin(parts, piece + 1, pieces);
    if (piece >= pieces)
    {
        return;
    }
    const uint8_t     *k = a.k + s.firstKey * a.kToken + keyHead * a.kHead, *v = a.v + s.firstKey * a.vToken + keyHead * a.vHead;

    using Copy = TileCopy<kGradKeys, DP, kGradThreads / 64>;
    auto load  = [&](int part, uint8_t *toK, uint8_t *toV)
    {
        const int key = part * kGradKeys;
        Copy::rows(wave, toK, k + key * a.kToken, (uint32_t)a.kToken, s.keys - key, a.dims);
        Copy::rows(wave, toV, v + key * a.vToken, (uint32_t)a.vToken, s.keys - key, a.dims);
    };
    if (from < to)
    {
        load(from, s_k0, s_v0);
    }
    Vec8<T> q[DP / 16], grad[DP / 16];
    LoadColumn<T, DP>(q, a.q + row.token * a.qToken + row.head * a.qHead, a.dims);
    LoadColumn<T, DP>(grad, a.grad + row.token * a.gradToken + row.head * a.gradHead, a.dims);
    const float base = ShareBase<T>(a.lse[(int64_t)row.head * a.sequences.rows + row.token]), scale = a.scale * kLog2E;
    // gradOut . out, here and for the other kernel
    float dot = 0;
    {
        Vec8<T> out[DP / 16];
        LoadColumn<T, DP>(out, a.out + row.token * a.outToken + row.head * a.outHead, a.dims);
#pragma unroll
        for (int step = 0; step < DP / 16; ++step)
        {
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                dot = __builtin_fmaf((float)out[step][i], (float)grad[step][i], dot);
            }
        }
        dot = BothSum(dot);
    }
    if (row.there && (threadIdx.x & 32) == 0 && piece == 0)
    {
        a.base[a.number(row)]  = base;
        a.delta[a.number(row)] = dot;
    }
    GradScale<T> grow;
    float        of = grow.factor * __builtin_amdgcn_exp2f(-kShareShift<T>), delta = dot * of;
    Acc16        sum[DP / 32] = {};
    auto         take = [&](int part, const uint8_t *fromK, const uint8_t *fromV, uint8_t *nextK, uint8_t *nextV)
    {
        const int key = part * kGradKeys;
        CopiesAndBarrier(); // (all have done the part before: its place may be written over)
        if (part + 1 < to)
        {
            load(part + 1, nextK, nextV);
        }
        if (key >= waveKeys)
        {
            return;
        }
        const bool hide = key + kGradKeys > seenKeys;
#pragma unroll
        for (int half = 0; half < kGradKeys / 32; ++half)
        {
            Acc16 shares = {}, grads = {};
#pragma unroll
            for (int step = 0; step < DP / 16; ++step)
            {
                Multiply(shares, RowsOperand<T, DP>(fromK, 32 * half, step), q[step]);
                Multiply(grads, RowsOperand<T, DP>(fromV, 32 * half, step), grad[step]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                const float share = __builtin_amdgcn_exp2f(__builtin_fmaf(shares[i], scale, -base));
                grads[i]          = share * __builtin_fmaf(grads[i], of, -delta);
            }
            if (hide)
            {
                KeepBranch();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    grads[i] = key + 32 * half + RowOf(i) <= row.limit ? grads[i] : 0.f;
                }
            }
            grow.fit(grads,
                     [&](float less)
                     {
                         of *= less, delta *= less;
#pragma unroll
                         for (int p = 0; p < DP / 32; ++p)
                         {
                             sum[p] *= less;
                         }
                     });
#pragma unroll
            for (int k16 = 0; k16 < 2; ++k16)
            {
                const Vec8<T> rounded = RoundedHalf<T>(grads, k16);
#pragma unroll
                for (int p = 0; p < DP / 32; ++p)
                {
                    Multiply(sum[p], ColumnsOperand<T, DP>(fromK, 32 * half + 16 * k16, p), rounded);
                }
            }
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
    const AttentionRow its(a.rows, CAUSAL, s, keyHead, ownFirst + (int)(Again(threadIdx.x) & 31));
    const float        factor = a.scale / grow.factor;
    uint8_t           *result = a.gradQ + its.token * a.gradQToken + its.head * a.gradQHead;
    float             *pieceOf = a.pieces + ((int64_t)piece * a.sequences.rows * a.heads + a.number(its)) * a.dims;
    auto hidden = [&](int n) { return k + (max(seenKeys, 0) + n) * a.kToken; };
    if (CAUSAL && AnyNotFinite(sum) &&
        RowsNotFinite<T>(a.dims, min((waveKeys + kGradKeys - 1) / kGradKeys * kGradKeys, s.keys) - max(seenKeys, 0), hidden))
    {
        // once more, without what the rows don't see (MultiplySeen)
        const uint32_t thread = Again(threadIdx.x);
        const int      lane   = (int)(thread & 63);
        LoadColumn<T, DP>(q, a.q + its.token * a.qToken + its.head * a.qHead, a.dims, thread);
        LoadColumn<T, DP>(grad, a.grad + its.token * a.gradToken + its.head * a.gradHead, a.dims, thread);
        for (int part = 0; part * 32 < a.dims; ++part)
        {
            Acc16 made = {};
            for (int key = from * kGradKeys; key < min(to * kGradKeys, waveKeys); key += 32)
            {
                const int own = min(key + (lane & 31), s.keys - 1);
                Acc16     shares = {}, grads = {};
                MultiplyRows<T, DP>(shares, k + own * a.kToken, a.dims, [&](int step) { return q[step]; });
                MultiplyRows<T, DP>(grads, v + own * a.vToken, a.dims, [&](int step) { return grad[step]; });
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    const float share = __builtin_amdgcn_exp2f(__builtin_fmaf(shares[i], scale, -base));
                    grads[i] = key + RowOf(i, lane) <= its.limit ? share * __builtin_fmaf(grads[i], of, -delta) : 0.f;
                }
                MultiplySeen<T>(made, grads, part, a.dims, s.keys - key, !__any(key + 31 > its.limit),
                                [&](int n) { return k + (key + n) * a.kToken; }, [&](int n) { return key + n <= its.limit; });
            }
            a.splits == 1 ? StoreColumnPart<T>(made, part, factor, result, its.there, a.dims)
                          : StorePiecePart(made, part, factor, pieceOf, its.there, a.dims);
        }
    }
    else if (a.splits == 1)
    {
        StoreColumn<T, DP>(sum, factor, result, its.there, a.dims);
    }
    else
    {
        StorePiece<DP>(sum, factor, pieceOf, its.there, a.dims);
    }
}

// ---- the keys' and values' gradients: 128 keys to a workgroup, 32 to a wave ------------------------------------------------
// With heads of 128 elements two gradients, keys and values would be 192 registers of the 256 that two waves to a SIMD have: keys and values
// stay in LDS, and eight waves go with them, of which two have the same keys and halves of each tile of rows, so that the
// workgroup of a long sequence's first keys, which all rows see, is done in half the time. (With 64 elements such pairs are slower:
// short sequences 64 us, 43 with four waves that take whole tiles.)
template<int DP>
constexpr bool kInPairs = DP > 64;
template<int DP>
constexpr int kOfThreads = kInPairs<DP> ? 512 : 256;

// A tile of rows: queries, gradients, and what their shares are made with.
template<int DP>
struct RowsPlace
{
    uint8_t *q, *grad;
    float   *base, *delta;
};

template<class T, int DP, bool CAUSAL>
__global__ __launch_bounds__(kOfThreads<DP>, 2) void AttentionGradKVKernel(const AttentionGradArgs a)
{
    constexpr int kWaves = kOfThreads<DP> / 64, kBytes = kOfRows * DP * 2;
    using Copy           = TileCopy<kOfRows, DP, kWaves>;
    __shared__ __attribute__((aligned(256))) uint8_t s_q0[kBytes], s_q1[kBytes], s_grad0[kBytes], s_grad1[kBytes];
    __shared__ __attribute__((aligned(256))) float   s_base0[kOfRows], s_base1[kOfRows], s_delta0[kOfRows], s_delta1[kOfRows];
    __shared__ __attribute__((aligned(256))) uint8_t s_k[kInPairs<DP> ? kOfKeys * DP * 2 : 16], s_v[kInPairs<DP> ? kOfKeys * DP * 2 : 16];
    const uint32_t     t       = a.keyHeads.Quotient(blockIdx.x);
    const int          keyHead = (int)(blockIdx.x - t * a.keyHeads.d);
    const SequenceTile s       = FindTile(a.sequences, t, a.keyTiles, kOfKeys, 1, true, CAUSAL);
    if (s.tile < 0)
    {
        return;
    }
    const uint32_t wave = WaveOfGroup(), ofKeys = wave % 4;
    const int      first = s.tile * kOfKeys, ownFirst = first + (int)ofKeys * 32, key = ownFirst + (int)(threadIdx.x & 31);
    const bool     there = key < s.keys;
    const int      group = a.rows.size(), all = s.rows * group;
    // the first row that sees one of these keys, and this piece's tiles of rows from there on
    const int seen   = FirstRowOfTile(a, s), tiles = (all - seen + kOfRows - 1) / kOfRows;
    const int pieces = PiecesOf(all - seen, a.keySplits), piece = (int)blockIdx.y;
    const int begin = seen + PieceBegin(tiles, piece, pieces) * kOfRows, last = seen + (PieceBegin(tiles, piece + 1, pieces) - 1) * kOfRows;
    if (piece >= pieces)
    {
        return;
    }
    auto      limitAt = [&](int r) { return LimitOf(CAUSAL, s, a.rows.token(min(r, all - 1))); };

    Vec8<T> k[kInPairs<DP> ? 1 : DP / 16], v[kInPairs<DP> ? 1 : DP / 16];
    if constexpr (kInPairs<DP>)
    {
        using Keys = TileCopy<kOfKeys, DP, kWaves>;
        Keys::rows(wave, s_k, a.k + (s.firstKey + first) * a.kToken + keyHead * a.kHead, (uint32_t)a.kToken, s.keys - first, a.dims);
        Keys::rows(wave, s_v, a.v + (s.firstKey + first) * a.vToken + keyHead * a.vHead, (uint32_t)a.vToken, s.keys - first, a.dims);
    }
    else
    {
        const int own = s.firstKey + min(key, s.keys - 1); // (columns behind the last key are made of it, and not stored)
        LoadColumn<T, DP>(k, a.k + own * a.kToken + keyHead * a.kHead, a.dims);
        LoadColumn<T, DP>(v, a.v + own * a.vToken + keyHead * a.vHead, a.dims);
    }
    auto keyOperand = [&](int step) { return kInPairs<DP> ? RowsOperand<T, DP>(s_k, 32 * ofKeys, step) : k[kInPairs<DP> ? 0 : step]; };
    auto valueOperand = [&](int step) { return kInPairs<DP> ? RowsOperand<T, DP>(s_v, 32 * ofKeys, step) : v[kInPairs<DP> ? 0 : step]; };
    GradScale<T> grow;
    float        of = grow.factor * __builtin_amdgcn_exp2f(-kShareShift<T>);
    const float  scale = a.scale * kLog2E;

    // the lane's places in a tile, from its first token's on
    uint32_t placeQ[Copy::kCount], placeGrad[Copy::kCount], placeValue;
    auto     places = [&](int at)
    {
        const int i0 = a.rows.token(at);
#pragma unroll
        for (int c = 0; c < Copy::kCount; ++c)
        {
            const int      r = Copy::rowOf(wave, c), i = a.rows.token(at + r);
            const uint32_t unit = Copy::unitOf(r), token = (uint32_t)(i - i0), head = (uint32_t)(at + r - i * group);
            const bool     some = (int)unit * 8 < a.dims;
            placeQ[c]           = some ? token * (uint32_t)a.qToken + head * (uint32_t)a.qHead + unit * 16 : Copy::kNowhere;
            placeGrad[c]        = some ? token * (uint32_t)a.gradToken + head * (uint32_t)a.gradHead + unit * 16 : Copy::kNowhere;
        }
        const int r = (int)(threadIdx.x & 63), i = a.rows.token(at + r);
        placeValue  = ((uint32_t)(i - i0) * (uint32_t)a.heads + (uint32_t)(at + r - i * group)) * 4;
    };
    // Rows from `at` on to LDS. Their buffers end with the sequence: rows behind it are zeros, which add nothing to any sum. (A token lies behind all
    // heads of the one before, or rows of the next sequence would stand there: tensors are wrapped in no other order, RequireHeads.)
    auto load = [&](int at, const RowsPlace<DP> &to)
    {
        using Place = __attribute__((address_space(3))) void;
        if (kOfRows % group != 0) // (where tiles have whole tokens, places are the same in all of them)
        {
            places(at);
        }
        const int      i0 = a.rows.token(at), tokens = s.rows - i0, token = s.firstRow + i0, head = keyHead * group;
        const int64_t  number = (int64_t)token * a.heads + head;
        const uint32_t bytes  = ((uint32_t)(min(tokens, kOfRows) - 1) * (uint32_t)a.heads + (uint32_t)group) * 4;
        // (every wave makes one of these two copies, so that all have as many on their way)
        const bool odd  = (wave & 1) != 0;
        const auto from = __builtin_amdgcn_make_buffer_rsrc((odd ? a.delta : a.base) + number, 0, (int)bytes, 0x00027000);
        const auto q    = Copy::buffer(a.q + token * a.qToken + head * a.qHead, tokens, a.qToken, group, a.qHead, a.dims);
        const auto grad = Copy::buffer(a.grad + token * a.gradToken + head * a.gradHead, tokens, a.gradToken, group, a.gradHead, a.dims);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Place *)(odd ? to.delta : to.base), 4, (int)placeValue, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < Copy::kCount; ++c)
        {
            Copy::copy(wave, c, to.q, q, placeQ[c], 0);
            Copy::copy(wave, c, to.grad, grad, placeGrad[c], 0);
        }
    };
    const RowsPlace<DP> place0 = {s_q0, s_grad0, s_base0, s_delta0}, place1 = {s_q1, s_grad1, s_base1, s_delta1};
    // From the last tile to the first: with `causal` workgroups of one sequence see the same last rows, which all but one read from L2.
    // (Of long sequences' reads four of five missed L2 the other way round, 44 of 100 do now: 621 us and 614.)
    if (begin <= last)
    {
        places(begin);
        load(last, place0);
    }
    Acc16 sumK[DP / 32] = {}, sumV[DP / 32] = {};
    auto  take = [&](int at, const RowsPlace<DP> &place, const RowsPlace<DP> &next)
    {
        CopiesAndBarrier(); // (all have done the tile before: its place may be written over)
        if (at > begin)
        {
            load(at - kOfRows, next);
        }
#pragma unroll
        for (int part = 0; part < (kInPairs<DP> ? 1 : 2); ++part)
        {
            const int half = kInPairs<DP> ? (int)wave / 4 : part, from = at + 32 * half;
            if (from >= all || limitAt(from + 31) < ownFirst)
            {
                continue;
            }
            Acc16 shares = {}, grads;
#pragma unroll
            for (int step = 0; step < DP / 16; ++step)
            {
                Multiply(shares, RowsOperand<T, DP>(place.q, 32 * half, step), keyOperand(step));
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4)
            {
                const float4 base = *reinterpret_cast<const float4 *>(place.base + 32 * half + RowOf(i));
                const float4 delta = *reinterpret_cast<const float4 *>(place.delta + 32 * half + RowOf(i));
                const float  b[4] = {base.x, base.y, base.z, base.w}, d[4] = {delta.x, delta.y, delta.z, delta.w};
#pragma unroll
                for (int n = 0; n < 4; ++n)
                {
                    shares[i + n] = __builtin_amdgcn_exp2f(__builtin_fmaf(shares[i + n], scale, -b[n]));
                    grads[i + n]  = -d[n];
                }
            }
#pragma unroll
            for (int step = 0; step < DP / 16; ++step)
            {
                Multiply(grads, RowsOperand<T, DP>(place.grad, 32 * half, step), valueOperand(step));
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                grads[i] = shares[i] * (std::is_same<T, Half>::value ? grads[i] * of : grads[i]);
            }
            if (limitAt(from) < ownFirst + 31)
            {
                KeepBranch();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    const bool takes = key <= limitAt(from + RowOf(i));
                    shares[i] = takes ? shares[i] : 0.f;
                    grads[i]  = takes ? grads[i] : 0.f;
                }
            }
            grow.fit(grads,
                     [&](float less)
                     {
                         of *= less;
#pragma unroll
                         for (int p = 0; p < DP / 32; ++p)
                         {
                             sumK[p] *= less;
                         }
                     });
#pragma unroll
            for (int r16 = 0; r16 < 2; ++r16)
            {
                const Vec8<T> share = RoundedHalf<T>(shares, r16), grad = RoundedHalf<T>(grads, r16);
#pragma unroll
                for (int p = 0; p < DP / 32; ++p)
                {
                    Multiply(sumV[p], ColumnsOperand<T, DP>(place.grad, 32 * half + 16 * r16, p), share);
                    Multiply(sumK[p], ColumnsOperand<T, DP>(place.q, 32 * half + 16 * r16, p), grad);
                }
            }
        }
    };
    for (int at = last; at >= begin; at -= 2 * kOfRows)
    {
        take(at, place0, place1);
        if (at > begin)
        {
            take(at - kOfRows, place1, place0);
        }
    }
    // (here, since two waves that go together may have other factors)
#pragma unroll
    for (int p = 0; p < DP / 32; ++p)
    {
        sumK[p] *= a.scale / grow.factor;
    }
    if constexpr (kInPairs<DP>)
    {
        // the second half's sums are added to the first's, by way of the tiles' places: a wave's sum of one gradient fits one of them
        float *place = reinterpret_cast<float *>(ofKeys == 0 ? s_q0 : ofKeys == 1 ? s_q1 : ofKeys == 2 ? s_grad0 : s_grad1) + (threadIdx.x & 63);
        auto   join  = [&](Acc16(&sum)[DP / 32])
        {
            __syncthreads();
            if (wave >= 4)
            {
#pragma unroll
                for (int i = 0; i < DP / 2; ++i)
                {
                    place[i * 64] = sum[i / 16][i % 16];
                }
            }
            __syncthreads();
            if (wave < 4)
            {
#pragma unroll
                for (int i = 0; i < DP / 2; ++i)
                {
                    sum[i / 16][i % 16] += place[i * 64];
                }
            }
        };
        join(sumK);
        join(sumV);
        if (wave >= 4)
        {
            return;
        }
    }
    const float   ofValues = __builtin_amdgcn_exp2f(-kShareShift<T>);
    const int     its      = ownFirst + (int)(Again(threadIdx.x) & 31), place = s.firstKey + its;
    const bool    stored   = its < s.keys;
    // 32 numbers of both gradients, from 32 * part on
    auto store = [&](int part, const Acc16 &ofK, float factorK, const Acc16 &ofV)
    {
        if (a.keySplits == 1)
        {
            StoreColumnPart<T>(ofK, part, factorK, a.gradK + place * a.gradKToken + keyHead * a.gradKHead, stored, a.dims);
            StoreColumnPart<T>(ofV, part, ofValues, a.gradV + place * a.gradVToken + keyHead * a.gradVHead, stored, a.dims);
        }
        else
        {
            const int64_t keys = (int64_t)a.sequences.keys * a.keyHeads.d, at = piece * keys + (int64_t)place * a.keyHeads.d + keyHead;
            StorePiecePart(ofK, part, factorK, a.pieces + at * a.dims, stored, a.dims);
            StorePiecePart(ofV, part, ofValues, a.pieces + (a.keySplits * keys + at) * a.dims, stored, a.dims);
        }
    };
    const int lane  = (int)(Again(threadIdx.x) & 63);
    auto      rowAt = [&](int row, int64_t tokenStride, int64_t headStride)
    {
        const int i = a.rows.token(row);
        return (int64_t)(s.firstRow + i) * tokenStride + (int64_t)(keyHead * group + row - i * group) * headStride;
    };
    auto queryAt = [&](int row) { return a.q + rowAt(row, a.qToken, a.qHead); };
    auto gradAt  = [&](int row) { return a.grad + rowAt(row, a.gradToken, a.gradHead); };
    // whether rows that don't see all of the wave's keys hold something that isn't finite
    auto hidden = [&]()
    {
        const int end   = min(min(last + kOfRows, all), max(min(ownFirst + 31 - (s.keys - s.rows), s.rows), 0) * group);
        const int count = end - begin;
        return RowsNotFinite<T>(a.dims, count, [&](int n) { return queryAt(begin + n); }) ||
               RowsNotFinite<T>(a.dims, count, [&](int n) { return gradAt(begin + n); });
    };
    if (CAUSAL && (AnyNotFinite(sumK) || AnyNotFinite(sumV)) && hidden())
    {
        // once more, of all rows here, without those that don't see a key (MultiplySeen)
        for (int part = 0; part * 32 < a.dims; ++part)
        {
            GradScale<T> grow;
            float        of = grow.factor * __builtin_amdgcn_exp2f(-kShareShift<T>);
            Acc16        madeK = {}, madeV = {};
            for (int from = begin; from < min(last + kOfRows, all); from += 32)
            {
                if (limitAt(from + 31) < ownFirst)
                {
                    continue;
                }
                const int own = min(from + (lane & 31), all - 1);
                Acc16     shares = {}, grads = {};
                MultiplyRows<T, DP>(shares, queryAt(own), a.dims, keyOperand);
                MultiplyRows<T, DP>(grads, gradAt(own), a.dims, valueOperand);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    const int     row = from + RowOf(i, lane);
                    const int64_t number = rowAt(min(row, all - 1), a.heads, 1);
                    const bool    takes = row < all && its <= limitAt(row);
                    shares[i] = takes ? __builtin_amdgcn_exp2f(__builtin_fmaf(shares[i], scale, -a.base[number])) : 0.f;
                    grads[i]  = takes ? shares[i] * ((grads[i] - a.delta[number]) * of) : 0.f;
                }
                grow.fit(grads, [&](float less) { of *= less, madeK *= less; });
                auto seen = [&](int n) { return its <= limitAt(from + n); };
                const bool every = limitAt(from) >= ownFirst + 31;
                MultiplySeen<T>(madeV, shares, part, a.dims, all - from, every, [&](int n) { return gradAt(from + n); }, seen);
                MultiplySeen<T>(madeK, grads, part, a.dims, all - from, every, [&](int n) { return queryAt(from + n); }, seen);
            }
            store(part, madeK, a.scale / grow.factor, madeV);
        }
        return;
    }
#pragma unroll
    for (int p = 0; p < DP / 32; ++p)
    {
        store(p, sumK[p], 1.f, sumV[p]);
    }
}

// ---- pieces joined: a tile of tokens to kJoinGroups workgroups, 8 elements of a row to a thread -----------------------------
constexpr int kJoinThreads = 256, kJoinGroups = 8;

template<class T, bool KEYS>
__global__ __launch_bounds__(kJoinThreads) void AttentionGradJoinKernel(const AttentionGradArgs a)
{
    const uint32_t     t       = a.keyHeads.Quotient(blockIdx.x);
    const int          keyHead = (int)(blockIdx.x - t * a.keyHeads.d), size = KEYS ? kOfKeys : kGradRows, units = a.dims / 8;
    const SequenceTile s       = FindTile(a.sequences, t, KEYS ? a.keyTiles : a.tiles, size, KEYS ? 1 : a.rows.size(), KEYS, a.causal);
    if (s.tile < 0)
    {
        return;
    }
    const int      first = s.tile * size, count = min((KEYS ? s.keys : s.rows * a.rows.size()) - first, size);
    const int64_t  rows = KEYS ? (int64_t)a.sequences.keys * a.keyHeads.d : (int64_t)a.sequences.rows * a.heads;
    const int      pieces = KEYS ? PiecesOf(s.rows * a.rows.size() - FirstRowOfTile(a, s), a.keySplits) : PiecesOf(KeysOfTile(a, s), a.splits);
    for (int i = (int)(blockIdx.y * kJoinThreads + threadIdx.x); i < count * units; i += kJoinGroups * kJoinThreads)
    {
        const int          r = i / units, d = (i - r * units) * 8;
        const AttentionRow row(a.rows, false, s, keyHead, first + r);
        const int          token = KEYS ? s.firstKey + first + r : row.token, head = KEYS ? keyHead : row.head;
        const int64_t      at    = KEYS ? (int64_t)token * a.keyHeads.d + head : a.number(row);
        auto               join  = [&](const float *from, uint8_t *to)
        {
            float sum[8] = {};
#pragma unroll 4
            for (int p = 0; p < pieces; ++p)
            {
                const Run<float, 8> piece = *reinterpret_cast<const Run<float, 8> *>(from + (p * rows + at) * a.dims + d);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    sum[k] += piece.v[k];
                }
            }
            Run<T, 8> made;
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                made.v[k] = FromFloat<T>(sum[k]);
            }
            *reinterpret_cast<Run<T, 8> *>(to + d * 2) = made;
        };
        if (KEYS)
        {
            join(a.pieces, a.gradK + token * a.gradKToken + head * a.gradKHead);
            join(a.pieces + a.keySplits * rows * a.dims, a.gradV + token * a.gradVToken + head * a.gradVHead);
        }
        else
        {
            join(a.pieces, a.gradQ + token * a.gradQToken + head * a.gradQHead);
        }
    }
}

// How a call is made, by its sizes alone: the sequences' lengths are on the device.
struct GradPlan
{
    int64_t rows, keys, heads, keyHeads, dims; // rows, keys: of all heads
    int64_t tiles, keyTiles;                   // at most, of a key head
    int64_t splits, keySplits;

    GradPlan(int64_t tokens, int64_t keyTokens, int64_t sequences, int64_t heads_, int64_t keyHeads_, int64_t dims_)
        : rows(tokens * heads_)
        , keys(keyTokens * keyHeads_)
        , heads(heads_)
        , keyHeads(keyHeads_)
        , dims(dims_)
    {
        const int64_t matrix = rows / keyHeads, most = std::max<int64_t>(sequences, 1), some = std::min(sequences, tokens), someKeys = std::min(sequences, keyTokens);
        const int64_t whole = (matrix + kGradRows - 1) / kGradRows, wholeKeys = (keyTokens + kOfKeys - 1) / kOfKeys;
        tiles     = whole + some;
        keyTiles  = wholeKeys + someKeys;
        // As many workgroups as fill the card's CUs twice; sequences of twice the mean length still have pieces of kPiece. (1200 rows of a
        // head that see 166 keys, 8 workgroups: the keys' kernel 54 us, 17.7 and 4.7 to join them; 151 rows before 6300 keys the queries' 106 us, 18.9
        // and 6.7; with up to 400 keys and rows, 72 workgroups, 19 and 22 us, 15 and 18 in pieces that take 5 each to join.)
        auto split = [](int64_t groups, int64_t each)
        { return each <= 2 * kPiece ? 1 : std::max<int64_t>(std::min({512 / std::max<int64_t>(groups, 1), (2 * each + kPiece - 1) / kPiece, kMostPieces}), 1); };
        splits    = split(std::max(whole, some) * keyHeads, keyTokens / most);
        keySplits = split(std::max(wholeKeys, someKeys) * keyHeads, matrix / most);
    }

    int64_t sums() const
    {
        return (2 * rows + 3) / 4 * 4; // (what follows is aligned)
    }

    int64_t bytes() const
    {
        const int64_t ofRows = splits > 1 ? splits * rows * dims : 0, ofKeys = keySplits > 1 ? 2 * keySplits * keys * dims : 0;
        return (sums() + std::max(ofRows, ofKeys)) * (int64_t)sizeof(float);
    }

    static constexpr int64_t kMostPieces = 32;
};

template<class T, int DP>
void Launch(const AttentionGradArgs &a, hipStream_t stream)
{
    if (a.tiles > 0)
    {
        const dim3 grid(a.tiles * a.keyHeads.d, (uint32_t)a.splits);
        if (a.causal)
        {
            AttentionGradQKernel<T, DP, true><<<grid, kGradThreads, 0, stream>>>(a);
        }
        else
        {
            AttentionGradQKernel<T, DP, false><<<grid, kGradThreads, 0, stream>>>(a);
        }
        CheckLaunch("attention's gradient (queries)");
        if (a.splits > 1)
        {
            AttentionGradJoinKernel<T, false><<<dim3(a.tiles * a.keyHeads.d, kJoinGroups), kJoinThreads, 0, stream>>>(a);
            CheckLaunch("attention's gradient (queries' pieces)");
        }
    }
    if (a.keyTiles > 0)
    {
        const dim3 grid(a.keyTiles * a.keyHeads.d, (uint32_t)a.keySplits);
        if (a.causal)
        {
            AttentionGradKVKernel<T, DP, true><<<grid, kOfThreads<DP>, 0, stream>>>(a);
        }
        else
        {
            AttentionGradKVKernel<T, DP, false><<<grid, kOfThreads<DP>, 0, stream>>>(a);
        }
        CheckLaunch("attention's gradient (keys)");
        if (a.keySplits > 1)
        {
            AttentionGradJoinKernel<T, true><<<dim3(a.keyTiles * a.keyHeads.d, kJoinGroups), kJoinThreads, 0, stream>>>(a);
            CheckLaunch("attention's gradient (keys' pieces)");
        }
    }
}

void SubmitGrad(hipStream_t stream, NVCVTensorHandle hgrad, NVCVTensorHandle hq, NVCVTensorHandle hk, NVCVTensorHandle hv, NVCVTensorHandle hout,
                NVCVTensorHandle hlse, NVCVTensorHandle hoffsets, NVCVTensorHandle hkeyOffsets, NVCVTensorHandle hkeyLengths,
                NVCVTensorHandle hgradQ, NVCVTensorHandle hgradK, NVCVTensorHandle hgradV, NVCVTensorHandle hworkspace, float scale, bool causal)
{
    const AttentionInputs in  = TakeAttention(hq, hk, hv, hoffsets, hkeyOffsets, hkeyLengths, hlse, false, scale);
    const HeadsView out = TakeHeadsLike(hout, in.q, "Output"), grad = TakeHeadsLike(hgrad, in.q, "Output's gradient");
    const HeadsView gradQ = TakeHeadsLike(hgradQ, in.q, "Queries' gradient"), gradK = TakeHeadsLike(hgradK, in.k, "Keys' gradient");
    const HeadsView gradV = TakeHeadsLike(hgradV, in.k, "Values' gradient");
    const GradPlan plan(in.q.tokens, in.k.tokens, in.sequences.count, in.q.heads, in.k.heads, in.q.dims);
    uint8_t *room = RequireWorkspace(hworkspace, plan.bytes());
    if (in.sequences.count == 0)
    {
        return;
    }
    float *base = reinterpret_cast<float *>(room);
    const AttentionGradArgs a = {
        in.q.base, in.k.base, in.v.base, out.base, grad.base, gradQ.base, gradK.base, gradV.base, in.q.tokenStride, in.q.headStride,
        in.k.tokenStride, in.k.headStride, in.v.tokenStride, in.v.headStride, out.tokenStride, out.headStride, grad.tokenStride, grad.headStride,
        gradQ.tokenStride, gradQ.headStride, gradK.tokenStride, gradK.headStride, gradV.tokenStride, gradV.headStride, in.sequences, in.lse,
        base, base + plan.rows, base + plan.sums(), {DivBy((uint32_t)(in.q.heads / in.k.heads))}, DivBy((uint32_t)in.k.heads), in.q.heads, in.q.dims,
        (uint32_t)plan.tiles, (uint32_t)plan.keyTiles, (int32_t)plan.splits, (int32_t)plan.keySplits, scale, causal};
    auto launch = [&](auto t)
    {
        using T = decltype(t);
        in.q.dims <= 64 ? Launch<T, 64>(a, stream) : Launch<T, 128>(a, stream);
    };
    in.q.elem == kRowF16 ? launch(Half{}) : launch(Bf16{});
}

} // namespace
} // namespace cvamd

using namespace cvamd;

extern "C"
{
CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionGradWorkspace(int64_t rows, int64_t keys, int64_t sequences, int32_t heads,
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
            *bytes = GradPlan(rows, keys, sequences, heads, keyHeads, dims).bytes();
        });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxAttentionGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle gradOut,
                                                    NVCVTensorHandle q, NVCVTensorHandle k, NVCVTensorHandle v,
                                                    NVCVTensorHandle out, NVCVTensorHandle lse, NVCVTensorHandle offsets,
                                                    NVCVTensorHandle keyOffsets, NVCVTensorHandle keyLengths,
                                                    NVCVTensorHandle gradQ, NVCVTensorHandle gradK, NVCVTensorHandle gradV,
                                                    NVCVTensorHandle workspace, float scale, int8_t causal)
{
    return Protect(
        [&]
        {
            (void)ToOperator<AttentionOperator>(handle);
            SubmitGrad(stream, gradOut, q, k, v, out, lse, offsets, keyOffsets, keyLengths, gradQ, gradK, gradV, workspace, scale, causal != 0);
        });
}
}
