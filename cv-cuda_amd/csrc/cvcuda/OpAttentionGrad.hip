// The gradient of attention (formulas: cvcuda/Attention.h; tiles and products: AttentionTiles.hpp).
//
// The shares p are made again from the scores and lse. Two kernels: one goes over the keys for 128 rows of queries and sums their gradient, one
// goes over the rows for 128 keys and sums the gradients of keys and values. So the products of scores and of gradOut . v are made
// twice (seven products of a pair where five would do), but every sum stays in the registers of one wave and is made in one
// order: there is nothing to add up by atomics in memory, and no gradient in 32 bits to write and read.
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
    float             *delta;   // [heads][rows]: gradOut . out
    float2            *largest; // F16: of each of the first kernel's workgroups, the largest squares of rows of gradOut and of v
    int32_t            largestCount;
    GroupRows          rows; // of a key head
    DivBy              keyHeads;
    int32_t            heads, dims;
    uint32_t           tiles, keyTiles;
    float              scale;
    bool               causal;

    // in lse and delta
    __device__ __forceinline__ int64_t number(const AttentionRow &row) const
    {
        return (int64_t)row.head * sequences.rows + row.token;
    }
};

// Shares, at most 1, are kept in F16 times 2^15: a share of 2^-29 has all of its bits then.
template<class T>
constexpr float kShareShift = std::is_same<T, Half>::value ? 15.f : 0.f;

// ---- gradOut . out, and for F16 what bounds the shares' gradients ------------------------------------------------------
constexpr int kDeltaThreads = 1024, kDeltaRows = kDeltaThreads / 16, kDeltaBlocks = 512;

__device__ __forceinline__ float SumOf16(float v)
{
#pragma unroll
    for (int d = 1; d < 16; d *= 2)
    {
        v += __shfl_xor(v, d);
    }
    return v;
}

// The sum of the products of 8 elements of two rows, in 32 bits.
template<class T>
__device__ __forceinline__ float Dot8(const uint8_t *a, const uint8_t *b)
{
    const Run<T, 8> x = *reinterpret_cast<const Run<T, 8> *>(a), y = *reinterpret_cast<const Run<T, 8> *>(b);
    float           s = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        s = __builtin_fmaf((float)x.v[i], (float)y.v[i], s);
    }
    return s;
}

// The larger of two sums of squares; one that is not finite (its sequence's gradients aren't either) counts for nothing.
__device__ __forceinline__ float Larger(float a, float b)
{
    return b < INFINITY ? fmaxf(a, b) : a;
}

// 16 lanes to a row, 8 elements to a lane.
template<class T>
__global__ __launch_bounds__(kDeltaThreads) void AttentionDeltaKernel(const AttentionGradArgs a)
{
    constexpr bool kBounds = std::is_same<T, Half>::value;
    const int      begin = a.sequences.firstRow(0), end = begin + a.sequences.rowsOf(a.sequences.count - 1, begin);
    const int      d = (int)(threadIdx.x % 16) * 8;
    const int64_t  first = (int64_t)blockIdx.x * kDeltaRows + threadIdx.x / 16, step = (int64_t)gridDim.x * kDeltaRows;
    float          ofGrad = 0, ofValues = 0;
    // (heads next to each other: rows of one token follow one another in memory)
    for (int64_t at = first, all = (int64_t)(end - begin) * a.heads; at < all; at += step)
    {
        const int token = begin + (int)(at / a.heads), head = (int)(at - (int64_t)(token - begin) * a.heads);
        float     dot = 0, square = 0;
        if (d < a.dims)
        {
            const uint8_t *grad = a.grad + token * a.gradToken + head * a.gradHead + d * 2;
            dot                 = Dot8<T>(grad, a.out + token * a.outToken + head * a.outHead + d * 2);
            square              = kBounds ? Dot8<T>(grad, grad) : 0.f;
        }
        dot = SumOf16(dot);
        if (kBounds)
        {
            ofGrad = Larger(ofGrad, SumOf16(square));
        }
        if (d == 0)
        {
            a.delta[(int64_t)head * a.sequences.rows + token] = dot;
        }
    }
    if constexpr (kBounds)
    {
        // values of sequences alone: a cache's places behind them hold anything
        const int32_t *starts = a.sequences.keyOffsets != nullptr ? a.sequences.keyOffsets : a.sequences.offsets;
        const int      heads  = (int)a.keyHeads.d;
        for (int64_t at = first, all = (int64_t)a.sequences.keys * heads; at < all; at += step)
        {
            const int token = (int)(at / heads), head = (int)(at - (int64_t)token * heads);
            int       low = 0, high = a.sequences.count; // the last sequence that begins at or before it lies between them
            while (high - low > 1)
            {
                const int middle = (low + high) / 2;
                (starts[middle] <= token ? low : high) = middle;
            }
            const int key = a.sequences.firstKey(low);
            float     square = 0;
            if (token >= key && token - key < a.sequences.keysOf(low, key) && d < a.dims)
            {
                const uint8_t *value = a.v + token * a.vToken + head * a.vHead + d * 2;
                square               = Dot8<T>(value, value);
            }
            ofValues = Larger(ofValues, SumOf16(square));
        }
        __shared__ float2 s_largest[kDeltaThreads / 64];
        ofGrad   = __uint_as_float(WaveLargest(__float_as_uint(ofGrad)));
        ofValues = __uint_as_float(WaveLargest(__float_as_uint(ofValues)));
        if ((threadIdx.x & 63) == 0)
        {
            s_largest[WaveOfGroup()] = make_float2(ofGrad, ofValues);
        }
        __syncthreads();
        if (threadIdx.x == 0)
        {
            float2 largest = s_largest[0];
            for (int w = 1; w < kDeltaThreads / 64; ++w)
            {
                largest = make_float2(Larger(largest.x, s_largest[w].x), Larger(largest.y, s_largest[w].y));
            }
            a.largest[blockIdx.x] = largest;
        }
    }
}

// The power of two by which the shares' gradients t are multiplied before they are rounded to T. In F16 small ones would be lost (its
// smallest number is 2^-24) and large ones have no bound in T, but |t| <= 2 |gradOut| |v| (out is a mean of values): with the longest of
// these rows it stays below 2^14, and what is 2^-28 of that keeps all of its bits.
template<class T>
__device__ __forceinline__ float GradFactor(const AttentionGradArgs &a)
{
    if constexpr (!std::is_same<T, Half>::value)
    {
        return 1.f;
    }
    float ofGrad = 0, ofValues = 0;
    for (int i = (int)(threadIdx.x & 63); i < a.largestCount; i += 64)
    {
        ofGrad   = Larger(ofGrad, a.largest[i].x);
        ofValues = Larger(ofValues, a.largest[i].y);
    }
    ofGrad            = __uint_as_float(WaveLargest(__float_as_uint(ofGrad)));
    ofValues          = __uint_as_float(WaveLargest(__float_as_uint(ofValues)));
    const float bound = sqrtf(ofGrad) * sqrtf(ofValues); // below 2^(ilogb + 1)
    return bound == 0 ? 1.f : ldexpf(1.f, min(max(12 - ilogbf(bound), -100), 100));
}

// What a row's scores are taken relative to: lse to the base 2, less the shift; a row without a key, or behind the end, has no share.
template<class T>
__device__ __forceinline__ float ShareBase(float lse, bool there)
{
    return !there || lse == -INFINITY ? INFINITY : __builtin_fmaf(lse, kLog2E, -kShareShift<T>);
}

// ---- the queries' gradient: 128 rows to a workgroup, 32 to a wave --------------------------------------------------------
constexpr int kGradRows = 128, kGradKeys = 64, kGradThreads = 256;

template<class T, int DP>
__global__ __launch_bounds__(kGradThreads, 2) void AttentionGradQKernel(const AttentionGradArgs a)
{
    __shared__ __attribute__((aligned(256))) uint8_t s_k[2][kGradKeys * DP * 2], s_v[2][kGradKeys * DP * 2];
    const uint32_t     t       = a.keyHeads.Quotient(blockIdx.x);
    const int          keyHead = (int)(blockIdx.x - t * a.keyHeads.d);
    const SequenceTile s       = FindTile(a.sequences, a.causal ? a.tiles - 1 - t : t, kGradRows, a.rows.size(), false);
    if (s.tile < 0)
    {
        return;
    }
    const int first = s.tile * kGradRows, ownFirst = first + (int)WaveOfGroup() * 32, all = s.rows * a.rows.size();
    const AttentionRow row(a.rows, a.causal, s, keyHead, ownFirst + (int)(threadIdx.x & 31));
    auto               limitAt  = [&](int r) { return LimitOf(a.causal, s, a.rows.token(min(r, all - 1))); };
    const int          tileKeys = max(limitAt(first + kGradRows - 1) + 1, 0), waveKeys = ownFirst < all ? limitAt(ownFirst + 31) + 1 : 0;
    const int          seenKeys = limitAt(ownFirst) + 1, parts = (tileKeys + kGradKeys - 1) / kGradKeys;
    const uint8_t     *k = a.k + s.firstKey * a.kToken + keyHead * a.kHead, *v = a.v + s.firstKey * a.vToken + keyHead * a.vHead;

    TileLoad<kGradKeys, DP, kGradThreads> nextK, nextV;
    auto load = [&](int part)
    {
        const int key = part * kGradKeys;
        nextK.get(threadIdx.x, k + key * a.kToken, a.kToken, s.keys - key, a.dims);
        nextV.get(threadIdx.x, v + key * a.vToken, a.vToken, s.keys - key, a.dims);
    };
    if (parts > 0)
    {
        load(0);
    }
    Vec8<T> q[DP / 16], grad[DP / 16];
    LoadColumn<T, DP>(q, a.q + row.token * a.qToken + row.head * a.qHead, a.dims);
    LoadColumn<T, DP>(grad, a.grad + row.token * a.gradToken + row.head * a.gradHead, a.dims);
    const float factor = GradFactor<T>(a), base = ShareBase<T>(a.lse[a.number(row)], row.there);
    const float scale = a.scale * kLog2E, of = factor * __builtin_amdgcn_exp2f(-kShareShift<T>), delta = a.delta[a.number(row)] * of;
    Acc16       sum[DP / 32] = {};
    for (int part = 0; part < parts; ++part)
    {
        const int at = part & 1, key = part * kGradKeys;
        nextK.put(threadIdx.x, s_k[at]);
        nextV.put(threadIdx.x, s_v[at]);
        __syncthreads();
        if (part + 1 < parts)
        {
            load(part + 1);
        }
        if (key >= waveKeys)
        {
            continue;
        }
        const bool hide = key + kGradKeys > seenKeys;
#pragma unroll
        for (int half = 0; half < kGradKeys / 32; ++half)
        {
            Acc16 shares = {}, grads = {};
#pragma unroll
            for (int step = 0; step < DP / 16; ++step)
            {
                Multiply(shares, RowsOperand<T, DP>(s_k[at], 32 * half, step), q[step]);
                Multiply(grads, RowsOperand<T, DP>(s_v[at], 32 * half, step), grad[step]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                const float share = __builtin_amdgcn_exp2f(__builtin_fmaf(shares[i], scale, -base));
                grads[i]          = share * __builtin_fmaf(grads[i], of, -delta);
            }
            if (hide)
            {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    grads[i] = key + 32 * half + RowOf(i) <= row.limit ? grads[i] : 0.f;
                }
            }
#pragma unroll
            for (int k16 = 0; k16 < 2; ++k16)
            {
                const Vec8<T> rounded = RoundedHalf<T>(grads, k16);
#pragma unroll
                for (int p = 0; p < DP / 32; ++p)
                {
                    Multiply(sum[p], ColumnsOperand<T, DP>(s_k[at], 32 * half + 16 * k16, p), rounded);
                }
            }
        }
    }
    StoreColumn<T, DP>(sum, a.scale / factor, a.gradQ + row.token * a.gradQToken + row.head * a.gradQHead, row.there, a.dims);
}

// ---- the keys' and values' gradients: 128 keys to a workgroup, 32 to a wave ------------------------------------------------
constexpr int kOfKeys = 128, kOfRows = 64;

template<class T, int DP>
__global__ __launch_bounds__(kGradThreads) void AttentionGradKVKernel(const AttentionGradArgs a)
{
    __shared__ __attribute__((aligned(256))) uint8_t s_q[2][kOfRows * DP * 2], s_grad[2][kOfRows * DP * 2];
    __shared__ __attribute__((aligned(16))) float    s_base[2][kOfRows], s_delta[2][kOfRows];
    __shared__ int                                   s_limit[2][kOfRows];
    const uint32_t     t       = a.keyHeads.Quotient(blockIdx.x);
    const int          keyHead = (int)(blockIdx.x - t * a.keyHeads.d);
    const SequenceTile s       = FindTile(a.sequences, t, kOfKeys, 1, true);
    if (s.tile < 0)
    {
        return;
    }
    const int  first = s.tile * kOfKeys, ownFirst = first + (int)WaveOfGroup() * 32, key = ownFirst + (int)(threadIdx.x & 31);
    const bool there = key < s.keys;
    const int  all   = s.rows * a.rows.size();
    // the first row that sees one of these keys
    const int  begin = a.causal ? min(max(first - (s.keys - s.rows), 0), s.rows) * a.rows.size() : 0;
    auto       limitAt = [&](int r) { return LimitOf(a.causal, s, a.rows.token(min(r, all - 1))); };

    TileLoad<kOfRows, DP, kGradThreads> nextQ, nextGrad;
    float                               nextBase = INFINITY, nextDelta = 0;
    int                                 nextLimit = -1;
    const float                         factor = GradFactor<T>(a), of = factor * __builtin_amdgcn_exp2f(-kShareShift<T>);
    auto load = [&](int at)
    {
        auto place = [&](const uint8_t *base, int64_t tokenStride, int64_t headStride, int r)
        {
            const int i = a.rows.token(at + r);
            return base + (s.firstRow + i) * tokenStride + (keyHead * a.rows.size() + (at + r - i * a.rows.size())) * headStride;
        };
        nextQ.get(threadIdx.x, all - at, a.dims, [&](int r) { return place(a.q, a.qToken, a.qHead, r); });
        nextGrad.get(threadIdx.x, all - at, a.dims, [&](int r) { return place(a.grad, a.gradToken, a.gradHead, r); });
        if (threadIdx.x < kOfRows)
        {
            const AttentionRow row(a.rows, a.causal, s, keyHead, at + (int)threadIdx.x);
            nextBase  = ShareBase<T>(a.lse[a.number(row)], row.there);
            nextDelta = row.there ? a.delta[a.number(row)] * of : 0.f;
            nextLimit = row.there ? row.limit : -1;
        }
    };
    if (begin < all)
    {
        load(begin);
    }
    Vec8<T> k[DP / 16], v[DP / 16];
    const int own = s.firstKey + min(key, s.keys - 1); // (columns behind the last key are made of it, and not stored)
    LoadColumn<T, DP>(k, a.k + own * a.kToken + keyHead * a.kHead, a.dims);
    LoadColumn<T, DP>(v, a.v + own * a.vToken + keyHead * a.vHead, a.dims);
    const float scale = a.scale * kLog2E;
    Acc16       sumK[DP / 32] = {}, sumV[DP / 32] = {};
    for (int at = begin, turn = 0; at < all; at += kOfRows, turn ^= 1)
    {
        nextQ.put(threadIdx.x, s_q[turn]);
        nextGrad.put(threadIdx.x, s_grad[turn]);
        if (threadIdx.x < kOfRows)
        {
            s_base[turn][threadIdx.x]  = nextBase;
            s_delta[turn][threadIdx.x] = nextDelta;
            s_limit[turn][threadIdx.x] = nextLimit;
        }
        __syncthreads();
        if (at + kOfRows < all)
        {
            load(at + kOfRows);
        }
        if (limitAt(at + kOfRows - 1) < ownFirst)
        {
            continue;
        }
        const bool hide = limitAt(at) < ownFirst + 31;
#pragma unroll
        for (int half = 0; half < kOfRows / 32; ++half)
        {
            Acc16 shares = {}, grads = {};
#pragma unroll
            for (int step = 0; step < DP / 16; ++step)
            {
                Multiply(shares, RowsOperand<T, DP>(s_q[turn], 32 * half, step), k[step]);
                Multiply(grads, RowsOperand<T, DP>(s_grad[turn], 32 * half, step), v[step]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                const int r = 32 * half + RowOf(i);
                shares[i]   = __builtin_amdgcn_exp2f(__builtin_fmaf(shares[i], scale, -s_base[turn][r]));
                grads[i]    = shares[i] * __builtin_fmaf(grads[i], of, -s_delta[turn][r]);
            }
            if (hide)
            {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    const bool seen = key <= s_limit[turn][32 * half + RowOf(i)];
                    shares[i]       = seen ? shares[i] : 0.f;
                    grads[i]        = seen ? grads[i] : 0.f;
                }
            }
#pragma unroll
            for (int r16 = 0; r16 < 2; ++r16)
            {
                const Vec8<T> share = RoundedHalf<T>(shares, r16), grad = RoundedHalf<T>(grads, r16);
#pragma unroll
                for (int p = 0; p < DP / 32; ++p)
                {
                    Multiply(sumV[p], ColumnsOperand<T, DP>(s_grad[turn], 32 * half + 16 * r16, p), share);
                    Multiply(sumK[p], ColumnsOperand<T, DP>(s_q[turn], 32 * half + 16 * r16, p), grad);
                }
            }
        }
    }
    StoreColumn<T, DP>(sumK, a.scale / factor, a.gradK + (s.firstKey + key) * a.gradKToken + keyHead * a.gradKHead, there, a.dims);
    StoreColumn<T, DP>(sumV, __builtin_amdgcn_exp2f(-kShareShift<T>), a.gradV + (s.firstKey + key) * a.gradVToken + keyHead * a.gradVHead, there,
                       a.dims);
}

int64_t GradBytes(int64_t rows, int64_t heads)
{
    return kDeltaBlocks * (int64_t)sizeof(float2) + rows * heads * (int64_t)sizeof(float);
}

template<class T, int DP>
void Launch(const AttentionGradArgs &a, hipStream_t stream)
{
    if (a.tiles > 0)
    {
        AttentionDeltaKernel<T><<<(uint32_t)a.largestCount, kDeltaThreads, 0, stream>>>(a);
        CheckLaunch("attention's gradient (sums)");
        AttentionGradQKernel<T, DP><<<a.tiles * a.keyHeads.d, kGradThreads, 0, stream>>>(a);
        CheckLaunch("attention's gradient (queries)");
    }
    if (a.keyTiles > 0)
    {
        AttentionGradKVKernel<T, DP><<<a.keyTiles * a.keyHeads.d, kGradThreads, 0, stream>>>(a);
        CheckLaunch("attention's gradient (keys)");
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
    uint8_t        *room  = RequireWorkspace(hworkspace, GradBytes(in.q.tokens, in.q.heads));
    if (in.sequences.count == 0)
    {
        return;
    }
    const int64_t group = in.q.heads / in.k.heads, rows = in.q.tokens, keys = in.k.tokens, sequences = in.sequences.count;
    const int64_t tiles    = (rows * group + kGradRows - 1) / kGradRows + std::min(sequences, rows);
    const int64_t keyTiles = (keys + kOfKeys - 1) / kOfKeys + std::min(sequences, keys);
    if (std::max(tiles, keyTiles) * in.k.heads > INT32_MAX / kGradThreads * 2)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Too many rows or keys");
    }
    const int64_t  all = std::max(rows * in.q.heads, keys * in.k.heads);
    float2        *largest = reinterpret_cast<float2 *>(room);
    const AttentionGradArgs a = {
        in.q.base, in.k.base, in.v.base, out.base, grad.base, gradQ.base, gradK.base, gradV.base, in.q.tokenStride, in.q.headStride,
        in.k.tokenStride, in.k.headStride, in.v.tokenStride, in.v.headStride, out.tokenStride, out.headStride, grad.tokenStride, grad.headStride,
        gradQ.tokenStride, gradQ.headStride, gradK.tokenStride, gradK.headStride, gradV.tokenStride, gradV.headStride, in.sequences, in.lse,
        reinterpret_cast<float *>(largest + kDeltaBlocks), largest,
        (int32_t)std::min<int64_t>((all + kDeltaRows - 1) / kDeltaRows, kDeltaBlocks), {DivBy((uint32_t)group)}, DivBy((uint32_t)in.k.heads),
        in.q.heads, in.q.dims, (uint32_t)tiles, (uint32_t)keyTiles, scale, causal};
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
            *bytes = GradBytes(rows, heads);
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
