// What the kernels of attention and of its gradient share (formulas: cvcuda/Attention.h).
//
// All products are 32 x 32 x 16 matrix instructions. Scores are made transposed, keys times queries, so that a lane has the scores of ONE
// query (column) and 16 keys of a tile's 32: their maximum and sum stay in the lane, but for one exchange with the lane that
// has the other 16. And what a lane has of them is, rounded and packed, what the next product takes as its right operand,
// without a move between lanes: of 16 keys the lower half wave has 0-3 and 8-11, the upper one 4-7 and 12-15, so the left operand's
// keys are read in that order too (a sum's order does not matter to the instruction).
//
// Tiles of rows (keys and values, or queries and gradients) lie in LDS as they lie in memory, in units of 16 bytes that are exchanged within
// a row by the row's number, so that neither eight rows' units of one column nor four rows' neighbouring units (a transposed read) meet
// in a bank.
#ifndef CVCUDA_AMD_ATTENTIONTILES_HPP
#define CVCUDA_AMD_ATTENTIONTILES_HPP

#include "AttentionOps.hpp"

#include <type_traits>

namespace cvamd {

constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// How far scores, to the base 2, may lie above what exponentials are taken relative to.
constexpr float kSlack = 8.f;

// Exponentials are kept in F16 times a power of two: a share of 2^-20 of the largest keeps all of its bits, one of 2^-30 one bit, and the largest reaches
// 2^14. BF16 has the exponents of F32: there none is above 1, so that its products with values stay as finite as these.
template<class T>
constexpr float kExpShift = std::is_same<T, Half>::value ? 6.f : -kSlack;

template<class T>
using Vec8 = T __attribute__((ext_vector_type(8)));
using Acc16 = float __attribute__((ext_vector_type(16)));
using Vec4s = short __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void Multiply(Acc16 &acc, Vec8<Bf16> a, Vec8<Bf16> b)
{
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}

__device__ __forceinline__ void Multiply(Acc16 &acc, Vec8<Half> a, Vec8<Half> b)
{
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}

// Largest and sum of a lane's and the other half's.
__device__ __forceinline__ float BothMax(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float BothSum(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A number that the compiler takes for another one than v: what is made of it once more doesn't wait in registers.
__device__ __forceinline__ uint32_t Again(uint32_t v)
{
    asm volatile("" : "+v"(v));
    return v;
}

// Keeps the compiler from making what stands in a branch in every case, and choosing afterwards.
__device__ __forceinline__ void KeepBranch()
{
    asm volatile("");
}

// ---- tiles in LDS ------------------------------------------------------------------------------------------------
// Row r of DP elements (64 or 128), its unit u of 16 bytes at place u ^ Swap(r). Of eleven exchanges that were tried these are the ones
// with which a wave's read of rows takes 7.0 clocks and a transposed one 5.5 (without any 32 and 5.5, 64 and 8.1).
template<int DP>
__device__ __forceinline__ uint32_t Swap(uint32_t row)
{
    return DP == 64 ? (row >> 1) & 7 : ((row & 7) << 1) | ((row >> 3) & 1);
}

template<int DP>
__device__ __forceinline__ uint32_t TileAt(uint32_t row, uint32_t unit)
{
    return row * (DP * 2) + ((unit ^ Swap<DP>(row)) << 4);
}

// Rows of a matrix as the instruction's left operand: lane l has row l % 32, elements 16 * step + 8 * (l / 32) to + 7.
template<class T, int DP>
__device__ __forceinline__ Vec8<T> RowsOperand(const uint8_t *tile, uint32_t firstRow, int step)
{
    const uint32_t lane = threadIdx.x & 63;
    return *reinterpret_cast<const Vec8<T> *>(tile + TileAt<DP>(firstRow + (lane & 31), 2 * step + (lane >> 5)));
}

// Columns 32 * part to + 31 of 16 rows as the left operand: lane l has column 32 * part + l % 32 of the rows 4 * (l / 32) to + 3 and 8 + 4 *
// (l / 32) to + 3. A transposed read gives each lane of 16 a column of the four rows that they read; firstRow is a multiple of 16.
template<class T, int DP>
__device__ __forceinline__ Vec8<T> ColumnsOperand(const uint8_t *tile, uint32_t firstRow, int part)
{
    using Place          = __attribute__((address_space(3))) Vec4s;
    const uint32_t lane  = threadIdx.x & 63;
    const uint32_t row   = firstRow + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const uint32_t unit  = 4 * part + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const uint8_t *first = tile + TileAt<DP>(row, unit) + 8 * (lane & 1), *second = tile + TileAt<DP>(row + 8, unit) + 8 * (lane & 1);
    struct
    {
        Vec4s low, high;
    } both = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((Place *)first), __builtin_amdgcn_ds_read_tr16_b64_v4i16((Place *)second)};
    return __builtin_bit_cast(Vec8<T>, both);
}

// Eight of a lane's 16 numbers, rounded: rows 16 * half to + 15 of a product as the next one's right operand. (Rounded, since a matrix instruction takes
// both operands in the 16 bits of the values or keys: each is off by half a step at most, and the sum by that of the magnitudes that are added, where
// the result's own rounding is half a step of it. Measured over a call, 0.0021 of BF16 results, of which 0.0016 are their rounding. A second
// product, for what the rounding took off, would take as long as the first.)
template<class T>
__device__ __forceinline__ Vec8<T> RoundedHalf(const Acc16 &v, int half)
{
    Vec8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        r[i] = (T)v[8 * half + i];
    }
    return r;
}

// The row that a lane's number i of a product lies in.
__device__ __forceinline__ int RowOf(int i, int lane)
{
    return (i >> 2) * 8 + (lane >> 5) * 4 + (i & 3);
}

__device__ __forceinline__ int RowOf(int i)
{
    return RowOf(i, (int)(threadIdx.x & 63));
}

// ROWS rows from memory to a tile in LDS, without a stop in registers, by WAVES waves. Each instruction moves 64 units to 64 places that
// follow one another: the lanes' addresses make the exchange of units. The buffer ends behind the last row, and what lies behind
// a buffer's end reads as zeros; lanes of units behind `dims` read there too.
template<int ROWS, int DP, int WAVES>
struct TileCopy
{
    static constexpr int kUnits = DP / 8, kOfOne = 64 / kUnits, kCount = ROWS / (kOfOne * WAVES);
    static_assert(ROWS % (kOfOne * WAVES) == 0, "whole instructions");
    static constexpr uint32_t kNowhere = 0x80000000u; // (tiles are smaller: kMostStride)

    // The lane's row of the tile and its unit in the wave's copy i.
    __device__ __forceinline__ static int rowOf(uint32_t wave, int i)
    {
        return (int)((uint32_t)(i * WAVES) + wave) * kOfOne + (int)((threadIdx.x & 63) / kUnits);
    }

    __device__ __forceinline__ static uint32_t unitOf(int row)
    {
        return ((threadIdx.x & 63) % kUnits) ^ Swap<DP>((uint32_t)row);
    }

    __device__ __forceinline__ static void copy(uint32_t wave, int i, uint8_t *tile, __amdgpu_buffer_rsrc_t from, uint32_t at, uint32_t atAll)
    {
        using Place = __attribute__((address_space(3))) void;
        uint8_t *to = tile + ((uint32_t)(i * WAVES) + wave) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Place *)to, 16, (int)at, (int)atAll, 0, 0);
    }

    // `tokens` tokens of `heads` heads from `base` on: as a buffer that ends behind the last one's last element, or after as many bytes as a tile's
    // addresses reach.
    __device__ __forceinline__ static __amdgpu_buffer_rsrc_t buffer(const uint8_t *base, int tokens, int64_t tokenStride, int heads, int64_t headStride,
                                                                    int dims)
    {
        const uint32_t bytes = (uint32_t)(min(tokens, ROWS) - 1) * (uint32_t)tokenStride + (uint32_t)(heads - 1) * (uint32_t)headStride + (uint32_t)dims * 2;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, (int)bytes, 0x00027000);
    }

    // Rows `stride` apart from `base` on, of which there are `count`, one at least.
    __device__ __forceinline__ static void rows(uint32_t wave, uint8_t *tile, const uint8_t *base, uint32_t stride, int count, int dims)
    {
        const uint32_t bytes = (uint32_t)(min(count, ROWS) - 1) * stride + (uint32_t)dims * 2;
        const auto     from  = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, (int)bytes, 0x00027000);
#pragma unroll
        for (int i = 0; i < kCount; ++i)
        {
            const int      row  = rowOf(wave, i) - i * WAVES * kOfOne;
            const uint32_t unit = unitOf(rowOf(wave, i));
            copy(wave, i, tile, from, (int)unit * 8 < dims ? (uint32_t)row * stride + unit * 16 : kNowhere, (uint32_t)(i * WAVES * kOfOne) * stride);
        }
    }
};

// A wave's tile of ROWS rows on its way to LDS in registers: where tiles follow one another without a barrier, and LDS holds one of them.
template<int ROWS, int DP>
struct TileLoad
{
    using Copy = TileCopy<ROWS, DP, 1>;
    using Unit = uint32_t __attribute__((ext_vector_type(4)));

    Unit unit[Copy::kCount];

    // As TileCopy::rows. PAST: as in LoadRun.
    template<bool PAST>
    __device__ __forceinline__ void get(const uint8_t *base, uint32_t stride, int count, int dims)
    {
        const uint32_t lane = threadIdx.x & 63, row = lane / Copy::kUnits, part = lane % Copy::kUnits;
        const uint32_t bytes = (uint32_t)(min(count, ROWS) - 1) * stride + (uint32_t)dims * 2;
        const uint32_t at    = (int)part * 8 < dims ? row * stride + part * 16 : Copy::kNowhere;
        const auto     from  = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, (int)bytes, 0x00027000);
#pragma unroll
        for (int i = 0; i < Copy::kCount; ++i)
        {
            unit[i] = __builtin_amdgcn_raw_buffer_load_b128(from, (int)at, (int)((uint32_t)(i * Copy::kOfOne) * stride), PAST ? 2 : 0);
        }
    }

    __device__ __forceinline__ void put(uint8_t *tile) const
    {
        const uint32_t lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < Copy::kCount; ++i)
        {
            *reinterpret_cast<Unit *>(tile + TileAt<DP>((uint32_t)(i * Copy::kOfOne) + lane / Copy::kUnits, lane % Copy::kUnits)) = unit[i];
        }
    }
};

// All waves' copies to LDS but each one's last LEFT have arrived, and their reads of it are done. (A barrier alone waits for no copy.)
template<int LEFT = 0>
__device__ __forceinline__ void CopiesAndBarrier()
{
    static_assert(LEFT < 64, "the counter's range");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (LEFT & 15) | (LEFT >> 4) << 14); // vmcnt(LEFT)
    __syncthreads();
}

// A row of a matrix as the right operand's column: elements 16 * step + 8 * (l / 32) to + 7 of it, zeros behind `dims`. Loads stand
// under no condition.
template<class T, int DP>
__device__ __forceinline__ void LoadColumn(Vec8<T> (&to)[DP / 16], const uint8_t *row, int dims, uint32_t thread = threadIdx.x)
{
    const int first = (int)((thread & 63) >> 5) * 8;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
    {
        to[s] = *reinterpret_cast<const Vec8<T> *>(row + min(16 * s + first, dims - 8) * 2);
    }
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
    {
        to[s] = 16 * s + first < dims ? to[s] : Vec8<T>{};
    }
}

// 32 numbers of a transposed product's columns, from 32 * part on, to rows of memory: lane l's column is the row at `row`, times `factor`, rounded.
// Lanes exchange what they have, so that each stores whole 16 bytes.
template<class T>
__device__ __forceinline__ void StoreColumnPart(const Acc16 &acc, int part, float factor, uint8_t *row, bool there, int dims)
{
    const int upper = (int)((Again(threadIdx.x) & 63) >> 5);
#pragma unroll
    for (int p = 0; p < 2; ++p)
    {
        uint32_t words[2][2]; // of the elements 16 * p + 4 * upper to + 3, and 8 + that
#pragma unroll
        for (int k = 0; k < 2; ++k)
        {
#pragma unroll
            for (int w = 0; w < 2; ++w)
            {
                struct
                {
                    T a, b;
                } two = {(T)(acc[8 * p + 4 * k + 2 * w] * factor), (T)(acc[8 * p + 4 * k + 2 * w + 1] * factor)};
                words[k][w] = __builtin_bit_cast(uint32_t, two);
            }
        }
        const auto x     = __builtin_amdgcn_permlane32_swap(words[0][0], words[1][0], false, false);
        const auto y     = __builtin_amdgcn_permlane32_swap(words[0][1], words[1][1], false, false);
        const int  first = part * 32 + 16 * p + 8 * upper;
        if (there && first < dims)
        {
            *reinterpret_cast<uint4 *>(row + first * 2) = make_uint4(x[0], y[0], x[1], y[1]);
        }
    }
}

template<class T, int DP>
__device__ __forceinline__ void StoreColumn(const Acc16 (&acc)[DP / 32], float factor, uint8_t *row, bool there, int dims)
{
#pragma unroll
    for (int part = 0; part < DP / 32; ++part)
    {
        StoreColumnPart<T>(acc[part], part, factor, row, there, dims);
    }
}

// The same to a row of F32, which is joined with those of other pieces.
__device__ __forceinline__ void StorePiecePart(const Acc16 &acc, int part, float factor, float *row, bool there, int dims)
{
#pragma unroll
    for (int i = 0; i < 16; i += 4)
    {
        const int d = 32 * part + RowOf(i);
        if (there && d < dims)
        {
            *reinterpret_cast<float4 *>(row + d) = make_float4(acc[i] * factor, acc[i + 1] * factor, acc[i + 2] * factor, acc[i + 3] * factor);
        }
    }
}

template<int DP>
__device__ __forceinline__ void StorePiece(const Acc16 (&acc)[DP / 32], float factor, float *row, bool there, int dims)
{
#pragma unroll
    for (int p = 0; p < DP / 32; ++p)
    {
        StorePiecePart(acc[p], p, factor, row, there, dims);
    }
}

// ---- values that are not finite ----------------------------------------------------------------------------------------------
// A tile's products give what a row does not see a weight of 0, and 0 times an infinity or NaN is NaN. So where a result is not finite, and something
// in its tiles that not all of its rows or keys see isn't either, its wave makes it once more, by itself and from memory, 32 numbers of the
// columns at a time (few registers): where something is hidden each row of the matrix has a product of its own, which only the columns that see it
// take. Finite inputs pay a sum over the results (long prompts 271.4 us, 272.4 before); a call whose inputs are all NaN takes up to 40 times
// as long.
template<int N>
__device__ __forceinline__ bool AnyNotFinite(const Acc16 (&sum)[N])
{
    Acc16 all = sum[0];
#pragma unroll
    for (int p = 1; p < N; ++p)
    {
        all += sum[p];
    }
    float one = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
    {
        one += all[i];
    }
    return __any(!(fabsf(one) < INFINITY)); // (a sum of these that overflows costs time alone)
}

// Rows of a matrix in memory, the row at `row` being the lane's and that of the lane 32 from it, times columns(step).
template<class T, int DP, class F>
__device__ __forceinline__ void MultiplyRows(Acc16 &sum, const uint8_t *row, int dims, F &&columns)
{
    const int first = (int)((Again(threadIdx.x) & 63) >> 5) * 8;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
    {
        const Vec8<T> part = *reinterpret_cast<const Vec8<T> *>(row + min(16 * s + first, dims - 8) * 2);
        Multiply(sum, 16 * s + first < dims ? part : Vec8<T>{}, columns(s));
        __builtin_amdgcn_sched_barrier(0); // (one after the other: few registers)
    }
}

// Whether `count` rows, in memory at rowAt(n), hold a number that is not finite.
template<class T, class R>
__device__ __forceinline__ bool RowsNotFinite(int dims, int count, R &&rowAt)
{
    constexpr uint32_t kExponent = std::is_same<T, Half>::value ? 0x7C00 : 0x7F80;
    const int          at        = (int)(Again(threadIdx.x) & 63) * 2;
    bool               some      = false;
    for (int n = 0; n < count; ++n)
    {
        const uint32_t two = at < dims ? *reinterpret_cast<const uint32_t *>(rowAt(n) + at * 2) : 0;
        some |= (two & kExponent) == kExponent || (two >> 16 & kExponent) == kExponent;
    }
    return __any(some);
}

// `count` rows of a matrix, up to 32, their columns 32 * part on times the columns of `weights`, to `sum`: row n, in memory at rowAt(n), to
// the columns of which seen(n); `all`: to all of them.
template<class T, class R, class F>
__device__ __forceinline__ void MultiplySeen(Acc16 &sum, const Acc16 &weights, int part, int dims, int count, bool all, R &&rowAt, F &&seen)
{
    using Words           = uint32_t __attribute__((ext_vector_type(4)));
    const uint32_t lane   = Again(threadIdx.x) & 63;
    const int      column = 32 * part + (int)(lane & 31);
#pragma unroll
    for (int half = 0; half < 2; ++half)
    {
        const Words packed = __builtin_bit_cast(Words, RoundedHalf<T>(weights, half));
        Words       values = {};
#pragma unroll 1
        for (int n = 0; n < min(16, count - 16 * half); ++n)
        {
            // the half wave and the element that have row n of 16
            const bool     own     = lane >> 5 == (uint32_t)(n >> 2 & 1);
            const int      element = (n >> 3) * 4 + (n & 3), shift = 16 * (element & 1);
            const uint32_t value   = own && column < dims ? (uint32_t)reinterpret_cast<const uint16_t *>(rowAt(16 * half + n))[column] << shift : 0;
            Words          weight;
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                values[i] = (all ? values[i] : 0) | (i == element / 2 ? value : 0);
                weight[i] = own && i == element / 2 ? packed[i] & 0xFFFFu << shift : 0;
            }
            if (!all)
            {
                const bool takes = seen(16 * half + n);
                Acc16      one   = {};
                Multiply(one, __builtin_bit_cast(Vec8<T>, values), __builtin_bit_cast(Vec8<T>, weight));
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    sum[i] = takes ? sum[i] + one[i] : sum[i];
                }
            }
        }
        if (all)
        {
            Multiply(sum, __builtin_bit_cast(Vec8<T>, values), __builtin_bit_cast(Vec8<T>, packed));
        }
    }
}

// ---- sequences -----------------------------------------------------------------------------------------------------
// A sequence and one of its tiles.
struct SequenceTile
{
    int firstRow, rows, firstKey, keys; // of the sequence
    int tile;                           // -1: there is none of that number
};

// Sum over the 64 lanes, as one number.
__device__ __forceinline__ uint32_t WaveTotal(uint32_t v)
{
    v += LaneStep<0>(v);
    v += LaneStep<1>(v);
    v += LaneStep<2>(v);
    v += LaneStep<3>(v);
    v += LaneStep<4>(v);
    v += LaneStep<5>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Tile `t` of all sequences' tiles, of `size` rows each, a token having `each` rows (of keys: `ofKeys`). Every wave finds it by itself.
// With `causal` a sequence's last tiles of rows have the most keys, its first tiles of keys the most rows. They come first, of all
// sequences (up to 64 of them), so that the workgroups that begin last are short ones (the gradient of 8 sequences of up to
// 2048 tokens, 32 heads on 8 of 128 elements, 863 us, 835 with it).
__device__ __forceinline__ SequenceTile FindTile(const AttentionSequences &s, uint32_t t, uint32_t most, int size, int each, bool ofKeys, bool causal)
{
    const int lane = (int)(threadIdx.x & 63);
    // the lane's sequence, with all that a tile needs of it, and its tiles
    SequenceTile own;
    uint32_t     tiles;
    auto         look = [&](int base)
    {
        const int b = min(base + lane, s.count - 1);
        own.firstRow = s.firstRow(b), own.rows = s.rowsOf(b, own.firstRow);
        own.firstKey = s.firstKey(b), own.keys = s.keysOf(b, own.firstKey);
        tiles = base + lane < s.count ? ((uint32_t)(ofKeys ? own.keys : own.rows) * (uint32_t)each + (uint32_t)size - 1) / (uint32_t)size : 0;
    };
    auto found = [&](int at, uint32_t tile)
    {
        return SequenceTile{__builtin_amdgcn_readlane(own.firstRow, at), __builtin_amdgcn_readlane(own.rows, at), __builtin_amdgcn_readlane(own.firstKey, at),
                            __builtin_amdgcn_readlane(own.keys, at), (int)tile};
    };
    if (causal && s.count <= 64)
    {
        look(0);
        // of the tiles that have at least `low` less heavy ones in their sequence there are more than t
        auto     of  = [&](uint32_t less) { return WaveTotal(tiles > less ? tiles - less : 0); };
        uint32_t low = 0, high = WaveLargest(tiles);
        if (of(0) <= t)
        {
            return {0, 0, 0, 0, -1};
        }
        while (high - low > 1)
        {
            const uint32_t middle = (low + high) / 2;
            of(middle) > t ? low = middle : high = middle;
        }
        const uint32_t rank = t - of(low + 1);
        const uint64_t some = __ballot(tiles > low);
        const uint32_t at   = __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
        const int      b    = (int)__builtin_ctzll(__ballot(tiles > low && at == rank));
        return found(b, ofKeys ? (uint32_t)__builtin_amdgcn_readlane((int)tiles, b) - 1 - low : low);
    }
    t               = causal && !ofKeys ? most - 1 - t : t;
    uint32_t before = 0; // tiles of the sequences that were looked at
    for (int base = 0; base < s.count; base += 64)
    {
        look(base);
        uint32_t upTo = tiles; // this sequence's and those of the lanes before
#pragma unroll
        for (int d = 1; d < 64; d *= 2)
        {
            const uint32_t v = __shfl_up(upTo, d);
            upTo += lane >= d ? v : 0;
        }
        const uint64_t behind = __ballot(before + upTo > t);
        if (behind != 0)
        {
            const int at = (int)__builtin_ctzll(behind);
            return found(at, t - before - ((uint32_t)__builtin_amdgcn_readlane((int)upTo, at) - (uint32_t)__builtin_amdgcn_readlane((int)tiles, at)));
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)upTo, 63);
    }
    return {0, 0, 0, 0, -1};
}

// The rows that a key head serves, as one matrix: row r of a sequence is head r % group of token r / group.
struct GroupRows
{
    DivBy group;

    __device__ __forceinline__ int size() const
    {
        return (int)group.d;
    }

    __device__ __forceinline__ int token(int r) const
    {
        return (int)group.Quotient((uint32_t)r);
    }
};

// The last key that token i of a sequence sees.
__device__ __forceinline__ int LimitOf(bool causal, const SequenceTile &s, int i)
{
    return causal ? i + s.keys - s.rows : s.keys - 1;
}

// Row r of that matrix. One behind the sequence's end counts as its last one, so that it changes no tile's borders.
struct AttentionRow
{
    int  token, head; // in q and out
    int  limit;
    bool there;

    __device__ __forceinline__ AttentionRow(const GroupRows &rows, bool causal, const SequenceTile &s, int keyHead, int r)
    {
        const int all = s.rows * rows.size(), at = min(r, all - 1), i = rows.token(at);
        token = s.firstRow + i;
        head  = keyHead * rows.size() + (at - i * rows.size());
        limit = LimitOf(causal, s, i);
        there = r < all;
    }
};

} // namespace cvamd

#endif // CVCUDA_AMD_ATTENTIONTILES_HPP
