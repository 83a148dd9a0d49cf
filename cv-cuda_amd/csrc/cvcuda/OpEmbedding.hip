// Lookup of rows of a table by token, and the table's gradient (formulas: cvcuda/Embedding.h). Both are bound by memory.
#include "RowOps.hpp"

#include <cvcuda/Embedding.h>

#include <algorithm>
#include <cmath>

namespace cvamd {

namespace {

struct LookupArgs
{
    RowPlaces   table, out;
    const void *tokens;
    int32_t     wide; // tokens of 64 bits
    int32_t     count, vocabulary, columns;
    float       scale;
    DivBy       runs; // of a row
};

__device__ __forceinline__ int64_t TokenAt(const void *tokens, int wide, int64_t i)
{
    return wide ? static_cast<const int64_t *>(tokens)[i] : static_cast<const int32_t *>(tokens)[i];
}

// The columns of a lane: N from `first` on. It loads N from `from` on, which lies before `first` where the row ends within
// them, so that every lane loads as all others do (loads under a condition wait for one another); the first `skip` are then not
// its own. It stores what it loaded: twice the same sums, where another lane has these columns too. Not where they are added to
// the table (ACCUMULATE): there it stores its own. NARROW: rows of fewer than N columns, one by one.
template<int N, bool NARROW, bool ACCUMULATE>
struct LaneColumns
{
    int first, from, columns;

    __device__ __forceinline__ LaneColumns(uint32_t tile, int of)
        : first((int)(tile * 64 + (threadIdx.x & 63)) * N)
        , from(max(0, min(first, of - N)))
        , columns(of)
    {
    }

    template<class T>
    __device__ __forceinline__ Run<T, N> get(const T *row) const
    {
        if constexpr (!NARROW)
        {
            return *reinterpret_cast<const Run<T, N> *>(row + from);
        }
        Run<T, N> r;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            r.v[i] = row[min(i, columns - 1)];
        }
        return r;
    }

    // s, which is not to be added to what is there
    template<class O>
    __device__ __forceinline__ void set(O *row, const float (&s)[N], float scale) const
    {
        if (first >= columns)
        {
            return;
        }
        if constexpr (!NARROW)
        {
            Run<O, N> r;
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                r.v[i] = FromFloat<O>(s[i] * scale);
            }
            *reinterpret_cast<Run<O, N> *>(row + from) = r;
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            if (i < columns)
            {
                row[i] = FromFloat<O>(s[i] * scale);
            }
        }
    }

    // s into a row of the table, of which `old` is what get() gave: to add to where ACCUMULATE
    template<class O>
    __device__ __forceinline__ void put(O *row, const float (&s)[N], float scale, const Run<O, N> &old) const
    {
        if constexpr (!ACCUMULATE)
        {
            set(row, s, scale);
            return;
        }
        Run<O, N> r;
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            r.v[i] = FromFloat<O>((float)old.v[i] + s[i] * scale);
        }
        if (first + N <= columns)
        {
            *reinterpret_cast<Run<O, N> *>(row + first) = r;
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            const int c = from + i;
            if (c >= first && c < columns)
            {
                row[c] = r.v[i];
            }
        }
    }

    template<class O>
    __device__ __forceinline__ void put(O *row, const float (&s)[N], float scale) const
    {
        put(row, s, scale, ACCUMULATE ? get(row) : Run<O, N>{});
    }
};

// Columns of a lane of a lookup: what makes 16 bytes of the narrower type.
template<class T, class O>
constexpr int kLookupRun = sizeof(T) < sizeof(O) ? kRunOf<T> : kRunOf<O>;

constexpr int kLookupRuns = 2, kLookupGroup = 256 * kLookupRuns; // of a lane, all on their way before the first is used; of a workgroup

// The runs of all rows are numbered through, so that narrow rows fill the lanes as well. The last run of a row whose width is no
// multiple begins earlier, as in LaneColumns. The token is read before its row: two waits for memory, which other waves fill.
// 32768 rows of 2048 from F32 to BF16 45 us, 5.0 TB/s; eight rows of 4096 3 us.
template<class T, class O, bool NARROW>
__global__ __launch_bounds__(256) void EmbeddingKernel(const LookupArgs a)
{
    constexpr int  N    = kLookupRun<T, O>;
    const uint32_t runs = a.runs.d; // of a row
    for (uint64_t first = (uint64_t)blockIdx.x * kLookupGroup; first < (uint64_t)a.count * runs; first += (uint64_t)gridDim.x * kLookupGroup)
    {
        const uint32_t row0 = (uint32_t)(first / runs), run0 = (uint32_t)(first - (uint64_t)row0 * runs);
        uint32_t       row[kLookupRuns];
        int            from[kLookupRuns];
        int64_t        token[kLookupRuns];
#pragma unroll
        for (int k = 0; k < kLookupRuns; ++k)
        {
            const uint32_t at = run0 + k * 256 + threadIdx.x, rows = a.runs.Quotient(at);
            row[k]   = row0 + rows;
            from[k]  = max(0, min((int)(at - rows * runs) * N, a.columns - N));
            token[k] = TokenAt(a.tokens, a.wide, min(row[k], (uint32_t)a.count - 1));
        }
        Run<T, N> r[kLookupRuns];
        bool      known[kLookupRuns];
#pragma unroll
        for (int k = 0; k < kLookupRuns; ++k)
        {
            known[k] = token[k] >= 0 && token[k] < a.vocabulary;
            r[k]     = {};
            if (a.vocabulary > 0) // (of the whole launch)
            {
                const T *p = reinterpret_cast<const T *>(a.table.at(known[k] ? (uint32_t)token[k] : 0));
                if constexpr (!NARROW)
                {
                    r[k] = *reinterpret_cast<const Run<T, N> *>(p + from[k]);
                }
                else
                {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                    {
                        r[k].v[i] = p[min(i, a.columns - 1)];
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kLookupRuns; ++k)
        {
            if (row[k] >= (uint32_t)a.count)
            {
                continue;
            }
            O        *to = reinterpret_cast<O *>(a.out.at(row[k]));
            Run<O, N> o;
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                o.v[i] = FromFloat<O>(known[k] ? (float)r[k].v[i] * a.scale : 0.f);
            }
            if constexpr (!NARROW)
            {
                *reinterpret_cast<Run<O, N> *>(to + from[k]) = o;
            }
            else
            {
#pragma unroll
                for (int i = 0; i < N; ++i)
                {
                    if (i < a.columns)
                    {
                        to[i] = o.v[i];
                    }
                }
            }
        }
    }
}

// ---- gradient: tokens in order ---------------------------------------------------------------------------------------
// The positions of equal tokens have to stand together, in their order. Tokens become keys (one that has no part in the
// gradient the key V, behind all others), and (key, position) are sorted by digits from the lowest up, each pass stable: the
// place of an element is the number of those with a smaller digit, and of those before it with the same one. Within a wave that
// number comes from the lanes that share the digit: a ballot for each bit of it.
struct TokenSource
{
    const void *tokens;
    int32_t     wide, count, vocabulary;
    int64_t     padding;

    __device__ __forceinline__ uint32_t key(uint32_t i) const
    {
        // (past the last one a load of that: loads under a condition wait for one another)
        const int64_t t = TokenAt(tokens, wide, min(i, (uint32_t)count - 1));
        return t >= 0 && t < vocabulary && t != padding && i < (uint32_t)count ? (uint32_t)t : (uint32_t)vocabulary;
    }
};

// The lanes of the wave whose digit of BITS bits is this lane's.
template<int BITS>
__device__ __forceinline__ uint64_t LanesOfDigit(uint32_t digit)
{
    uint64_t same = ~0ull;
#pragma unroll
    for (int b = 0; b < BITS; ++b)
    {
        const bool     set = (digit >> b) & 1;
        const uint64_t on  = __ballot(set);
        same &= set ? on : ~on;
    }
    return same;
}

__device__ __forceinline__ int LanesBefore(uint64_t lanes)
{
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
}

// Counts this lane's digit in its wave's counters and gives the number of those before it. (the wave's lanes go through here
// together and LDS serves a wave in order: all read before one of each digit writes)
template<int BITS>
__device__ __forceinline__ uint32_t CountDigit(volatile uint32_t *counters, uint32_t digit)
{
    const uint64_t same   = LanesOfDigit<BITS>(digit);
    const int      before = LanesBefore(same);
    const uint32_t had    = counters[digit];
    __builtin_amdgcn_wave_barrier();
    if (before == 0)
    {
        counters[digit] = had + (uint32_t)__popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
    return had + before;
}

// Inclusive sum over the lanes before and this one.
__device__ __forceinline__ uint32_t WaveScan(uint32_t v)
{
#pragma unroll
    for (int s = 1; s < 64; s <<= 1)
    {
        const uint32_t o = __shfl_up(v, s);
        v += (int)(threadIdx.x & 63) >= s ? o : 0;
    }
    return v;
}

// The sum of the first `n` of N numbers in LDS: all of them on their way at once.
template<int N>
__device__ __forceinline__ uint32_t SumOfFirst(const uint32_t (&v)[N], uint32_t n)
{
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
        s += (uint32_t)i < n ? v[i] : 0;
    }
    return s;
}

// `bytes` from `p` on, which begins with an element of 2 or 4 bytes, by a wave: 16 bytes per lane from the first multiple of 16
// on, as streaming stores.
__device__ __forceinline__ void ClearBytes(uint8_t *p, int64_t bytes, int element)
{
    typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
    const int64_t lane = threadIdx.x & 63, head = min((int64_t)(-reinterpret_cast<uintptr_t>(p) & 15), bytes);
    const int64_t body = (bytes - head) / 16 * 16, tail = bytes - head - body;
    for (int64_t i = lane * 16; i < body; i += 64 * 16)
    {
        __builtin_nontemporal_store(U32x4{0, 0, 0, 0}, reinterpret_cast<U32x4 *>(p + head + i));
    }
    // the ends: up to seven elements each
    const int64_t at = lane < 16 ? lane * element : head + body + (lane - 16) * element;
    if (lane < 16 ? at < head : at < head + body + tail)
    {
        element == 4 ? (void)(*reinterpret_cast<uint32_t *>(p + at) = 0) : (void)(*reinterpret_cast<uint16_t *>(p + at) = 0);
    }
}

// Rows of the table that are cleared beside the sort, whose few workgroups leave the card to others: by the workgroups of a
// launch from the `sorting`-th on. What tokens name among them is written once more by the sums.
struct ClearArgs
{
    RowPlaces table;
    int64_t   rowBytes;
    int32_t   element;
    int32_t   dense; // rows follow one another without a gap: cleared as pieces of kClearBytes
    uint32_t  row, rows;
    uint32_t  sorting;
};

constexpr int kClearBytes = 16384;

__device__ __forceinline__ void ClearBeside(const ClearArgs &a)
{
    const uint32_t waves = blockDim.x / 64;
    const int64_t  bytes = a.rows * a.rowBytes, parts = a.dense ? (bytes + kClearBytes - 1) / kClearBytes : a.rows;
    for (int64_t p = (int64_t)(blockIdx.x - a.sorting) * waves + WaveOfGroup(); p < parts; p += (int64_t)(gridDim.x - a.sorting) * waves)
    {
        if (a.dense)
        {
            ClearBytes(a.table.at(a.row) + p * kClearBytes, min((int64_t)kClearBytes, bytes - p * kClearBytes), a.element);
        }
        else
        {
            ClearBytes(a.table.at(a.row + (uint32_t)p), a.rowBytes, a.element);
        }
    }
}

constexpr int kSmallThreads = 1024, kSmallBits = 6;
constexpr int kMostSmall    = 4 * kSmallThreads;

// All of up to K * 1024 tokens by one workgroup, in LDS. A wave owns 64 K consecutive elements; 16 waves with 64 digits
// each have a counter per thread. 1003 tokens among 30011 7 us: three passes, one wait after another.
template<int K>
__global__ __launch_bounds__(kSmallThreads) void EmbeddingSortSmallKernel(const TokenSource src, uint32_t *keys, uint32_t *places, int bits,
                                                                         const ClearArgs clear)
{
    if (blockIdx.x > 0)
    {
        ClearBeside(clear);
        return;
    }
    __shared__ uint32_t s_key[K * kSmallThreads];
    __shared__ uint16_t s_place[K * kSmallThreads];
    __shared__ uint32_t s_count[16][1 << kSmallBits];
    __shared__ uint32_t s_sum[16];
    const uint32_t      wave = threadIdx.x >> 6, lane = threadIdx.x & 63, first = wave * 64 * K + lane;
    uint32_t            key[K], place[K], rank[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
        place[k] = first + 64 * k;
        key[k]   = src.key(place[k]);
    }
    for (int shift = 0; shift < bits; shift += kSmallBits)
    {
        s_count[wave][lane] = 0; // (a wave's own)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            rank[k] = CountDigit<kSmallBits>(s_count[wave], (key[k] >> shift) & 63);
        }
        __syncthreads();
        // what comes before each counter, by digit and then by wave: thread t holds digit t / 16 of wave t % 16
        const uint32_t mine = s_count[threadIdx.x & 15][threadIdx.x >> 4], upTo = WaveScan(mine);
        if (lane == 63)
        {
            s_sum[wave] = upTo;
        }
        __syncthreads();
        s_count[threadIdx.x & 15][threadIdx.x >> 4] = upTo - mine + SumOfFirst(s_sum, wave);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            const uint32_t to = s_count[wave][(key[k] >> shift) & 63] + rank[k];
            s_key[to]         = key[k];
            s_place[to]       = (uint16_t)place[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            key[k]   = s_key[first + 64 * k];
            place[k] = s_place[first + 64 * k];
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
        if (first + 64 * k < (uint32_t)src.count)
        {
            keys[first + 64 * k]   = key[k];
            places[first + 64 * k] = place[k];
        }
    }
}

// More tokens: tiles of them, two launches for each digit. The first counts the digits of each tile, the second adds up what
// comes before each digit of its tile and puts the tile's elements there. 65536 tokens among 128000 38 us, the time in which 128 MiB
// of the table are cleared beside it.
constexpr int kTileThreads = 512, kTileBits = 9, kDigits = 1 << kTileBits;

// Keys of a thread. Small tiles are quick, but each reads the counts of all others: 64 small ones at most (16384 tokens' sort 30 us,
// 35 with four keys), then 128 of eight, then sixteen.
constexpr int KeysOf(int64_t tokens)
{
    return tokens <= 64 * 2 * kTileThreads ? 2 : tokens <= 128 * 8 * kTileThreads ? 8 : 16;
}

constexpr int kCountsAtOnce = 16; // of tiles that a thread reads: a digit's counts are padded to as many

struct TileArgs
{
    TokenSource     src;
    const uint32_t *keys, *places; // nullptr: the tokens themselves, at their places
    uint32_t       *toKeys, *toPlaces;
    uint32_t       *counts; // [kDigits][pitch]
    int32_t         tiles, pitch, shift;

    __device__ __forceinline__ uint32_t key(uint32_t i) const
    {
        if (keys == nullptr)
        {
            return src.key(i);
        }
        const uint32_t k = keys[min(i, (uint32_t)src.count - 1)];
        return i < (uint32_t)src.count ? k : (uint32_t)src.vocabulary;
    }
};

template<int KEYS>
__global__ __launch_bounds__(kTileThreads) void EmbeddingCountKernel(const TileArgs a, const ClearArgs clear)
{
    if (blockIdx.x >= clear.sorting)
    {
        ClearBeside(clear);
        return;
    }
    __shared__ uint32_t s_count[kDigits];
    const uint32_t      first = blockIdx.x * (KEYS * kTileThreads) + threadIdx.x;
    uint32_t            key[KEYS];
    s_count[threadIdx.x] = 0;
#pragma unroll
    for (int k = 0; k < KEYS; ++k)
    {
        key[k] = a.key(first + k * kTileThreads);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KEYS; ++k)
    {
        if (first + k * kTileThreads < (uint32_t)a.src.count)
        {
            atomicAdd(&s_count[(key[k] >> a.shift) & (kDigits - 1)], 1u);
        }
    }
    __syncthreads();
    a.counts[(size_t)threadIdx.x * a.pitch + blockIdx.x] = s_count[threadIdx.x];
}

template<int KEYS>
__global__ __launch_bounds__(kTileThreads) void EmbeddingPlaceKernel(const TileArgs a, const ClearArgs clear)
{
    if (blockIdx.x >= clear.sorting)
    {
        ClearBeside(clear);
        return;
    }
    constexpr int       kWaves = kTileThreads / 64;
    __shared__ uint32_t s_count[kWaves][kDigits];
    __shared__ uint32_t s_sum[kWaves];
    const uint32_t      wave = threadIdx.x >> 6, lane = threadIdx.x & 63, first = blockIdx.x * (KEYS * kTileThreads) + wave * 64 * KEYS + lane;
    uint32_t            key[KEYS], place[KEYS], rank[KEYS];
#pragma unroll
    for (int k = 0; k < KEYS; ++k)
    {
        const uint32_t i = first + 64 * k;
        key[k]           = a.key(i);
        place[k]         = a.keys == nullptr ? i : a.places[min(i, (uint32_t)a.src.count - 1)];
    }
    for (int w = 0; w < kWaves; ++w)
    {
        s_count[w][threadIdx.x] = 0;
    }
    // thread d: the elements of digit d before this tile, and all of them
    const uint32_t *row = a.counts + (size_t)threadIdx.x * a.pitch;
    uint32_t        before = 0, all = 0;
    for (int t = 0; t < a.pitch; t += kCountsAtOnce)
    {
        const Run<uint32_t, kCountsAtOnce> c = *reinterpret_cast<const Run<uint32_t, kCountsAtOnce> *>(row + t);
#pragma unroll
        for (int i = 0; i < kCountsAtOnce; ++i)
        {
            before += t + i < (int)blockIdx.x ? c.v[i] : 0;
            all += t + i < a.tiles ? c.v[i] : 0;
        }
    }
    const uint32_t upTo = WaveScan(all);
    if (lane == 63)
    {
        s_sum[wave] = upTo;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KEYS; ++k)
    {
        // (past the last token: the highest digit, behind all others of the last tile)
        const uint32_t digit = first + 64 * k < (uint32_t)a.src.count ? (key[k] >> a.shift) & (kDigits - 1) : kDigits - 1;
        rank[k]              = CountDigit<kTileBits>(s_count[wave], digit);
    }
    uint32_t base = before + upTo - all + SumOfFirst(s_sum, wave);
    __syncthreads();
    for (int w = 0; w < kWaves; ++w)
    {
        const uint32_t c        = s_count[w][threadIdx.x];
        s_count[w][threadIdx.x] = base;
        base += c;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KEYS; ++k)
    {
        if (first + 64 * k < (uint32_t)a.src.count)
        {
            const uint32_t to = s_count[wave][(key[k] >> a.shift) & (kDigits - 1)] + rank[k];
            a.toKeys[to]      = key[k];
            a.toPlaces[to]    = place[k];
        }
    }
}

// ---- gradient: sums ----------------------------------------------------------------------------------------------------
// The sorted positions are cut into pieces of PIECE, whatever their tokens: every wave adds up the same number of rows, of 64
// lanes' columns. A token whose positions lie within a piece is done there. What reaches over a piece's ends is joined by the
// workgroup, whose waves have pieces that follow one another, and what reaches over the workgroup's is left in the workspace,
// where a second launch adds it up: always in the order of the positions. Rows of the table that no token names are cleared
// beside that by waves that look for their keys among the sorted ones.
constexpr int kSumWaves = 8, kSmallPiece = 8, kPiece = 32, kFewTokens = kSumWaves * kSmallPiece;

// Small pieces where there are too few to fill the card (2^24 elements are 1024 waves of large ones): their time is that of
// one wait after another (1003 tokens of width 515 28 -> 21.5 us, 16384 of 64 40 -> 32; 16384 of 4096 would take 141 for 135).
constexpr int PieceOf(int64_t tokens, int64_t columns)
{
    return tokens <= kFewTokens || tokens * columns <= 1 << 24 ? kSmallPiece : kPiece;
}

struct SumArgs
{
    RowPlaces       grad, table;
    const uint32_t *keys, *places;
    float          *partial; // [groups][2][columns]: of the token that began before the group, of the one that goes on behind it
    int32_t         count, vocabulary, columns, accumulate;
    uint32_t        groups, group; // workgroups' shares of the positions, and how many that is
    uint32_t        columnTiles, joinTiles, sumGroups, clearGroups, clearRows;
    uint32_t        rowsToClear; // the others have been
    int32_t         dense;       // the table's rows follow one another without a gap
    float           scale;
};

// A wave clears as many rows as make 16 KiB, 32 at most: what all waves write lies close together at any time (16 rows of
// 2048 floats each: 5.3 TB/s).
constexpr int kMostClearRows = 32;

// The first place among `n` sorted keys that holds `key` or more.
__device__ __forceinline__ uint32_t FirstOf(const uint32_t *keys, uint32_t n, uint32_t key)
{
    uint32_t lo = 0; // keys before it are less
    uint32_t len = n;
    while (len > 0)
    {
        // 64 places of the rest at once
        const uint32_t step = (len + 63) / 64, at = lo + (threadIdx.x & 63) * step;
        const uint64_t less = __ballot(at < lo + len && keys[at] < key);
        const uint32_t k    = (uint32_t)__popcll(less);
        if (k == 0)
        {
            break;
        }
        const uint32_t end = min(lo + len, lo + k * step);
        lo += (k - 1) * step + 1;
        len = end - lo;
    }
    return lo;
}

// Clears the rows from row0 on that have no bit in `named`; what follows one another without a gap as one run of bytes.
template<class O>
__device__ __forceinline__ void ClearNotNamed(const SumArgs &a, uint32_t row0, uint32_t rows, uint32_t named)
{
    for (uint32_t r = 0; r < rows;)
    {
        if ((named >> r) & 1)
        {
            ++r;
            continue;
        }
        const uint32_t many = a.dense ? min(rows - r, (uint32_t)__builtin_ctzll((named >> r) | 1ull << 32)) : 1;
        ClearBytes(a.table.at(row0 + r), (int64_t)many * a.columns * (int64_t)sizeof(O), (int)sizeof(O));
        r += many;
    }
}

template<class O>
__device__ __forceinline__ void ClearRows(const SumArgs &a, uint32_t wave)
{
    const uint32_t lane = threadIdx.x & 63, row0 = wave * a.clearRows, rows = min(a.clearRows, a.rowsToClear - row0);
    const uint32_t lo = FirstOf(a.keys, a.count, row0), key = lo + lane < (uint32_t)a.count ? a.keys[lo + lane] : 0xFFFFFFFFu;
    const uint64_t here  = __ballot(key < row0 + rows);
    uint32_t       named = 0;
    if (here != ~0ull)
    {
        for (uint64_t rest = here; rest != 0;) // a key at a time
        {
            const uint32_t one = (uint32_t)__builtin_amdgcn_readlane(key, __builtin_ctzll(rest));
            named |= 1u << (one - row0);
            rest &= ~__ballot(key == one);
        }
    }
    else
    {
        // more keys than lanes, of frequent tokens: lane r looks for row r's (64 at a time the first rows of 65536 words took 90 us)
        uint32_t from = lo, many = (uint32_t)a.count - lo;
        while (__ballot(many > 0) != 0)
        {
            const uint32_t half = many / 2;
            if (many > 0)
            {
                const bool less = a.keys[from + half] < row0 + lane;
                from            = less ? from + half + 1 : from;
                many            = less ? many - half - 1 : half;
            }
        }
        named = (uint32_t)__ballot(lane < rows && from < (uint32_t)a.count && a.keys[min(from, (uint32_t)a.count - 1)] == row0 + lane);
    }
    ClearNotNamed<O>(a, row0, rows, named);
}

// What a piece leaves of the tokens that reach over its ends, and whether: its first one began before it, that one goes on
// behind it as well, its last one goes on behind it.
enum PieceFlags
{
    kHead       = 1,
    kHeadGoesOn = 2,
    kTail       = 4
};

// Sums a piece: tokens within it into the table, the others into `head` and `tail`, a lane's N one after another. Returns the flags.
template<class T, class O, int PIECE, bool ACCUMULATE, class COLUMNS, int N>
__device__ __forceinline__ uint32_t SumPiece(const SumArgs &a, uint32_t piece, const COLUMNS &columns, float (&head)[64][N], float (&tail)[64][N])
{
    // rows that are loaded at once; what they are added to comes with them (read where a sum is done it was a wait for each
    // token: 20000 tokens of width 4096, BF16, 98 us, so 88; many rows of F32 178, so 188)
    constexpr int  kBatch = PIECE < 16 || ACCUMULATE ? 8 : 16;
    const uint32_t lane = threadIdx.x & 63, first = piece * PIECE, many = min((uint32_t)PIECE, (uint32_t)a.count - first);
    // lane k: the piece's k-th key and place (behind its end the last one's); the keys before and behind the piece
    const uint32_t mine  = first + min(lane, many - 1);
    const uint32_t myKey = a.keys[mine], myPlace = a.places[mine];
    const uint32_t before = first > 0 ? a.keys[first - 1] : 0xFFFFFFFFu;
    const uint32_t behind = first + many < (uint32_t)a.count ? a.keys[first + many] : 0xFFFFFFFFu;

    uint32_t flags = 0;
    float    s[N]  = {};
    bool     open  = (uint32_t)__builtin_amdgcn_readlane(myKey, 0) == before; // the sum began in an earlier piece
    for (uint32_t k0 = 0; k0 < many; k0 += kBatch)
    {
        Run<T, N> row[kBatch];
        Run<O, N> old[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
        {
            row[j] = columns.get(reinterpret_cast<const T *>(a.grad.at(__builtin_amdgcn_readlane(myPlace, k0 + j))));
            if constexpr (ACCUMULATE)
            {
                const uint32_t key = __builtin_amdgcn_readlane(myKey, k0 + j);
                old[j]             = columns.get(reinterpret_cast<const O *>(a.table.at(min(key, (uint32_t)a.vocabulary - 1))));
            }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
        {
            const uint32_t k   = k0 + j;
            const uint32_t key = __builtin_amdgcn_readlane(myKey, k);
            if (k >= many || key == (uint32_t)a.vocabulary)
            {
                return flags; // (all others are behind the table's last row)
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                s[i] += (float)row[j].v[i];
            }
            const uint32_t next = k + 1 < many ? (uint32_t)__builtin_amdgcn_readlane(myKey, k + 1) : behind;
            if (next == key && k + 1 < many)
            {
                continue;
            }
            if (!open && next != key)
            {
                columns.put(reinterpret_cast<O *>(a.table.at(key)), s, a.scale, old[j]);
            }
            else
            {
                float (&to)[N] = open ? head[lane] : tail[lane];
#pragma unroll
                for (int i = 0; i < N; ++i)
                {
                    to[i] = s[i];
                }
                flags |= !open ? kTail : next == key ? kHead | kHeadGoesOn : kHead;
            }
            open = false;
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                s[i] = 0;
            }
        }
    }
    return flags;
}

// kSumWaves pieces that follow one another, of 64 lanes' columns.
template<class T, class O, int PIECE, bool NARROW, bool ACCUMULATE>
__device__ __forceinline__ void SumGroup(const SumArgs &a, uint32_t group, uint32_t tile)
{
    constexpr int       N = kRunOf<T>;
    __shared__ float    s_head[kSumWaves][64][N], s_tail[kSumWaves][64][N];
    __shared__ uint32_t s_flags[kSumWaves];
    const LaneColumns<N, NARROW, ACCUMULATE> columns(tile, a.columns);

    const uint32_t wave = WaveOfGroup(), lane = threadIdx.x & 63, piece = group * kSumWaves + wave;
    uint32_t       flags = 0;
    if ((uint64_t)piece * PIECE < (uint64_t)a.count)
    {
        flags = SumPiece<T, O, PIECE, ACCUMULATE>(a, piece, columns, s_head[wave], s_tail[wave]);
    }
    if (lane == 0)
    {
        s_flags[wave] = flags;
    }
    __syncthreads();
    if (wave == 0)
    {
        bool  here = false, any = false; // of the sum that is open: began in this group; there is one
        float s[N] = {};
        for (uint32_t w = 0; w < kSumWaves; ++w)
        {
            const uint32_t f = __builtin_amdgcn_readfirstlane(s_flags[w]);
            if (f & kHead)
            {
                any = true;
#pragma unroll
                for (int i = 0; i < N; ++i)
                {
                    s[i] += s_head[w][lane][i];
                }
                if (!(f & kHeadGoesOn))
                {
                    if (here)
                    {
                        const uint32_t key = __builtin_amdgcn_readfirstlane(a.keys[(size_t)(group * kSumWaves + w) * PIECE]);
                        columns.put(reinterpret_cast<O *>(a.table.at(key)), s, a.scale);
                    }
                    else
                    {
                        columns.set(a.partial + (size_t)group * 2 * a.columns, s, 1.f);
                    }
                    any = false;
                }
            }
            if (f & kTail)
            {
                here = any = true;
#pragma unroll
                for (int i = 0; i < N; ++i)
                {
                    s[i] = s_tail[w][lane][i];
                }
            }
        }
        if (any)
        {
            columns.set(a.partial + ((size_t)group * 2 + (here ? 1 : 0)) * a.columns, s, 1.f);
        }
    }
    __syncthreads(); // (before the next group's)
}

// A workgroup is one of tokens, or waves that clear rows. 65536 tokens of width 2048, BF16, into 128000 rows of F32, of which the
// sort has cleared some: 215 us, 5.3 TB/s.
template<class T, class O, int PIECE, bool NARROW, bool ACCUMULATE>
__global__ __launch_bounds__(64 * kSumWaves) void EmbeddingSumKernel(const SumArgs a)
{
    if (blockIdx.x >= a.sumGroups)
    {
        const uint64_t waves = ((uint64_t)a.rowsToClear + a.clearRows - 1) / a.clearRows;
        for (uint64_t w = (uint64_t)(blockIdx.x - a.sumGroups) * kSumWaves + WaveOfGroup(); w < waves; w += (uint64_t)a.clearGroups * kSumWaves)
        {
            ClearRows<O>(a, (uint32_t)w);
        }
        return;
    }
    for (uint64_t w = blockIdx.x; w < (uint64_t)a.groups * a.columnTiles; w += a.sumGroups)
    {
        SumGroup<T, O, PIECE, NARROW, ACCUMULATE>(a, (uint32_t)(w / a.columnTiles), (uint32_t)(w % a.columnTiles));
    }
}

// Few tokens, a group of small pieces: one launch and no workspace. The workgroups that sum put all of them in order by themselves:
// the place of a key is the number of those that are less, and of the same ones before it. The waves that clear hold a key
// in each lane. Three tokens of width 640 added to a table 7 us a call, 12 with the sort; 64 of 4544 into 4625 rows 16, 21.
static_assert(kFewTokens == 64, "a key in each lane");

// Larger tables are cleared whole by a launch of their own, whose waves wait for no token: 1.01 GB 175 us, so 187; 123 MB 29, so 22.
constexpr int64_t kFewClearBytes = (int64_t)512 << 20;

// Clears rows that no key names, region by region as ClearRows.
template<class O>
__device__ __forceinline__ void ClearFew(const SumArgs &a, uint32_t key)
{
    const uint32_t waves = (a.rowsToClear + a.clearRows - 1) / a.clearRows;
    for (uint32_t w = (blockIdx.x - a.columnTiles) * kSumWaves + WaveOfGroup(); w < waves; w += a.clearGroups * kSumWaves)
    {
        const uint32_t row0 = w * a.clearRows, rows = min(a.clearRows, a.rowsToClear - row0);
        uint32_t       named = 0;
        for (uint64_t rest = __ballot(key - row0 < rows); rest != 0; rest &= rest - 1)
        {
            named |= 1u << ((uint32_t)__builtin_amdgcn_readlane(key, __builtin_ctzll(rest)) - row0);
        }
        ClearNotNamed<O>(a, row0, rows, named);
    }
}

// Clears the rows of a table.
__global__ __launch_bounds__(kSmallThreads) void EmbeddingClearKernel(const ClearArgs clear)
{
    ClearBeside(clear);
}

template<class T, class O, bool NARROW, bool ACCUMULATE>
__global__ __launch_bounds__(64 * kSumWaves) void EmbeddingFewKernel(const TokenSource src, SumArgs a)
{
    __shared__ uint32_t s_keys[kFewTokens], s_places[kFewTokens];
    const uint32_t      lane = threadIdx.x & 63, key = src.key(lane); // (behind the last one the table's length, as without a part in it)
    if (blockIdx.x >= a.columnTiles)
    {
        ClearFew<O>(a, key);
        return;
    }
    if (WaveOfGroup() == 0)
    {
        uint32_t place = 0;
#pragma unroll
        for (uint32_t j = 0; j < kFewTokens; ++j)
        {
            const uint32_t other = __builtin_amdgcn_readlane(key, j);
            place += other < key || (other == key && j < lane) ? 1 : 0;
        }
        s_keys[place]   = key;
        s_places[place] = lane;
    }
    __syncthreads();
    a.keys   = s_keys;
    a.places = s_places;
    SumGroup<T, O, kSmallPiece, NARROW, ACCUMULATE>(a, 0, blockIdx.x);
}

constexpr int kJoinRun = 4, kJoinWaves = 4; // columns of a lane; each wave adds up a part of the groups

// The sum of a token that begins in a group and goes on behind it.
template<class O, bool NARROW, bool ACCUMULATE>
__device__ __forceinline__ void JoinGroups(const SumArgs &a, uint32_t group, uint32_t tile)
{
    const uint64_t first = (uint64_t)group * a.group, behind = first + a.group;
    const uint32_t key = __builtin_amdgcn_readfirstlane(a.keys[behind - 1]);
    if (key == (uint32_t)a.vocabulary || a.keys[behind] != key || (group > 0 && a.keys[first] == key && a.keys[first - 1] == key))
    {
        return;
    }
    constexpr int    N = kJoinRun, kAhead = 8;
    __shared__ float s_part[kJoinWaves][64][N];
    const LaneColumns<N, NARROW, ACCUMULATE> columns(tile, a.columns);
    // the group of the last of them, first: sums whose number is known are on their way together
    const uint32_t wave = WaveOfGroup(), lane = threadIdx.x & 63;
    const uint32_t all = (FirstOf(a.keys, a.count, key + 1) - 1) / a.group - group, each = (all + kJoinWaves - 1) / kJoinWaves;
    const uint32_t from = group + 1 + wave * each, to = min(group + 1 + all, from + each);
    float          s[N] = {};
    for (uint32_t p = from; p < to; p += kAhead)
    {
        Run<float, N> part[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
        {
            part[j] = columns.get(a.partial + (size_t)min(p + j, to - 1) * 2 * a.columns);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
        {
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                s[i] += p + j < to ? part[j].v[i] : 0.f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
    {
        s_part[wave][lane][i] = s[i];
    }
    __syncthreads();
    if (wave == 0)
    {
        const Run<float, N> began = columns.get(a.partial + ((size_t)group * 2 + 1) * a.columns);
#pragma unroll
        for (int i = 0; i < N; ++i)
        {
            s[i] = began.v[i];
#pragma unroll
            for (int w = 0; w < kJoinWaves; ++w)
            {
                s[i] += s_part[w][lane][i];
            }
        }
        columns.put(reinterpret_cast<O *>(a.table.at(key)), s, a.scale);
    }
    __syncthreads(); // (before the next group's)
}

// A workgroup per group but the last, which nothing follows, and 64 lanes' columns (3 to 6 us).
template<class O, bool NARROW, bool ACCUMULATE>
__global__ __launch_bounds__(64 * kJoinWaves) void EmbeddingJoinKernel(const SumArgs a)
{
    for (uint64_t w = blockIdx.x; w < (uint64_t)(a.groups - 1) * a.joinTiles; w += gridDim.x)
    {
        JoinGroups<O, NARROW, ACCUMULATE>(a, (uint32_t)(w / a.joinTiles), (uint32_t)(w % a.joinTiles));
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------
// Workgroups of one kind in a launch: a dimension of the grid holds fewer than 2^32 threads.
constexpr int kMostGroups = 1 << 21;

int64_t Parts(int64_t v, int64_t of)
{
    return (v + of - 1) / of;
}

int64_t RoundUp(int64_t v, int64_t to)
{
    return Parts(v, to) * to;
}

// Parts of the workspace, each from a multiple of 256 bytes on.
struct GradRoom
{
    int64_t keys, places, otherKeys, otherPlaces, counts, partial, bytes;

    GradRoom(int64_t tokens, int64_t columns)
    {
        const int64_t list = RoundUp(tokens * 4, 256), tiles = tokens > kMostSmall ? Parts(tokens, KeysOf(tokens) * kTileThreads) : 0;
        const int64_t groups = Parts(tokens, kSumWaves * PieceOf(tokens, columns));
        keys        = 0;
        places      = keys + list;
        otherKeys   = places + list;
        otherPlaces = otherKeys + (tiles > 0 ? list : 0);
        counts      = otherPlaces + (tiles > 0 ? list : 0);
        partial     = counts + RoundUp(tiles, kCountsAtOnce) * kDigits * 4;
        bytes       = tokens > kFewTokens ? partial + (groups > 1 ? groups * 2 * columns * 4 : 0) : 0;
    }
};

template<class T, class O>
void LaunchLookup(LookupArgs &a, hipStream_t stream)
{
    constexpr int N = kLookupRun<T, O>;
    a.runs          = DivBy((uint32_t)Parts(a.columns, N));
    const dim3 grid((uint32_t)std::min<int64_t>(Parts((int64_t)a.count * a.runs.d, kLookupGroup), kMostGroups));
    if (a.columns < N)
    {
        hipLaunchKernelGGL((EmbeddingKernel<T, O, true>), grid, dim3(256), 0, stream, a);
    }
    else
    {
        hipLaunchKernelGGL((EmbeddingKernel<T, O, false>), grid, dim3(256), 0, stream, a);
    }
    CheckLaunch("EmbeddingKernel");
}

// Rows that are cleared beside the sort, the table's last ones: all where that writes a quarter of them again at most, else what
// the card writes in the time that the sort takes (about 7 us for a workgroup's, 26 in four launches; the sums clear the others).
uint32_t RowsBesideSort(int64_t tokens, int64_t vocabulary, int64_t rowBytes)
{
    if (tokens == 0)
    {
        return 0;
    }
    const int64_t bytes = tokens <= kMostSmall ? 32 << 20 : 128 << 20;
    return (uint32_t)(tokens * 4 <= vocabulary ? vocabulary : std::min(vocabulary, bytes / rowBytes));
}

// Launches of a sort that clear rows beside it, each its share of those left.
struct Clearing
{
    ClearArgs args;
    uint32_t  left;   // rows
    int       launches;

    // The workgroups to add to `sorting`, each of `waves` waves.
    uint32_t next(uint32_t sorting, int waves)
    {
        args.row += args.rows;
        args.rows    = left / (uint32_t)launches + (left % (uint32_t)launches != 0 ? 1 : 0);
        args.sorting = sorting;
        left -= args.rows;
        --launches;
        const int64_t parts = args.dense ? Parts(args.rows * args.rowBytes, kClearBytes) : args.rows;
        return (uint32_t)std::min<int64_t>(Parts(parts, waves), 1 << 20);
    }
};

// Sorts into the workspace's keys and places.
void SortTokens(const TokenSource &src, uint8_t *room, const GradRoom &at, Clearing clearing, hipStream_t stream)
{
    auto     part = [&](int64_t offset) { return reinterpret_cast<uint32_t *>(room + offset); };
    uint32_t *keys = part(at.keys), *places = part(at.places);
    const int bits = src.vocabulary > 0 ? 32 - __builtin_clz((uint32_t)src.vocabulary) : 1;
    if (src.count <= kMostSmall)
    {
        clearing.launches   = 1;
        const uint32_t more = clearing.next(1, kSmallThreads / 64);
        auto           launch = [&](auto kernel)
        { hipLaunchKernelGGL(kernel, dim3(1 + more), dim3(kSmallThreads), 0, stream, src, keys, places, bits, clearing.args); };
        src.count <= kSmallThreads ? launch(EmbeddingSortSmallKernel<1>) : launch(EmbeddingSortSmallKernel<4>);
        CheckLaunch("EmbeddingSortSmallKernel");
        return;
    }
    const int64_t tiles = Parts(src.count, KeysOf(src.count) * kTileThreads);
    TileArgs a      = {src, nullptr, nullptr, nullptr, nullptr, part(at.counts), (int32_t)tiles, (int32_t)RoundUp(tiles, kCountsAtOnce), 0};
    int      passes = DivUp(bits, kTileBits);
    clearing.launches = 2 * passes;
    for (int p = 0; p < passes; ++p)
    {
        // the last pass ends in keys and places
        const bool to = (passes - 1 - p) % 2 == 0;
        a.toKeys      = to ? keys : part(at.otherKeys);
        a.toPlaces    = to ? places : part(at.otherPlaces);
        a.shift       = p * kTileBits;
        auto launch = [&](auto kernel)
        {
            const uint32_t more = clearing.next(a.tiles, kTileThreads / 64);
            hipLaunchKernelGGL(kernel, dim3(a.tiles + more), dim3(kTileThreads), 0, stream, a, clearing.args);
            CheckLaunch("EmbeddingSortKernel");
        };
        switch (KeysOf(src.count))
        {
        case 2:
            launch(EmbeddingCountKernel<2>);
            launch(EmbeddingPlaceKernel<2>);
            break;
        case 8:
            launch(EmbeddingCountKernel<8>);
            launch(EmbeddingPlaceKernel<8>);
            break;
        default:
            launch(EmbeddingCountKernel<16>);
            launch(EmbeddingPlaceKernel<16>);
        }
        a.keys   = a.toKeys;
        a.places = a.toPlaces;
    }
}

// All of a gradient of few tokens.
template<class T, class O, bool NARROW>
void LaunchFew(const TokenSource &src, const SumArgs &a, hipStream_t stream)
{
    const auto kernel = a.accumulate ? EmbeddingFewKernel<T, O, NARROW, true> : EmbeddingFewKernel<T, O, NARROW, false>;
    hipLaunchKernelGGL(kernel, dim3(a.columnTiles + a.clearGroups), dim3(64 * kSumWaves), 0, stream, src, a);
    CheckLaunch("EmbeddingFewKernel");
}

uint32_t Groups(int64_t groups)
{
    return (uint32_t)std::min<int64_t>(groups, kMostGroups);
}

template<class K>
void Launch(K plain, K accumulate, const SumArgs &a, uint32_t grid, int waves, hipStream_t stream)
{
    hipLaunchKernelGGL(a.accumulate ? accumulate : plain, dim3(grid), dim3(64 * waves), 0, stream, a);
}

template<class T, class O, int PIECE>
void LaunchSum(const SumArgs &a, uint32_t grid, hipStream_t stream)
{
    a.columns < kRunOf<T>
        ? Launch(EmbeddingSumKernel<T, O, PIECE, true, false>, EmbeddingSumKernel<T, O, PIECE, true, true>, a, grid, kSumWaves, stream)
        : Launch(EmbeddingSumKernel<T, O, PIECE, false, false>, EmbeddingSumKernel<T, O, PIECE, false, true>, a, grid, kSumWaves, stream);
}

template<class T, class O>
void LaunchGrad(const TokenSource &src, SumArgs &a, hipStream_t stream)
{
    a.columnTiles = (uint32_t)Parts(a.columns, 64 * kRunOf<T>);
    a.joinTiles   = (uint32_t)Parts(a.columns, 64 * kJoinRun);
    a.clearRows   = (uint32_t)std::max<int64_t>(1, std::min<int64_t>(kMostClearRows, kClearBytes / (a.columns * (int64_t)sizeof(O))));
    a.sumGroups   = Groups((int64_t)a.groups * a.columnTiles);
    a.clearGroups = Groups(Parts(Parts(a.rowsToClear, a.clearRows), kSumWaves));
    if (a.count > 0 && a.count <= kFewTokens)
    {
        a.columns < kRunOf<T> ? LaunchFew<T, O, true>(src, a, stream) : LaunchFew<T, O, false>(src, a, stream);
        return;
    }
    if (const uint32_t grid = a.sumGroups + a.clearGroups)
    {
        if (a.group == kSumWaves * kSmallPiece)
        {
            LaunchSum<T, O, kSmallPiece>(a, grid, stream);
        }
        else
        {
            LaunchSum<T, O, kPiece>(a, grid, stream);
        }
        CheckLaunch("EmbeddingSumKernel");
    }
    if (a.groups > 1)
    {
        const uint32_t grid = Groups((int64_t)(a.groups - 1) * a.joinTiles);
        a.columns < kJoinRun ? Launch(EmbeddingJoinKernel<O, true, false>, EmbeddingJoinKernel<O, true, true>, a, grid, kJoinWaves, stream)
                             : Launch(EmbeddingJoinKernel<O, false, false>, EmbeddingJoinKernel<O, false, true>, a, grid, kJoinWaves, stream);
        CheckLaunch("EmbeddingJoinKernel");
    }
}

struct Tokens
{
    const void *base;
    int32_t     count, wide;
};

Tokens TakeTokens(NVCVTensorHandle h)
{
    const DenseView v = RequireDense(h, "Tokens", NVCV_DATA_TYPE_NONE);
    if (v.dtype != NVCV_DATA_TYPE_S32 && v.dtype != NVCV_DATA_TYPE_S64)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tokens must be S32 or S64");
    }
    if (v.count > INT32_MAX)
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Too many tokens");
    }
    return {v.base, (int32_t)v.count, v.dtype == NVCV_DATA_TYPE_S64};
}

void RequireScale(float scale)
{
    if (!std::isfinite(scale))
    {
        throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Scale must be finite");
    }
}

class Embedding final : public IOperator
{
public:
    void submit(hipStream_t stream, NVCVTensorHandle htable, NVCVTensorHandle htokens, NVCVTensorHandle hout, float scale) const
    {
        const RowsView table = RequireRows(htable, "Table"), out = RequireRows(hout, "Output");
        const Tokens   tokens = TakeTokens(htokens);
        RequireScale(scale);
        if (out.rows != tokens.count || out.columns != table.columns)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Output must have a row per token (%d) with the table's elements (%d), not %d of %d",
                          tokens.count, table.columns, out.rows, out.columns);
        }
        if (out.elem != table.elem && table.elem != kRowF32)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Output must have the table's type, or the table's must be F32");
        }
        if (tokens.count == 0 || table.columns == 0)
        {
            return;
        }
        LookupArgs a = {RowPlaces(table), RowPlaces(out), tokens.base, tokens.wide, tokens.count, table.rows, table.columns, scale, DivBy(1)};
        if (table.elem == kRowF16)
        {
            LaunchLookup<Half, Half>(a, stream);
        }
        else if (table.elem == kRowBf16)
        {
            LaunchLookup<Bf16, Bf16>(a, stream);
        }
        else if (out.elem == kRowF32)
        {
            LaunchLookup<float, float>(a, stream);
        }
        else if (out.elem == kRowF16)
        {
            LaunchLookup<float, Half>(a, stream);
        }
        else
        {
            LaunchLookup<float, Bf16>(a, stream);
        }
    }

    static void submitGrad(hipStream_t stream, NVCVTensorHandle hgrad, NVCVTensorHandle htokens, NVCVTensorHandle htable,
                           NVCVTensorHandle hworkspace, float scale, int64_t padding, bool accumulate)
    {
        const RowsView grad = RequireRows(hgrad, "Output's gradient"), table = RequireRows(htable, "Table's gradient");
        const Tokens   tokens = TakeTokens(htokens);
        RequireScale(scale);
        if (grad.rows != tokens.count || grad.columns != table.columns)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Output's gradient must have a row per token (%d) with the table's elements (%d), not %d of %d",
                          tokens.count, table.columns, grad.rows, grad.columns);
        }
        if (table.elem != grad.elem && table.elem != kRowF32)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Table's gradient must have the type of the output's gradient, or F32");
        }
        if (padding < -1)
        {
            throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Padding must be a token, or -1 for none, not %ld", (long)padding);
        }
        const GradRoom at(tokens.count, table.columns);
        uint8_t       *room = RequireWorkspace(hworkspace, at.bytes);
        if (table.rows == 0 || table.columns == 0)
        {
            return;
        }
        const int64_t  rowBytes = table.columns * (int64_t)RowElemSize(table.elem);
        const bool     dense    = table.inner == table.rows && table.innerStride == rowBytes;
        const bool     few      = tokens.count > 0 && tokens.count <= kFewTokens;
        const uint32_t beside   = accumulate ? 0
                                : few        ? (table.rows * rowBytes > kFewClearBytes ? table.rows : 0)
                                             : RowsBesideSort(tokens.count, table.rows, rowBytes);
        const TokenSource src      = {tokens.base, tokens.wide, tokens.count, table.rows, padding};
        Clearing          clearing = {{RowPlaces(table), rowBytes, RowElemSize(table.elem), dense, table.rows - beside, 0, 0}, beside, 0};
        if (tokens.count > kFewTokens)
        {
            SortTokens(src, room, at, clearing, stream);
        }
        else if (beside > 0)
        {
            clearing.launches   = 1;
            const uint32_t grid = clearing.next(0, kSmallThreads / 64);
            hipLaunchKernelGGL(EmbeddingClearKernel, dim3(grid), dim3(kSmallThreads), 0, stream, clearing.args);
            CheckLaunch("EmbeddingClearKernel");
        }
        const uint32_t group = (uint32_t)(kSumWaves * PieceOf(tokens.count, table.columns));
        SumArgs a = {RowPlaces(grad), RowPlaces(table), nullptr, nullptr, nullptr, tokens.count,
                     table.rows, table.columns, accumulate, (uint32_t)Parts(tokens.count, group), group, 0, 0, 0, 0, 0,
                     accumulate ? 0 : (uint32_t)table.rows - beside, dense, scale};
        if (room != nullptr)
        {
            a.keys    = reinterpret_cast<const uint32_t *>(room + at.keys);
            a.places  = reinterpret_cast<const uint32_t *>(room + at.places);
            a.partial = reinterpret_cast<float *>(room + at.partial);
        }
        if (grad.elem == kRowF32)
        {
            LaunchGrad<float, float>(src, a, stream);
        }
        else if (grad.elem == kRowF16)
        {
            table.elem == kRowF32 ? LaunchGrad<Half, float>(src, a, stream) : LaunchGrad<Half, Half>(src, a, stream);
        }
        else
        {
            table.elem == kRowF32 ? LaunchGrad<Bf16, float>(src, a, stream) : LaunchGrad<Bf16, Bf16>(src, a, stream);
        }
    }
};

} // namespace
} // namespace cvamd

using namespace cvamd;

extern "C"
{
CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingCreate(NVCVOperatorHandle *handle)
{
    return CreateOperator<Embedding>(handle);
}

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle table,
                                                NVCVTensorHandle tokens, NVCVTensorHandle out, float scale)
{
    return Protect([&] { ToOperator<Embedding>(handle).submit(stream, table, tokens, out, scale); });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingGradWorkspace(int64_t tokens, int64_t vocabulary, int64_t columns, int64_t *bytes)
{
    return Protect(
        [&]
        {
            if (bytes == nullptr)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Pointer to output must not be NULL");
            }
            if (tokens < 0 || tokens > INT32_MAX || vocabulary < 0 || vocabulary > INT32_MAX || columns < 0 || columns > INT32_MAX)
            {
                throw OpError(NVCV_ERROR_INVALID_ARGUMENT, "Tokens, rows of the table and row elements must be in [0, %d], not %ld, %ld and %ld",
                              INT32_MAX, (long)tokens, (long)vocabulary, (long)columns);
            }
            *bytes = GradRoom(tokens, columns).bytes; // (whatever the vocabulary)
        });
}

CVCUDA_PUBLIC NVCVStatus cvcudaxEmbeddingGradSubmit(NVCVOperatorHandle handle, hipStream_t stream, NVCVTensorHandle gradOut,
                                                    NVCVTensorHandle tokens, NVCVTensorHandle gradTable,
                                                    NVCVTensorHandle workspace, float scale, int64_t padding,
                                                    int8_t accumulate)
{
    return Protect(
        [&]
        {
            (void)ToOperator<Embedding>(handle);
            Embedding::submitGrad(stream, gradOut, tokens, gradTable, workspace, scale, padding, accumulate != 0);
        });
}
}
