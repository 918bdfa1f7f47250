// What the two attention kernels of a paged cache share: the rows of a block, the
// storages as operands of the matrix cores, and values in 16-bit parts.
#pragma once

#include "paged_device.h"

namespace wsp::paged
{
// What a call asks, beside the cache and the rows.
struct Query
{
    const float* q;
    int q_stride;
    int heads, group; // group: query heads a cached head serves
    int causal;
    float scale; // times log2(e): the softmax runs in powers of two
    float* out;
    int out_stride;
};

// How a call's keys are split: `splits` blocks of `span` keys each take a row
// tile's keys, their partial rows lie at [tile unit][split][row slot], and a unit's
// counter tells its last block (zero between launches; null: another launch joins).
struct Split
{
    int splits, span, row_slots;
    float* partials;
    unsigned int* counters;
};

// The rows one block computes: for one sequence and one cached head, `tile`
// consecutive (new row, query head of the group) pairs, row-major.
struct RowTile
{
    int first_row;   // the sequence's first packed row
    int pairs;       // rows to compute times group
    int past;        // position of the first new row (before 0: none)
    int length;
    int bound;       // no row looks further (Rows::key_bound)
    int first, last; // this tile's pairs
    int least, most; // keys that its first and its last row see
    bool poisoned;   // the length passes max_length
};

__device__ __forceinline__ int keys_seen(const Query& query, const RowTile& t, int pair)
{
    const long long position = (long long) t.past + pair / query.group;
    return position < 0 ? 0 : min(query.causal ? (int) position + 1 : t.length, t.bound);
}

// False where the tile has no row.
__device__ __forceinline__ bool find_tile(const Rows& rows, const Query& query, int sequence, int tile, int tile_rows,
                                          RowTile& t)
{
    // (All three in flight at once.)
    t.first_row = rows.starts[sequence];
    const int end = rows.starts[sequence + 1];
    t.length = rows.lengths[sequence];
    t.bound = rows.key_bound;
    if (t.first_row < 0 || end <= t.first_row)
        return false;
    const int count = end - t.first_row;
    t.past = max(t.length, 0) - count;
    t.pairs = min(min(count, rows.max_count), rows.rows - t.first_row) * query.group;
    t.first = tile * tile_rows;
    t.last = min(t.first + tile_rows, t.pairs) - 1;
    if (t.last < t.first)
        return false;
    t.poisoned = t.length > rows.max_length;
    t.least = keys_seen(query, t, t.first);
    t.most = keys_seen(query, t, t.last);
    return true;
}

// Blocks whose keys some row of the tile sees.
__device__ __forceinline__ int splits_used(const RowTile& t, int span)
{
    return t.poisoned ? 1 : max(1, (t.most + span - 1) / span);
}

__device__ __forceinline__ float* out_of(const RowTile& t, const Query& query, int head, int pair, int width, int c)
{
    return query.out + (size_t) (t.first_row + pair / query.group) * query.out_stride
           + (size_t) (head * query.group + pair % query.group) * width + c;
}

__device__ __forceinline__ float* partial_row(const Split& split, int unit, int which, int slot, int width)
{
    return split.partials + (((size_t) unit * split.splits + which) * split.row_slots + slot) * (width + 2);
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32u __attribute__((aligned(1)));

// Two E4M3 bytes (the low or high half of `packed`) times a power of two as two fp16.
template <bool HIGH>
__device__ __forceinline__ uint32_t e4m3_to_halves(uint32_t packed, float power)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int) packed, power, HIGH));
}

// What the matrix cores multiply a storage as, and its bytes.
template <int ST>
constexpr int operand_of = ST == kE4M3 ? (int) kF16 : ST;
template <int ST>
constexpr int bytes_of = ST == kF32 ? 4 : ST == kE4M3 ? 1 : 2;

// Two fp32 values as 16-bit parts packed in dwords: their sum is within 2^-22 of
// each (two fp16 parts) or exact (three bf16 parts).
template <int OT>
__device__ __forceinline__ void cut_pair(float a, float b, uint32_t (&parts)[3])
{
    if constexpr (OT == kF16)
    {
        typedef _Float16 half2v __attribute__((ext_vector_type(2)));
        uint32_t packed = __builtin_bit_cast(uint32_t, half2v {(_Float16) a, (_Float16) b});
        // (Opaque, so that each difference is one multiply-add that reads its half of the
        // pair, not a rounding anew, a widening and a subtraction.)
        float minus = -1.f;
        asm("" : "+v"(packed), "+s"(minus));
        const half2v high = __builtin_bit_cast(half2v, packed);
        const half2v low = {(_Float16) __builtin_fmaf((float) high[0], minus, a),
                            (_Float16) __builtin_fmaf((float) high[1], minus, b)};
        parts[0] = packed;
        parts[1] = __builtin_bit_cast(uint32_t, low);
    }
    else
    {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int p = 0; p < 3; ++p)
        {
            const bf16x2 high = {(__bf16) a, (__bf16) b};
            parts[p] = __builtin_bit_cast(uint32_t, high);
            a -= (float) high[0];
            b -= (float) high[1];
        }
    }
}

// The bits of a dword's 16-bit halves that are finite, of type OT.
template <int OT>
__device__ __forceinline__ uint32_t finite_halves(uint32_t pair)
{
    constexpr uint32_t kTop = OT == kF16 ? 0x7C00u : 0x7F80u;
    uint32_t kept = 0;
    if ((pair & kTop) != kTop)
        kept |= pair & 0xFFFFu;
    if ((pair & (kTop << 16)) != kTop << 16)
        kept |= pair & 0xFFFF0000u;
    return kept;
}

// E4M3 values as operands. A row's values times its power of two, relative to a base,
// are fp16 values exactly where the power is 2^kLeastShift to 2^kMostShift of the base's.
// A tile of keys with another power among them (a row of zeros has the least there is)
// goes as bf16, which holds four significant bits at any power, and its weights in three
// bf16 parts, exact: a quarter more products, and no power or weight is out of reach.
// What is summed leaves out the base: the first key's power within kLeastBase and
// kMostBase; from the first such tile on kLeastBase, near which ordinary rows lie; from
// one with a power past kLoudest on kLoudBase, where neither fp32's largest values pass
// its range as sums nor the least rows bf16's. (All as exponent bytes.)
constexpr int kLeastShift = -15, kMostShift = 7;
constexpr int kLeastBase = kExponentBias - 7, kMostBase = kExponentBias + 34;
constexpr int kLoudest = kExponentBias + 64, kLoudBase = kExponentBias + 35;

// Rows and sums of E4M3 values leave a kernel's loop times 2^-kSumShift: without the
// weights' bias of 2^14, and so that the values nearest fp32's end can be summed.
constexpr int kSumShift = 34;

__device__ __forceinline__ int first_base(int byte)
{
    return min(max(byte, kLeastBase), kMostBase);
}

// The base of a tile whose powers `base` does not take.
__device__ __forceinline__ int wide_base(int base, bool loud)
{
    return base == kLoudBase || loud ? kLoudBase : kLeastBase;
}

// Whether powers from `low` to `high` fit the operands.
__device__ __forceinline__ bool base_takes(int base, int low, int high)
{
    return low - base >= kLeastShift && high - base <= kMostShift;
}

// Two E4M3 bytes (the low or high half of `packed`) times 2^shift as two bf16, exact
// (magnitudes past fp32's range become infinities).
template <bool HIGH>
__device__ __forceinline__ uint32_t e4m3_to_bf16(uint32_t packed, int shift)
{
    const auto pair = __builtin_amdgcn_cvt_pk_f32_fp8((int) packed, HIGH);
    return __builtin_amdgcn_perm(__float_as_uint(ldexpf(pair[1], shift)), __float_as_uint(ldexpf(pair[0], shift)),
                                 0x07060302);
}

// A stored value widened, E4M3 without its row's power.
template <int ST>
__device__ __forceinline__ float stored_value(const void* pool, size_t index)
{
    if constexpr (ST == kE4M3)
        return __builtin_amdgcn_cvt_f32_fp8((int) static_cast<const uint8_t*>(pool)[index], 0);
    else
        return load1<ST>(pool, index);
}

template <int WORDS>
__device__ __forceinline__ void load_words(const char* at, uint32_t (&words)[WORDS])
{
    if constexpr (WORDS == 1)
        words[0] = *global(reinterpret_cast<const uint32_t*>(at));
    else if constexpr (WORDS == 2)
    {
        const u32x2 v = *global(reinterpret_cast<const u32x2*>(at));
        words[0] = v[0];
        words[1] = v[1];
    }
    else
    {
        static_assert(WORDS % 4 == 0);
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i)
        {
            const u32x4 v = global(reinterpret_cast<const u32x4*>(at))[i];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                words[4 * i + j] = v[j];
        }
    }
}

// One launch over row tiles first_tile on and sequences first_sequence on (its
// grid: splits·heads, tiles, sequences), by the kernel for many rows (paged_chunk.hip).
void launch_chunks(hipStream_t stream, dim3 grid, int storage, const Cache& cache, const Rows& rows,
                   const Query& query, const Split& split, int first_tile, int first_sequence);
} // namespace wsp::paged
