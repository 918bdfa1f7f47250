// The paged cache's arithmetic that needs no device: what the entry points
// refuse, where a position lies, and which packed row is whose. The kernels take
// every address from here (constexpr functions are both host and device code),
// so a bad table, length or start never leads outside the pool.
#pragma once

#include "../../include/wsp_hip.h"

#include <algorithm>
#include <cstdarg>
#include <cstddef>
#include <cstdint>
#include <cstdio>

namespace wsp::paged
{
constexpr int kMaxHeadWidth = 128;
constexpr int kMinPageRows = 16, kMaxPageRows = 1024;

// The page of `position` in a sequence's row of the table, or -1: a position
// before the sequence or past the table, or a page that is not in the pool.
constexpr int page_of(const int* table, int table_width, int page_shift, int pages, int position)
{
    const int block = position >> page_shift;
    if (position < 0 || block >= table_width)
        return -1;
    const int page = table[block];
    return page >= 0 && page < pages ? page : -1;
}

// The pool's row of a head at a place in a page (rows of head_width values).
constexpr size_t pool_row(int page, int head, int place, int heads, int page_shift)
{
    return ((((size_t) page * heads + head) << page_shift) + place);
}

// The sequence of packed row `row`, or -1. The guess (row r is sequence r's, as
// in a step of one token each) saves such a step the search.
constexpr int sequence_of(const int* starts, int sequences, int row)
{
    if (row < sequences && starts[row] == row && starts[row + 1] == row + 1)
        return row;
    int first = 0, last = sequences; // starts[i] <= row for i < first, > row for i >= last
    while (first < last)
    {
        const int middle = first + (last - first) / 2;
        if (starts[middle] <= row)
            first = middle + 1;
        else
            last = middle;
    }
    const int sequence = first - 1;
    return sequence >= 0 && row < starts[sequence + 1] ? sequence : -1;
}

// Packed row `row`'s position (before 0: none), given its sequence.
constexpr long long position_of(const int* starts, const int* lengths, int sequence, int row)
{
    return (long long) lengths[sequence] - ((long long) starts[sequence + 1] - row);
}

constexpr int shift_of(int page_rows)
{
    int shift = 0;
    while ((1 << shift) < page_rows)
        ++shift;
    return shift;
}

inline int say(char* why, size_t size, int code, const char* format, ...)
{
    va_list args;
    va_start(args, format);
    std::vsnprintf(why, size, format, args);
    va_end(args);
    return code;
}

// Positions past this are not attended (a length past it counts as past max_length).
constexpr int kMostLength = 1 << 30;

// Keys that an attention call can meet: max_length, and of a table that ends before it
// one key past the table, which makes NaN of the rows that see it.
inline int key_bound(const wsp_paged_rows& rows, int page_rows)
{
    const long long held = (long long) rows.table_width * page_rows + 1;
    long long bound = rows.max_length < kMostLength ? rows.max_length : kMostLength;
    return (int) (bound < held ? bound : held);
}

// How an attention call is cut: blocks of tile_rows pairs (new row, query head
// of a cached head's group), `splits` blocks of `span` keys along the keys, and
// launches of at most `slice` sequences. Splits leave partial rows of
// head_width + 2 floats, row_slots to a block, in a scratch of scratch_floats.
struct Plan
{
    int tile_rows, tiles;
    int splits, span, row_slots;
    bool fused; // the splits are joined by the last block of their tile
    int slice;
};

constexpr int kChunkRows = 128;   // of the kernel for many rows
constexpr int kChunkBlocks = 384; // from so many of its blocks on it is taken
// Least keys of a cut of its (4096 pairs over 30000 E4M3 keys of 8 heads of 64: 1317 us
// uncut, 660 in three, 1016 in blocks of 32 rows; of 128, 1617, 1178 and 1652).
constexpr int kChunkSpan = 2048;
// Blocks that run at once, three a CU: of 16 and 32 rows, and of 128 rows of 64-wide fp16 and
// E4M3 heads. (The others of 128 rows run two a CU or one, so their cuts may take more than
// a round: 4096 pairs over 30000 bf16 keys of 8 heads of 128, 1725 us in three, 1665 uncut;
// in fp16, 1074 and 1342.)
constexpr int kRoundBlocks = 768;
constexpr int kLeastSpan = 256;   // two turns of a block's waves
// Longer spans are cut even where the blocks already fill the chip: lengths differ. (64
// sequences of up to 8192, eight cached heads of 128 in E4M3: 189 us in spans of 1024,
// 162 of 2048, 150 of 4096, where a block's start and its hand-over weigh least.)
constexpr int kMostSpan = 4096;
constexpr int kSplitUnits = 4096; // counters, one for each row tile of a cached head
constexpr int kJoinRows = 4096;   // partial rows that one block joins
// Splits that the last block of a tile of few rows joins itself; more, and those of many
// rows, are joined by a launch of their own (one token over 131072 positions, 96 splits:
// 110 us so, 124 by the last block; four tokens over 1500 of 16 streams, three splits: 25
// and 23.5).
constexpr int kFusedSplits = 16;
constexpr int kMostSequences = 65535; // a launch's z extent
constexpr size_t kPartialBytes = (size_t) 64 << 20; // of wsp_hip_ctx_create's contexts, for partial rows

inline Plan plan_attention(const wsp_paged_cache& cache, const wsp_paged_rows& rows, int group, size_t scratch_floats)
{
    Plan plan {};
    const int storage = cache.storage, heads = cache.heads, head_width = cache.head_width;
    const long long pairs = (long long) (rows.max_count < rows.rows ? rows.max_count : rows.rows) * group;
    const int keys = key_bound(rows, cache.page_rows);
    plan.slice = rows.sequences < kMostSequences ? rows.sequences : kMostSequences;
    auto per_unit = [&](int slots) { return (size_t) slots * (head_width + 2); };
    auto held = [&](long long units, int slots) { // splits whose partial rows the scratch holds
        return (long long) (scratch_floats / per_unit(slots) / units);
    };
    // Blocks of 128 rows where they, cut along long keys, make a round and a half of the
    // chip: each takes longer than smaller ones, and more of it lies idle behind a
    // sequence's last row. 512 rows over 2048 keys of 12 heads of 64, fp16, 16 sequences:
    // 128 us and 176 in blocks of 32, 8 sequences 97 and 95, 4 sequences 87 and 55; heads
    // of 128, 261 and 412 in blocks of 16, 139 and 213, 107 and 114. 14 sequences of up to
    // 333 rows over up to 13554 bf16 keys of 14 heads of 64, 656 and 420. (The packed rows
    // tell how many blocks there are at most, but for half a block a sequence.)
    const long long chunks = (pairs + kChunkRows - 1) / kChunkRows * heads * plan.slice;
    const long long filled =
        ((long long) rows.rows * group / kChunkRows + rows.sequences / 2 + 1) * heads; // about
    long long chunk_splits = kRoundBlocks / chunks;
    // (Lengths differ: 200 rows of each of four sequences of up to 54000 fp16 keys of 13 heads of
    // 64, 419 us in 7 cuts and 325 in 13; all four of 54000, 478 and 503.)
    if (chunks < kRoundBlocks / 3 && chunk_splits < keys / kMostSpan)
        chunk_splits = keys / kMostSpan;
    if (chunk_splits > kFusedSplits)
        chunk_splits = kFusedSplits;
    if (chunk_splits > keys / kChunkSpan)
        chunk_splits = keys / kChunkSpan;
    if (chunk_splits > held(chunks, kChunkRows))
        chunk_splits = held(chunks, kChunkRows);
    if (chunk_splits < 1)
        chunk_splits = 1;
    if (storage != WSP_F32 && pairs > kChunkRows / 2 && std::min(chunks, filled) * chunk_splits >= kChunkBlocks)
        plan.tile_rows = kChunkRows;
    else
        plan.tile_rows = pairs <= 16 || head_width > 64 ? 16 : 32;
    plan.tiles = (int) ((pairs + plan.tile_rows - 1) / plan.tile_rows);
    plan.row_slots = (int) (pairs < plan.tile_rows ? pairs : plan.tile_rows);
    const long long units = (long long) plan.tiles * heads * plan.slice;
    // As many splits as still run at once, or as keep the spans short.
    long long splits = (keys + kLeastSpan - 1) / kLeastSpan;
    if (splits > kRoundBlocks / units)
        splits = kRoundBlocks / units;
    if (splits < (keys + kMostSpan - 1) / kMostSpan)
        splits = (keys + kMostSpan - 1) / kMostSpan;
    if (splits > kJoinRows / plan.row_slots)
        splits = kJoinRows / plan.row_slots;
    if (splits > held(units, plan.row_slots))
        splits = held(units, plan.row_slots);
    if (splits < 2 || units > kSplitUnits)
        splits = 1;
    if (plan.tile_rows == kChunkRows)
        splits = chunk_splits;
    plan.span = (int) (((keys + splits - 1) / splits + 63) / 64 * 64);
    plan.span = plan.span < 64 ? 64 : plan.span;
    plan.splits = splits == 1 ? 1 : (keys + plan.span - 1) / plan.span;
    plan.fused = plan.splits <= kFusedSplits && plan.tile_rows != kChunkRows;
    return plan;
}

// Why a call over this cache and these rows is refused: WSP_OK, or a status
// with the reason in `why`.
inline int refusal(const wsp_paged_cache* cache, const wsp_paged_rows* rows, char* why, size_t size)
{
    if (cache == nullptr || rows == nullptr)
        return say(why, size, WSP_ERR_ARGUMENT, "paged: null cache or rows");
    if (cache->storage != WSP_F32 && cache->storage != WSP_F16 && cache->storage != WSP_BF16
        && cache->storage != WSP_E4M3)
        return say(why, size, WSP_ERR_ARGUMENT, "paged: unknown storage %d", cache->storage);
    if (cache->pages <= 0 || cache->heads <= 0)
        return say(why, size, WSP_ERR_ARGUMENT, "paged: %d pages of %d heads", cache->pages, cache->heads);
    if (cache->head_width <= 0 || cache->head_width % 16 != 0 || cache->head_width > kMaxHeadWidth)
        return say(why, size, WSP_ERR_LOGIC, "paged: heads up to %d wide in multiples of 16, and not %d", kMaxHeadWidth,
                   cache->head_width);
    if (cache->page_rows < kMinPageRows || cache->page_rows > kMaxPageRows
        || (cache->page_rows & (cache->page_rows - 1)) != 0)
        return say(why, size, WSP_ERR_LOGIC, "paged: pages hold a power of two of %d to %d positions, and not %d", kMinPageRows,
                   kMaxPageRows, cache->page_rows);
    if (cache->keys == nullptr || cache->values == nullptr)
        return say(why, size, WSP_ERR_ARGUMENT, "paged: null pool");
    if (reinterpret_cast<uintptr_t>(cache->keys) % 16 != 0 || reinterpret_cast<uintptr_t>(cache->values) % 16 != 0)
        return say(why, size, WSP_ERR_ARGUMENT, "paged: pools lie at 16 bytes");
    if (cache->storage == WSP_E4M3 && (cache->key_exponents == nullptr || cache->value_exponents == nullptr))
        return say(why, size, WSP_ERR_ARGUMENT, "paged: E4M3 without exponents");
    if (rows->sequences < 0 || rows->rows < 0 || rows->max_count < 0 || rows->max_length < 0 || rows->table_width < 0)
        return say(why, size, WSP_ERR_ARGUMENT, "paged: %d sequences, %d rows, at most %d of %d, %d pages a sequence",
                   rows->sequences, rows->rows, rows->max_count, rows->max_length, rows->table_width);
    if (rows->sequences > 0 && (rows->starts == nullptr || rows->lengths == nullptr))
        return say(why, size, WSP_ERR_ARGUMENT, "paged: null starts or lengths");
    if (rows->sequences > 0 && rows->table_width > 0 && rows->pages == nullptr)
        return say(why, size, WSP_ERR_ARGUMENT, "paged: null table");
    return WSP_OK;
}

// The same for packed tensors of `heads` heads, rows `stride` floats apart.
inline int refusal_of_tensor(const wsp_paged_cache* cache, const wsp_paged_rows* rows, const char* name,
                             const void* data, int heads, int stride, char* why, size_t size)
{
    if (data == nullptr && rows->rows > 0)
        return say(why, size, WSP_ERR_ARGUMENT, "paged: null %s", name);
    if (stride < (long long) heads * cache->head_width)
        return say(why, size, WSP_ERR_SHAPE, "paged: %s rows of %d heads of %d lie %d floats apart", name, heads,
                   cache->head_width, stride);
    return WSP_OK;
}

// The same for the query heads of an attention call. The kernels count a sequence's
// pairs (new row, query head of a cached head's group) in 32 bits, a tile past the last.
constexpr int kMostPairs = (1 << 30) + (1 << 29);

inline int refusal_of_attention(const wsp_paged_cache* cache, const wsp_paged_rows* rows, int heads, char* why,
                                size_t size)
{
    if (heads <= 0 || heads % cache->heads != 0)
        return say(why, size, WSP_ERR_SHAPE, "paged attention: %d query heads over %d cached ones", heads,
                   cache->heads);
    const int count = std::min(rows->rows, rows->max_count), group = heads / cache->heads;
    if ((long long) count * group > kMostPairs)
        return say(why, size, WSP_ERR_CAPACITY,
                   "paged attention: %d rows of a sequence times %d query heads a cached one", count, group);
    return WSP_OK;
}
} // namespace wsp::paged
