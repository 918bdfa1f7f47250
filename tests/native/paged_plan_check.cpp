// The paged cache's refusals and its look-ups (whispereacp_amd/csrc/paged_plan.h)
// on the CPU: bad tables, lengths and starts never lead outside the pool or the
// arrays. Prints "ok <case>" per passing case; exits 1 on the first failure.
#include "../../whispereacp_amd/csrc/paged_plan.h"

#include <algorithm>
#include <climits>
#include <cstdlib>
#include <cstring>
#include <vector>

using namespace wsp::paged;

static void expect(bool condition, const char* what)
{
    if (!condition)
    {
        std::printf("FAIL %s\n", what);
        std::exit(1);
    }
    std::printf("ok %s\n", what);
}

static wsp_paged_cache good_cache()
{
    wsp_paged_cache cache {};
    cache.storage = WSP_E4M3;
    cache.pages = 4;
    cache.page_rows = 16;
    cache.heads = 2;
    cache.head_width = 64;
    cache.keys = reinterpret_cast<void*>(256);
    cache.values = reinterpret_cast<void*>(512);
    cache.key_exponents = reinterpret_cast<uint8_t*>(3);
    cache.value_exponents = reinterpret_cast<uint8_t*>(5);
    return cache;
}

static wsp_paged_rows good_rows()
{
    wsp_paged_rows rows {};
    rows.sequences = 2;
    rows.rows = 3;
    rows.max_count = 2;
    rows.max_length = 20;
    rows.table_width = 2;
    rows.starts = rows.lengths = rows.pages = reinterpret_cast<const int*>(64);
    return rows;
}

template <class Change>
static int refused_cache(Change change)
{
    wsp_paged_cache cache = good_cache();
    const wsp_paged_rows rows = good_rows();
    change(cache);
    char why[256] = {0};
    const int status = refusal(&cache, &rows, why, sizeof(why));
    return status != WSP_OK && std::strlen(why) == 0 ? 1 : status;
}

template <class Change>
static int refused_rows(Change change)
{
    const wsp_paged_cache cache = good_cache();
    wsp_paged_rows rows = good_rows();
    change(rows);
    char why[256] = {0};
    const int status = refusal(&cache, &rows, why, sizeof(why));
    return status != WSP_OK && std::strlen(why) == 0 ? 1 : status;
}

int main()
{
    char why[256];
    const wsp_paged_cache cache = good_cache();
    const wsp_paged_rows rows = good_rows();
    expect(refusal(&cache, &rows, why, sizeof(why)) == WSP_OK, "a good cache and rows pass");
    expect(refusal(nullptr, &rows, why, sizeof(why)) == WSP_ERR_ARGUMENT, "a null cache is refused");
    expect(refusal(&cache, nullptr, why, sizeof(why)) == WSP_ERR_ARGUMENT, "null rows are refused");
    expect(refused_cache([](auto& c) { c.storage = 4; }) == WSP_ERR_ARGUMENT, "an unknown storage is refused");
    expect(refused_cache([](auto& c) { c.pages = 0; }) == WSP_ERR_ARGUMENT, "an empty pool is refused");
    expect(refused_cache([](auto& c) { c.heads = 0; }) == WSP_ERR_ARGUMENT, "no heads are refused");
    expect(refused_cache([](auto& c) { c.head_width = 72; }) == WSP_ERR_LOGIC, "a head width of 72 is refused");
    expect(refused_cache([](auto& c) { c.head_width = 144; }) == WSP_ERR_LOGIC, "a head width of 144 is refused");
    expect(refused_cache([](auto& c) { c.page_rows = 8; }) == WSP_ERR_LOGIC, "pages of 8 positions are refused");
    expect(refused_cache([](auto& c) { c.page_rows = 48; }) == WSP_ERR_LOGIC, "pages of 48 positions are refused");
    expect(refused_cache([](auto& c) { c.page_rows = 2048; }) == WSP_ERR_LOGIC, "pages of 2048 positions are refused");
    expect(refused_cache([](auto& c) { c.keys = nullptr; }) == WSP_ERR_ARGUMENT, "a null pool is refused");
    expect(refused_cache([](auto& c) { c.values = reinterpret_cast<void*>(520); }) == WSP_ERR_ARGUMENT,
           "a pool at 8 bytes is refused");
    expect(refused_cache([](auto& c) { c.value_exponents = nullptr; }) == WSP_ERR_ARGUMENT,
           "E4M3 without exponents is refused");
    expect(refused_cache([](auto& c) {
               c.storage = WSP_BF16;
               c.key_exponents = c.value_exponents = nullptr;
           }) == WSP_OK,
           "other storages need no exponents");
    expect(refused_rows([](auto& r) { r.rows = -1; }) == WSP_ERR_ARGUMENT, "negative rows are refused");
    expect(refused_rows([](auto& r) { r.sequences = -1; }) == WSP_ERR_ARGUMENT, "negative sequences are refused");
    expect(refused_rows([](auto& r) { r.max_length = -1; }) == WSP_ERR_ARGUMENT, "a negative length is refused");
    expect(refused_rows([](auto& r) { r.starts = nullptr; }) == WSP_ERR_ARGUMENT, "null starts are refused");
    expect(refused_rows([](auto& r) { r.pages = nullptr; }) == WSP_ERR_ARGUMENT, "a null table is refused");
    expect(refused_rows([](auto& r) {
               r.sequences = 0;
               r.starts = r.lengths = r.pages = nullptr;
           }) == WSP_OK,
           "no sequences need no arrays");
    const float x = 0.f;
    expect(refusal_of_tensor(&cache, &rows, "key", &x, 2, 128, why, sizeof(why)) == WSP_OK, "a dense tensor passes");
    expect(refusal_of_tensor(&cache, &rows, "key", &x, 2, 127, why, sizeof(why)) == WSP_ERR_SHAPE,
           "overlapping rows are refused");
    expect(refusal_of_tensor(&cache, &rows, "key", nullptr, 2, 128, why, sizeof(why)) == WSP_ERR_ARGUMENT,
           "a null tensor is refused");

    // Pages: what is outside the pool or the table is -1.
    const std::vector<int> table = {3, -1, 4, INT_MAX, INT_MIN, 0};
    const int width = (int) table.size();
    const int expected[] = {3, -1, -1, -1, -1, 0};
    bool right = true;
    for (int p = 0; p < 16 * width; ++p)
        right = right && page_of(table.data(), width, 4, 4, p) == expected[p / 16];
    expect(right, "pages outside the pool are none");
    for (int p : {-1, INT_MIN, 16 * width, INT_MAX})
        right = right && page_of(table.data(), width, 4, 4, p) == -1;
    expect(right && page_of(nullptr, 0, 4, 4, 0) == -1, "positions outside the table are none");
    expect(pool_row(1 << 20, 31, 1023, 32, 10) == (((size_t) (1 << 20) * 32 + 31) << 10) + 1023,
           "a pool row passes 32 bits");

    // Whose row: against a walk over the starts, empty sequences among them.
    const std::vector<int> starts = {0, 0, 3, 3, 4, 9, 9};
    const int sequences = (int) starts.size() - 1;
    right = true;
    for (int r = 0; r < 12; ++r)
    {
        int owner = -1;
        for (int s = 0; s < sequences; ++s)
            if (starts[s] <= r && r < starts[s + 1])
                owner = s;
        right = right && sequence_of(starts.data(), sequences, r) == owner;
    }
    expect(right, "rows find their sequence");
    const std::vector<int> one = {0, 1, 2, 3};
    for (int r = 0; r < 5; ++r)
        right = right && sequence_of(one.data(), 3, r) == (r < 3 ? r : -1);
    expect(right && sequence_of(starts.data(), 0, 0) == -1, "a step's rows find their sequence");
    const std::vector<int> late = {2, 5};
    expect(sequence_of(late.data(), 1, 1) == -1 && sequence_of(late.data(), 1, 2) == 0
               && sequence_of(late.data(), 1, 5) == -1,
           "rows before the first start are nobody's");
    // Starts that descend, or lie outside the rows, stay inside the arrays (the
    // sanitizer watches) and give a sequence or none.
    const std::vector<int> odd = {7, -3, INT_MAX, 2, INT_MIN};
    for (int r = 0; r < 20; ++r)
    {
        const int s = sequence_of(odd.data(), 4, r);
        right = right && s >= -1 && s < 4;
        if (s >= 0)
            (void) position_of(odd.data(), odd.data(), s, r);
    }
    expect(right, "odd starts stay inside the arrays");
    const std::vector<int> lengths = {5, 2};
    const std::vector<int> packed = {0, 3, 6};
    expect(position_of(packed.data(), lengths.data(), 0, 0) == 2 && position_of(packed.data(), lengths.data(), 0, 2) == 4
               && position_of(packed.data(), lengths.data(), 1, 3) == -1,
           "new rows are the last positions");
    expect(shift_of(16) == 4 && shift_of(1024) == 10, "page shifts");

    // Plans: what the launches index fits the scratch, the counters, the join's factors
    // and a launch's extents, and the splits cover every key a row can see.
    const size_t scratch = kPartialBytes / sizeof(float);
    right = true;
    int split = 0, chunked = 0, cut_chunks = 0;
    for (int storage = WSP_F32; storage <= WSP_E4M3; ++storage)
        for (int width : {16, 64, 80, 128})
            for (int heads : {1, 6, 20, 200, 5000})
                for (int group : {1, 4, 17})
                    for (int count : {1, 5, 40, 513, 100000, INT_MAX})
                        for (int sequences : {1, 64, 70000})
                            for (int length : {0, 1, 255, 257, 448, 9000, 131072, INT_MAX})
                            {
                                wsp_paged_cache c = good_cache();
                                c.storage = storage;
                                c.head_width = width;
                                c.heads = heads;
                                wsp_paged_rows r = good_rows();
                                r.sequences = sequences;
                                r.rows = 200000;
                                r.max_count = count;
                                r.max_length = length;
                                r.table_width = 1 << 20;
                                const Plan p = plan_attention(c, r, group, scratch);
                                const long long pairs = (long long) std::min(count, r.rows) * group;
                                const long long units = (long long) p.tiles * heads * p.slice;
                                right = right && (long long) p.tiles * p.tile_rows >= pairs && p.slice >= 1
                                        && p.slice <= kMostSequences && p.splits >= 1 && p.span >= 32
                                        && (p.splits > 1 || p.span >= key_bound(r, c.page_rows));
                                if (p.splits > 1)
                                {
                                    ++split;
                                    right = right
                                            && (unsigned long long) units * p.splits * p.row_slots * (width + 2) <= scratch
                                            && (!p.fused || (units <= kSplitUnits && p.splits * p.row_slots <= kJoinRows))
                                            && p.row_slots >= std::min<long long>(pairs, p.tile_rows)
                                            && p.span % 64 == 0
                                            && (long long) p.span * p.splits >= key_bound(r, c.page_rows);
                                    cut_chunks += p.tile_rows == kChunkRows;
                                }
                                chunked += p.tile_rows == kChunkRows;
                                right = right && (storage != WSP_F32 || p.tile_rows != kChunkRows);
                            }
    expect(right && split > 100 && chunked > 100 && cut_chunks > 20, "plans fit what they index");
    wsp_paged_rows table_rows = good_rows(); // 2 pages of 16
    table_rows.max_length = 1000;
    expect(key_bound(table_rows, 16) == 33, "a row that sees past the table sees one key there");
    table_rows.max_length = 20;
    expect(key_bound(table_rows, 16) == 20, "the longest length bounds the keys");
    return 0;
}
