// The paged attention's largest calls (whispereacp_amd/csrc/paged_plan.h) on the CPU:
// the pairs of new rows and query heads that its kernels count in 32 bits. Prints
// "ok <case>" per passing case; exits 1 on the first failure.
#include "../../whispereacp_amd/csrc/paged_plan.h"

#include <climits>
#include <cstdlib>
#include <cstring>

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

int main()
{
    char why[256] = {0};
    wsp_paged_cache cache {};
    cache.storage = WSP_F16;
    cache.pages = 4;
    cache.page_rows = 16;
    cache.heads = 1;
    cache.head_width = 16;
    auto attended = [&](int rows, int max_count, int heads) {
        wsp_paged_rows r {};
        r.sequences = 1;
        r.rows = rows;
        r.max_count = max_count;
        r.max_length = 64;
        r.table_width = 4;
        why[0] = 0;
        const int status = refusal_of_attention(&cache, &r, heads, why, sizeof(why));
        expect((status == WSP_OK) == (std::strlen(why) == 0), "a refusal says why");
        if (status == WSP_OK) // its plan's tiles, and the rows behind the last, are counted without a wrap
        {
            const Plan p = plan_attention(cache, r, heads / cache.heads, kPartialBytes / sizeof(float));
            const long long pairs = (long long) (max_count < rows ? max_count : rows) * heads / cache.heads;
            expect((long long) p.tiles * p.tile_rows >= pairs && (long long) p.tiles * p.tile_rows + kChunkRows <= INT_MAX,
                   "tiles fit 32 bits");
        }
        return status;
    };
    expect(attended(1 << 27, 1 << 27, 16) == WSP_ERR_CAPACITY, "2^31 pairs of a sequence are refused");
    expect(attended(INT_MAX, INT_MAX, 1) == WSP_ERR_CAPACITY, "as many rows are");
    expect(attended(1 << 27, 1 << 26, 16) == WSP_OK, "half of them pass");
    expect(attended(1 << 27, 1, 16) == WSP_OK, "as do single tokens of many sequences");
    cache.heads = 16;
    expect(attended(1 << 27, 1 << 27, 16) == WSP_OK, "or heads that share nothing");
    expect(attended(1, 1, 24) == WSP_ERR_SHAPE && attended(1, 1, 0) == WSP_ERR_SHAPE, "query heads are whole groups");
    return 0;
}
