// How an attention call over a paged cache is cut (whispereacp_amd/csrc/paged_plan.h):
// storage, cached heads, group, head width, page rows, table width, sequences, rows,
// max_count, max_length -> tile rows, splits, span, whether the splits are joined by
// the last block of their tile.
#include "../../whispereacp_amd/csrc/paged_plan.h"

#include <cstdlib>

int main(int argc, char** argv)
{
    if (argc != 11)
        return 2;
    int given[10];
    for (int i = 0; i < 10; ++i)
        given[i] = std::atoi(argv[i + 1]);
    wsp_paged_cache cache {};
    cache.storage = given[0];
    cache.heads = given[1];
    cache.head_width = given[3];
    cache.page_rows = given[4];
    wsp_paged_rows rows {};
    rows.table_width = given[5];
    rows.sequences = given[6];
    rows.rows = given[7];
    rows.max_count = given[8];
    rows.max_length = given[9];
    const wsp::paged::Plan plan =
        wsp::paged::plan_attention(cache, rows, given[2], wsp::paged::kPartialBytes / sizeof(float));
    std::printf("%d %d %d %d\n", plan.tile_rows, plan.splits, plan.span, (int) plan.fused);
    return 0;
}
