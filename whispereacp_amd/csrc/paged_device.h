// What the paged cache's kernels share: their arguments, the look-up of a page
// and the choice of a kernel by storage.
#pragma once

#include "device_common.h"
#include "paged_plan.h"

#include <type_traits>

namespace wsp::paged
{
constexpr int kE4M3 = WSP_E4M3;
constexpr int kExponentBias = 127;

// What the kernels take of a cache and its rows.
struct Cache
{
    int pages, page_shift, heads, head_width;
    void* keys;
    void* values;
    uint8_t* key_exponents;
    uint8_t* value_exponents;
};
struct Rows
{
    int sequences, rows, max_count, max_length, key_bound, table_width;
    const int* starts;
    const int* lengths;
    const int* pages;
};

__device__ __forceinline__ int page_at(const Cache& cache, const Rows& rows, int sequence, int position)
{
    return page_of(rows.pages + (size_t) sequence * rows.table_width, rows.table_width, cache.page_shift, cache.pages,
                   position);
}

inline Cache device_cache(const wsp_paged_cache& c)
{
    return {c.pages, shift_of(c.page_rows), c.heads, c.head_width, c.keys, c.values, c.key_exponents, c.value_exponents};
}

inline Rows device_rows(const wsp_paged_cache& c, const wsp_paged_rows& r)
{
    return {r.sequences,   r.rows,   r.max_count, r.max_length < kMostLength ? r.max_length : kMostLength,
            key_bound(r, c.page_rows), r.table_width, r.starts,    r.lengths, r.pages};
}

// f called with the storage as a compile-time constant.
template <class F>
void by_storage(int storage, F&& f)
{
    switch (storage)
    {
        case WSP_F32: return f(std::integral_constant<int, kF32> {});
        case WSP_F16: return f(std::integral_constant<int, kF16> {});
        case WSP_BF16: return f(std::integral_constant<int, kBF16> {});
        default: return f(std::integral_constant<int, kE4M3> {});
    }
}
} // namespace wsp::paged
