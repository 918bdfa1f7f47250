// Attention over the pages of a cache (include/wsp_hip.h,
// wsp_hip_paged_attention), on the matrix cores.
#include "paged.h"
#include "paged_attention.h"

#include <algorithm>

namespace wsp::paged
{
namespace
{
// The largest over the four 16-lane groups, in each of their lanes.
__device__ __forceinline__ float groups_max(float v)
{
    const uint32_t row = __float_as_uint(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(row, row, false, false);
    v = fmaxf(__uint_as_float((uint32_t) rows[0]), __uint_as_float((uint32_t) rows[1]));
    const uint32_t half = __float_as_uint(v);
    const auto halves = __builtin_amdgcn_permlane32_swap(half, half, false, false);
    return fmaxf(__uint_as_float((uint32_t) halves[0]), __uint_as_float((uint32_t) halves[1]));
}

__device__ __forceinline__ float groups_sum(float v)
{
    const uint32_t row = __float_as_uint(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(row, row, false, false);
    v = __uint_as_float((uint32_t) rows[0]) + __uint_as_float((uint32_t) rows[1]);
    const uint32_t half = __float_as_uint(v);
    const auto halves = __builtin_amdgcn_permlane32_swap(half, half, false, false);
    return __uint_as_float((uint32_t) halves[0]) + __uint_as_float((uint32_t) halves[1]);
}

// ---------------------------------------------------------------------------
// Few rows: attention of a tile of 16·QT pairs (new row, head of the group) over
// keys [split·span, +span) of one cached head, as query_attention_kernel does it
// for contiguous fp32 caches: a wave takes 32 keys at a time straight from
// memory into operand registers, with no barrier in the loop, and keeps an
// online (maximum, sum, row) of each pair; the waves are merged through LDS.
//
// S^T = K·Q^T leaves lane (li, g) with keys 4g + r (r < 4) of each 16 and pair li,
// which is the operand order of O^T = V^T·P^T when the product's eight keys of
// lane group g are those 4g + r of both sixteens: nothing crosses lanes. A value
// operand wants eight keys of one channel, and a row in memory holds channels of
// one key: lane li reads W / 16 channels of its group's eight keys and pairs the
// halves up itself (v_perm).
//
// q, and the weights, go in 16-bit parts (cut_pair), so a product with what the
// storage holds is as exact as fp32's; fp16 parts of q are of q·2^-e, e from the
// pair's largest magnitude, and the weights are exp2(s - max + 14), which puts
// both far from fp16's ends. An E4M3 key row's power of two multiplies its scores, a
// value row's its operands (relative to a base: paged_attention.h), so weights, maxima
// and sums are those of the scores alone. fp32 storage runs in fp32.
//
// Bound by the cache's read where rows are few and sequences long: a wave keeps the
// next 32 keys and values in flight while it works on these. One token over 131072
// bf16 positions of eight heads of 128, four query heads each: 96 us and 8 of the join,
// 5.6 TB/s; 64 such sequences of up to 8192 in E4M3 150 us, 4.0 TB/s, where the vector
// units are busy two fifths of the time (16 pairs' softmax for four real ones, and the widening)
// and two waves a SIMD do not hide the rest (a third spills; a second tile in flight,
// or loads into registers just used up, change nothing); a row of zeros in every 64
// positions, which sends their tiles through bf16, 166 us. Short sequences are bound by a
// block's chain start, page, keys, scores, values, merge: 5.6 us for one stream of 131
// positions, 11 for 32 of up to 448 in 20 heads. fp32 is bound by its matrix
// instructions: five rows over up to 1500 positions of 16 heads of 80, eight streams,
// 23.5 us.
// ---------------------------------------------------------------------------
constexpr int kKeys = 32;

template <int ST, int W>
struct Tile // one lane's part of 32 keys and values, as stored
{
    uint32_t k[2][W / 4 * bytes_of<ST> / 4];     // key 16b + li, 16-byte runs g, g + 4, ... of the row
    uint32_t v[2][4][W / 16 * bytes_of<ST> / 4]; // value 16b + 4g + r, channels W / 16·li on
    uint32_t ke[2], ve[2];                       // E4M3: the exponents of rows 16b + 4g .. + 3
    bool bad[2];                                 // the page of keys 16b .. is none
};

// The pages of keys k0 .. k0 + 15 and k0 + 16 .. k0 + 31 (-1: none).
struct Pages
{
    int page[2];
};
__device__ __forceinline__ Pages find_pages(const Cache& cache, const int* table, int table_width, int k0)
{
    return {{page_of(table, table_width, cache.page_shift, cache.pages, k0),
             page_of(table, table_width, cache.page_shift, cache.pages, k0 + 16)}};
}

// Where a lane's parts of a key and of a value row lie in a sixteen's rows, in bytes.
struct Offsets
{
    uint32_t key, value;
};

// Keys and values k0 .. k0 + 31 of a cached head. k0 is below `end`; of a sixteen
// that begins at or past it the first is read again (nothing there counts). (The pages
// are the same for the wave: what is not in `at` is scalar.)
template <int ST, int W, bool FULL>
__device__ __forceinline__ void load_tile(const Cache& cache, const Pages& pages, int head, int k0, int end, Offsets at,
                                          Tile<ST, W>& t)
{
    const int g = threadIdx.x % kWave / 16;
    const int mask = (1 << cache.page_shift) - 1, row_bytes = (FULL ? W : cache.head_width) * bytes_of<ST>;
#pragma unroll
    for (int b = 0; b < 2; ++b)
    {
        const bool second = b == 1 && k0 + 16 < end;
        const int page = second ? pages.page[1] : pages.page[0];
        t.bad[b] = page < 0;
        const size_t row = pool_row(max(page, 0), head, (second ? k0 + 16 : k0) & mask, cache.heads, cache.page_shift);
        if constexpr (ST == kE4M3) // (looked at first)
        {
            using Four = const __attribute__((address_space(1))) u32u;
            t.ke[b] = *(Four*) (cache.key_exponents + row + (uint32_t) (4 * g));
            t.ve[b] = *(Four*) (cache.value_exponents + row + (uint32_t) (4 * g));
        }
        const char* keys = static_cast<const char*>(cache.keys) + row * row_bytes;
        const char* values = static_cast<const char*>(cache.values) + row * row_bytes;
        constexpr int kRuns = W * bytes_of<ST> / 64;
#pragma unroll
        for (int i = 0; i < kRuns; ++i) // (a run lies in the row or past it)
        {
            uint32_t run[4] = {0, 0, 0, 0};
            if (FULL || 16 * (4 * i + g) < row_bytes)
                load_words(keys + 64 * i + at.key, run);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                t.k[b][4 * i + j] = run[j];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            load_words(values + r * row_bytes + at.value, t.v[b][r]);
    }
}

// Stored key words as operands: eight channels of 16 bits each.
template <int ST, int W>
__device__ __forceinline__ u32x4 key_operand(const Tile<ST, W>& t, int b, int j)
{
    if constexpr (ST == kE4M3)
    {
        const uint32_t x = t.k[b][2 * j], y = t.k[b][2 * j + 1];
        return u32x4 {e4m3_to_halves<false>(x, 1.f), e4m3_to_halves<true>(x, 1.f), e4m3_to_halves<false>(y, 1.f),
                      e4m3_to_halves<true>(y, 1.f)};
    }
    else
        return u32x4 {t.k[b][4 * j], t.k[b][4 * j + 1], t.k[b][4 * j + 2], t.k[b][4 * j + 3]};
}

// The exponent byte of the key (value) row 16b + 4g + r.
__device__ __forceinline__ int exponent_of(const uint32_t (&rows)[2], int b, int r)
{
    return (int) (rows[b] >> (8 * r) & 255u);
}

// Channels 2i and 2i + 1 of a stored value row, 16 bits each of type VT; E4M3 ones
// times their row's power relative to the base.
template <int ST, int VT, int W>
__device__ __forceinline__ uint32_t value_pair(const Tile<ST, W>& t, int b, int r, int i, int base)
{
    if constexpr (ST == kE4M3 && VT == kBF16)
    {
        const int shift = exponent_of(t.ve, b, r) - base;
        return i % 2 == 0 ? e4m3_to_bf16<false>(t.v[b][r][i / 2], shift) : e4m3_to_bf16<true>(t.v[b][r][i / 2], shift);
    }
    else if constexpr (ST == kE4M3)
    {
        const float power = __uint_as_float((uint32_t) (exponent_of(t.ve, b, r) + kExponentBias - base) << 23);
        return i % 2 == 0 ? e4m3_to_halves<false>(t.v[b][r][i / 2], power)
                          : e4m3_to_halves<true>(t.v[b][r][i / 2], power);
    }
    else
        return t.v[b][r][i];
}

constexpr int kTileWaves = 4;

// A float that blocks of one launch hand to each other.
__device__ __forceinline__ void store_shared(float* at, float value)
{
    __hip_atomic_store(at, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_shared(const float* at)
{
    return __hip_atomic_load(const_cast<float*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The weights of 32 keys (4g + r of either sixteen) for 16·QT pairs, in parts for values
// of type VT.
template <int VT_, int QT>
struct Weights
{
    static constexpr int VT = VT_;
    uint32_t part[QT][parts_of<VT>()][VT == kF32 ? 8 : 4];
};

// Pair t's from its scores; their sum joins l.
template <int VT, int QT>
__device__ __forceinline__ void weigh(float4v (&s)[2], float offset, int t, Weights<VT, QT>& weights, float& l)
{
    float own = 0.f;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
        {
            s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - offset);
            own += s[b][r];
        }
    l += own;
#pragma unroll
    for (int i = 0; i < (VT == kF32 ? 8 : 4); ++i)
        if constexpr (VT == kF32)
            weights.part[t][0][i] = __float_as_uint(s[i / 4][i % 4]);
        else
        {
            uint32_t cut[3];
            cut_pair<VT>(s[i / 2][2 * (i % 2)], s[i / 2][2 * (i % 2) + 1], cut);
#pragma unroll
            for (int p = 0; p < parts_of<VT>(); ++p)
                weights.part[t][p][i] = cut[p];
        }
}

// Adds 32 keys' value rows, as type VT, by their weights to the pairs' rows, two channels
// of each lane's at a time. A weight of zero hides a value only while it is finite: the
// careful way counts values that no pair sees (`shown`) as zero, and where some pairs see
// a key and others do not (`mixed`), non-finite values too; `odd` tells of those.
template <int ST, int VT, int W, int QT>
__device__ __forceinline__ void add_rows(const Tile<ST, W>& kv, int base, const Weights<VT, QT>& weights, bool careful,
                                         bool mixed, const uint32_t (&shown)[4], float4v (&o)[QT][W / 16], bool& odd)
{
    constexpr int CPL = W / 16;
#pragma unroll
    for (int c = 0; c < CPL; c += 2)
    {
        // Channels CPL·li + c and + c + 1 of keys 16b + 4g + r.
        if constexpr (VT == kF32)
        {
            float v[2][8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    v[e][i] = __uint_as_float(kv.v[i / 4][i % 4][c + e]);
            if (careful)
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if ((shown[i / 2] & (i % 2 == 0 ? 0xFFFFu : 0xFFFF0000u)) == 0)
                            v[e][i] = 0.f;
            if (mixed)
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                    {
                        odd = odd || !isfinite(v[e][i]);
                        v[e][i] = isfinite(v[e][i]) ? v[e][i] : 0.f;
                    }
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        o[t][c + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                            v[e][i], __uint_as_float(weights.part[t][0][i]), o[t][c + e], 0, 0, 0);
                }
        }
        else
        {
            u32x4 v[2];
#pragma unroll
            for (int d = 0; d < 4; ++d)
            {
                const uint32_t x = value_pair<ST, VT>(kv, d / 2, 2 * (d % 2), c / 2, base);
                const uint32_t y = value_pair<ST, VT>(kv, d / 2, 2 * (d % 2) + 1, c / 2, base);
                v[0][d] = __builtin_amdgcn_perm(y, x, 0x05040100); // the low halves
                v[1][d] = __builtin_amdgcn_perm(y, x, 0x07060302); // the high ones
            }
            if (careful)
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        v[e][d] &= shown[d];
            if (mixed)
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                    {
                        const uint32_t kept = finite_halves<VT>(v[e][d]);
                        odd = odd || kept != v[e][d];
                        v[e][d] = kept;
                    }
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                {
#pragma unroll
                    for (int p = parts_of<VT>() - 1; p >= 0; --p)
                        o[t][c + e] = mfma16<VT>(v[e],
                                                 u32x4 {weights.part[t][p][0], weights.part[t][p][1],
                                                        weights.part[t][p][2], weights.part[t][p][3]},
                                                 o[t][c + e]);
                }
        }
    }
}

// What a part of a row (a wave's, a split's) is multiplied by where its parts are put
// together, the largest of their maxima being `largest`; zero for a part without a key of
// finite score. Parts count by the product however small it is: NaN times zero is NaN.
__device__ __forceinline__ float part_factor(float top, float largest)
{
    return top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - largest);
}

// Waves a SIMD the registers are kept to.
template <int ST, int W, int QT>
constexpr int kTileOccupancy = QT == 1 && W == 64 && ST != kF32 ? 3 : 2;

template <int ST, int W, bool FULL, int QT>
__global__ void __launch_bounds__(kTileWaves* kWave, (kTileOccupancy<ST, W, QT>))
    tile_attention_kernel(Cache cache, Rows rows, Query query, Split split, int first_tile, int first_sequence)
{
    constexpr int OT = operand_of<ST>, kParts = parts_of<OT>(), kWaves = kTileWaves, CPL = W / 16;
    constexpr float kBias = OT == kF16 ? 14.f : 0.f; // the weights' exponent (see above)
    __shared__ float tops[kWaves][16], totals[kWaves][16];
    __shared__ float sums[kWaves][16][W];

    const int which = blockIdx.x % split.splits, head = blockIdx.x / split.splits;
    const int unit = ((int) blockIdx.z * (int) gridDim.y + (int) blockIdx.y) * cache.heads + head;
    const int sequence = first_sequence + blockIdx.z;
    const int tile = first_tile + (int) (gridDim.y - 1 - blockIdx.y); // (the tiles that see most come first)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, li = lane % 16, g = lane / 16;
    const int width = FULL ? W : cache.head_width;
    // A block's start is a chain of round trips to memory: the first keys' pages are
    // looked up beside the sequence's starts and length, and the first keys and values
    // are in flight while the queries arrive and are cut.
    const int* table = rows.pages + (size_t) sequence * rows.table_width;
    constexpr int kStride = kKeys * kWaves;
    const int begin = which * split.span;
    int k0 = begin + kKeys * wave;
    Pages pages = find_pages(cache, table, rows.table_width, k0);
    RowTile tl;
    if (!find_tile(rows, query, sequence, tile, 16 * QT, tl))
        return;
    const int used = splits_used(tl, split.span);
    if (which >= used)
        return;
    const int end = tl.poisoned ? 0 : min(begin + split.span, tl.most);
    // (Value lanes past the row read its start: they hold channels nobody stores.)
    const int row_bytes = width * bytes_of<ST>, channel = FULL || li * CPL < width ? li * CPL : 0;
    const Offsets at {(uint32_t) (li * row_bytes + 16 * g), (uint32_t) (4 * g * row_bytes + channel * bytes_of<ST>)};
    Tile<ST, W> now;
    if (k0 < end)
    {
        load_tile<ST, W, FULL>(cache, pages, head, k0, end, at, now);
        if (k0 + kStride < end)
            pages = find_pages(cache, table, rows.table_width, k0 + kStride);
    }

    // The queries: lane (li, g) holds the channels of pair li that it holds of a key.
    uint32_t qp[QT][OT == kF32 ? 1 : kParts][OT == kF32 ? W / 4 : W / 8];
    float left[QT]; // the power of two that the parts leave out,
    int lift[QT];   // E4M3: its exponent less a key byte's bias
    int seen[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t)
    {
        const int pair = tl.first + 16 * t + li;
        const bool real = pair <= tl.last;
        seen[t] = real ? min(keys_seen(query, tl, pair), end) : end;
        float x[W / 4];
        const float* from = query.q + (size_t) (tl.first_row + (real ? pair : tl.first) / query.group) * query.q_stride
                          + (size_t) (head * query.group + (real ? pair : tl.first) % query.group) * width;
#pragma unroll
        for (int i = 0; i < W / 4; i += 4)
        {
            constexpr int kRun = 16 / bytes_of<ST>;
            const int c = (4 * (i / kRun) + g) * kRun + i % kRun;
            float4v run = {0.f, 0.f, 0.f, 0.f};
            if (real && (FULL || c < width))
                run = *reinterpret_cast<const float4u*>(from + c);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[i + j] = run[j] * query.scale;
        }
        left[t] = 1.f;
        lift[t] = 0;
        if constexpr (OT == kF32)
#pragma unroll
            for (int i = 0; i < W / 4; ++i)
                qp[t][0][i] = __float_as_uint(x[i]);
        else
        {
            if constexpr (OT == kF16)
            {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < W / 4; ++i)
                    top = fmaxf(top, fabsf(x[i]));
                top = groups_max(top);
                // 2^13 <= top·2^shift < 2^14 (a pair of zeros, or not finite: as it is)
                int shift = 140 - (int) (__float_as_uint(top) >> 23);
                shift = top > 0.f && top < INFINITY ? min(shift, 126) : 0;
#pragma unroll
                for (int i = 0; i < W / 4; ++i)
                    x[i] = ldexpf(x[i], shift);
                left[t] = ldexpf(1.f, -shift);
                lift[t] = -shift - kExponentBias;
            }
#pragma unroll
            for (int i = 0; i < W / 8; ++i)
            {
                uint32_t cut[3];
                cut_pair<OT>(x[2 * i], x[2 * i + 1], cut);
#pragma unroll
                for (int p = 0; p < kParts; ++p)
                    qp[t][p][i] = cut[p];
            }
        }
    }

    float4v o[QT][CPL];
    float m[QT], l[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t)
    {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int c = 0; c < CPL; ++c)
            o[t][c] = float4v {0.f, 0.f, 0.f, 0.f};
    }

    int base = kExponentBias; // E4M3: the power that the value operands leave out
    if (ST == kE4M3 && k0 < end)
        base = first_base((int) (__builtin_amdgcn_readfirstlane(now.ve[0]) & 255u));

    auto work = [&](const Tile<ST, W>& kv, int k0) {
        // Keys that not every pair sees, or whose page is none, take the careful way.
        const bool careful = k0 + kKeys > min(tl.least, end) || kv.bad[0] || kv.bad[1];
        bool wide = false; // E4M3: the values go as bf16
        if constexpr (ST == kE4M3)
        {
            int low = 255, high = 0;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                {
                    low = min(low, exponent_of(kv.ve, b, r));
                    high = max(high, exponent_of(kv.ve, b, r));
                }
            if (careful) // (rows that nobody sees may hold anything)
            {
                low = high = base;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!kv.bad[b] && k0 + 16 * b + 4 * g + r < end)
                        {
                            low = min(low, exponent_of(kv.ve, b, r));
                            high = max(high, exponent_of(kv.ve, b, r));
                        }
            }
            if (__any(!base_takes(base, low, high))) // (rare)
            {
                const int next = wide_base(base, __any(high > kLoudest));
                const float by = ldexpf(1.f, base - next);
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int c = 0; c < CPL; ++c)
                        o[t][c] *= by;
                base = next;
                wide = __any(!base_takes(base, low, high));
            }
        }
        float offset[QT];      // from scores to the weights' powers
        float4v scores[QT][2]; // of keys 4g + r of either sixteen
        Weights<OT, QT> weights;
#pragma unroll
        for (int t = 0; t < QT; ++t)
        {
            float4v (&s)[2] = scores[t];
#pragma unroll
            for (int b = 0; b < 2; ++b)
            {
                if constexpr (OT == kF32)
                {
                    // Four partial sums a score: short chains of roundings, and products
                    // that need not wait for each other.
                    float4v part[4];
#pragma unroll
                    for (int i = 0; i < W / 4; ++i)
                        if (FULL || i < 4 || 16 * (i / 4) < width) // (past the row there are zeros)
                            part[i % 4] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                            __uint_as_float(kv.k[b][i]), __uint_as_float(qp[t][0][i]),
                            i < 4 ? float4v {0.f, 0.f, 0.f, 0.f} : part[i % 4], 0, 0, 0);
                    s[b] = (part[0] + part[1]) + (part[2] + part[3]);
                }
                else
                {
                    s[b] = float4v {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < W / 32; ++j)
                    {
                        const u32x4 key = key_operand<ST, W>(kv, b, j);
#pragma unroll
                        for (int p = kParts - 1; p >= 0; --p)
                            s[b] = mfma16<OT>(key,
                                              u32x4 {qp[t][p][4 * j], qp[t][p][4 * j + 1], qp[t][p][4 * j + 2],
                                                     qp[t][p][4 * j + 3]},
                                              s[b]);
                    }
                }
            }
            // Scores in powers of two.
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if constexpr (ST == kE4M3)
                        s[b][r] = ldexpf(s[b][r], exponent_of(kv.ke, b, r) + lift[t]);
                    else if constexpr (OT == kF16)
                        s[b][r] *= left[t];
            if (careful)
            {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                    {
                        if (kv.bad[b])
                            s[b][r] = __builtin_nanf("");
                        s[b][r] = k0 + 16 * b + 4 * g + r < seen[t] ? s[b][r] : -INFINITY;
                    }
            }
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    top = fmaxf(top, s[b][r]);
            // The maximum is rounded up to a whole power of two, so that what it rescales
            // and the bias stay exact however often it grows. (Before a key of finite
            // score, zero in its place: the weights are zero.)
            const float m_new = fmaxf(m[t], ceilf(groups_max(top)));
            const float finite = m_new == -INFINITY ? 0.f : m_new;
            offset[t] = finite - kBias;
            if (__any(m_new != m[t])) // (seldom, but for the first keys)
            {
                const float alpha = __builtin_amdgcn_exp2f(m[t] - finite);
                l[t] *= alpha;
#pragma unroll
                for (int c = 0; c < CPL; ++c)
                    o[t][c] *= alpha;
                m[t] = m_new;
            }
            if constexpr (ST != kE4M3)
                weigh(scores[t], offset[t], t, weights, l[t]);
        }

        // The rows. Non-finite values of keys that some pairs see and others do not are
        // added behind the products, to those that see them alone.
        bool odd = false;
        const bool mixed = careful && tl.least < tl.most;
        uint32_t shown[4]; // of keys 2d and 2d + 1 of a lane's eight: all bits of those that some pair sees
        if (careful)
#pragma unroll
            for (int d = 0; d < 4; ++d)
            {
                const int key = k0 + 16 * (d / 2) + 4 * g + 2 * (d % 2);
                shown[d] = kv.bad[d / 2] ? 0u : (key < end ? 0xFFFFu : 0u) | (key + 1 < end ? 0xFFFF0000u : 0u);
            }
        if (ST == kE4M3 && wide)
        {
            Weights<kBF16, QT> parts;
#pragma unroll
            for (int t = 0; t < QT; ++t)
                weigh(scores[t], offset[t], t, parts, l[t]);
            add_rows(kv, base, parts, careful, mixed, shown, o, odd);
        }
        else
        {
            if constexpr (ST == kE4M3)
#pragma unroll
                for (int t = 0; t < QT; ++t)
                    weigh(scores[t], offset[t], t, weights, l[t]);
            add_rows(kv, base, weights, careful, mixed, shown, o, odd);
        }
        if (mixed && __any(odd)) // (rare: infinities or NaN among the new rows' values)
#pragma unroll
            for (int t = 0; t < QT; ++t)
            {
                constexpr int kDwords = OT == kF32 ? 8 : 4;
                uint32_t parts[kDwords]; // (opaque: nothing of this is worked out before it is needed)
                if constexpr (ST != kE4M3)
#pragma unroll
                    for (int i = 0; i < kDwords; ++i)
                    {
                        parts[i] = weights.part[t][0][i];
                        asm("" : "+v"(parts[i]));
                    }
#pragma unroll 1
                for (int key = 0; key < kKeys; ++key)
                {
                    // Key 16b + 4g + r is held by lane group g. (Only that its weight is not zero
                    // matters: the first part of it does. E4M3 has no infinities, and NaN is NaN
                    // by any weight.)
                    float weight = 1.f;
                    if constexpr (ST != kE4M3)
                    {
                        uint32_t held = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (4 * (key / 16) + key % 4 == i)
                                held = OT == kF32   ? parts[i * kDwords / 8]
                                       : i % 2 == 0 ? parts[i * kDwords / 8] << 16
                                                    : parts[i * kDwords / 8] & 0xFFFF0000u;
                        weight = __uint_as_float(__shfl(held, li + 16 * (key / 4 % 4)));
                    }
                    const int position = k0 + key;
                    const int page = page_of(table, rows.table_width, cache.page_shift, cache.pages, position);
                    if (position >= seen[t] || page < 0)
                        continue;
                    const size_t row = pool_row(page, head, position & ((1 << cache.page_shift) - 1), cache.heads,
                                                cache.page_shift);
#pragma unroll
                    for (int c = 0; c < CPL; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                        {
                            const int channel = (4 * g + r) * CPL + c;
                            const float value =
                                channel < width ? stored_value<ST>(cache.values, row * width + channel) : 0.f;
                            if (!isfinite(value))
                                o[t][c][r] += weight * value;
                        }
                }
            }
    };

    // The next keys are in flight while these are worked on (not where two tiles
    // do not fit the registers), and the pages of those behind them looked up.
    constexpr bool kAhead = ST != kF32 || W == 64;
    if (k0 < end)
    {
        for (; k0 + kStride < end; k0 += kStride)
        {
            if constexpr (!kAhead)
                work(now, k0);
            Tile<ST, W> next;
            load_tile<ST, W, FULL>(cache, pages, head, k0 + kStride, end, at, next);
            if (k0 + 2 * kStride < end)
                pages = find_pages(cache, table, rows.table_width, k0 + 2 * kStride);
            if constexpr (kAhead)
            {
                __builtin_amdgcn_sched_barrier(0);
                work(now, k0);
            }
            now = next;
        }
        work(now, k0);
    }

    // The waves merged, 16 pairs at a time. o[t][c][r] is channel CPL·(4g + r) + c of pair li.
#pragma unroll
    for (int t = 0; t < QT; ++t)
    {
        const float total = groups_sum(l[t]) * (ST == kE4M3 ? ldexpf(1.f, -kSumShift) : 1.f);
        const float power = ST == kE4M3 ? ldexpf(1.f, base - kExponentBias - kSumShift) : 1.f;
        if (t > 0)
            __syncthreads(); // (the rows before are read)
        if (g == 0)
        {
            tops[wave][li] = m[t];
            totals[wave][li] = total;
        }
        if (tl.first + 16 * t + li <= tl.last)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < CPL; c += 4)
                    *reinterpret_cast<float4v*>(&sums[wave][li][CPL * (4 * g + r) + c]) =
                        float4v {o[t][c][r], o[t][c + 1][r], o[t][c + 2][r], o[t][c + 3][r]} * power;
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * W; i += kWaves * kWave)
        {
            const int at = i / W, c = i % W, pair = tl.first + 16 * t + at;
            if (pair > tl.last || (!FULL && c >= width))
                continue;
            float largest = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                largest = fmaxf(largest, tops[w][at]);
            float numerator = 0.f, denominator = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
            {
                const float factor = part_factor(tops[w][at], largest);
                numerator += factor * sums[w][at][c];
                denominator += factor * totals[w][at];
            }
            if (tl.poisoned)
                numerator = denominator = __builtin_nanf("");
            if (used == 1)
                *out_of(tl, query, head, pair, width, c) = denominator == 0.f ? 0.f : numerator / denominator;
            else
            {
                float* part = partial_row(split, unit, which, 16 * t + at, width);
                store_shared(part + 2 + c, numerator);
                if (c == 0)
                {
                    store_shared(part, largest);
                    store_shared(part + 1, denominator);
                }
            }
        }
    }
    if (used == 1 || split.counters == nullptr)
        return;

    // Few splits: the last block of a row tile to come here joins its splits, in their order. The
    // partial rows pass between blocks by device-scope accesses, which no cache of one
    // chiplet keeps: each wave waits until its own are done, the barrier until every
    // wave's are, and only then the count goes up. (Fences instead, which write back and
    // drop the whole cache for each block, made a step of 64 long sequences 728 us.)
    __shared__ int joins;
    wait_loads<0>();
    __syncthreads();
    if (threadIdx.x == 0)
        joins = __hip_atomic_fetch_add(&split.counters[unit], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                == (unsigned) (used - 1);
    __syncthreads();
    if (!joins)
        return;
    // First what each split's row of a pair is multiplied by (a row is a wave's at a
    // time), then the rows.
    static_assert(sizeof(sums) >= kJoinRows * sizeof(float), "a factor for each partial row");
    float* const factors = &sums[0][0][0]; // [row slot][split]
    const int slots = tl.last - tl.first + 1;
    for (int slot = wave; slot < slots; slot += kWaves)
    {
        const float* first = partial_row(split, unit, 0, slot, width);
        const size_t pitch = (size_t) split.row_slots * (width + 2);
        float largest = -INFINITY;
        for (int i = lane; i < used; i += kWave)
        {
            const float top = load_shared(first + i * pitch);
            factors[slot * used + i] = top;
            largest = fmaxf(largest, top);
        }
        largest = wave_max(largest);
        float total = 0.f;
        for (int i = lane; i < used; i += kWave)
        {
            const float factor = part_factor(factors[slot * used + i], largest);
            factors[slot * used + i] = factor;
            total += factor * load_shared(first + i * pitch + 1);
        }
        total = wave_sum(total);
        if (lane == 0)
            (&totals[0][0])[slot] = total;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < slots * width; i += kWaves * kWave)
    {
        const int slot = i / width, c = i % width;
        const float* column = partial_row(split, unit, 0, slot, width) + 2 + c;
        const size_t pitch = (size_t) split.row_slots * (width + 2);
        float numerator = 0.f;
        constexpr int kAtOnce = 8;
        for (int w0 = 0; w0 < used; w0 += kAtOnce)
        {
            float part[kAtOnce];
#pragma unroll
            for (int w = 0; w < kAtOnce; ++w)
                part[w] = load_shared(column + min(w0 + w, used - 1) * pitch);
#pragma unroll
            for (int w = 0; w < kAtOnce; ++w)
                if (w0 + w < used)
                    numerator += factors[slot * used + w0 + w] * part[w];
        }
        const float denominator = (&totals[0][0])[slot];
        *out_of(tl, query, head, tl.first + slot, width, c) = denominator == 0.f ? 0.f : numerator / denominator;
    }
    if (threadIdx.x == 0) // (zero again for the next launch)
        __hip_atomic_store(&split.counters[unit], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The partial rows of many splits joined by a launch of their own (one block of the
// last launch would read them too slowly): a block for each (pair, cached
// head, tile, sequence) of the launch before, whose grid this one's y and z
// repeat. Its four waves take every fourth split, several in flight.
constexpr int kJoinWaves = 4, kJoinAhead = 8;

__global__ void __launch_bounds__(kJoinWaves* kWave) join_kernel(Cache cache, Rows rows, Query query, Split split,
                                                                 int tile_rows, int first_tile, int first_sequence)
{
    __shared__ float sums[kJoinWaves][kMaxHeadWidth], totals[kJoinWaves];
    const int slot = blockIdx.x % split.row_slots, head = blockIdx.x / split.row_slots;
    RowTile tl;
    if (!find_tile(rows, query, first_sequence + blockIdx.z, first_tile + (int) (gridDim.y - 1 - blockIdx.y), tile_rows,
                   tl))
        return;
    const int pair = tl.first + slot, used = splits_used(tl, split.span);
    if (pair > tl.last || used == 1)
        return;
    const int width = cache.head_width, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int unit = ((int) blockIdx.z * (int) gridDim.y + (int) blockIdx.y) * cache.heads + head;
    const float* first = partial_row(split, unit, 0, slot, width);
    const size_t pitch = (size_t) split.row_slots * (width + 2);

    // Every wave the largest of all; then a wave each fourth split, eight in flight.
    float largest = -INFINITY;
    for (int i = lane; i < used; i += kWave)
        largest = fmaxf(largest, first[i * pitch]);
    largest = wave_max(largest);

    const int c0 = min(lane, width - 1), c1 = min(lane + kWave, width - 1);
    float low = 0.f, high = 0.f, denominator = 0.f;
    for (int i0 = wave; i0 < used; i0 += kJoinAhead * kJoinWaves)
    {
        float top[kJoinAhead], total[kJoinAhead], a[kJoinAhead], b[kJoinAhead];
#pragma unroll
        for (int i = 0; i < kJoinAhead; ++i)
        {
            const float* part = first + min(i0 + i * kJoinWaves, used - 1) * pitch;
            top[i] = part[0];
            total[i] = part[1];
            a[i] = part[2 + c0];
            b[i] = part[2 + c1];
        }
#pragma unroll
        for (int i = 0; i < kJoinAhead; ++i)
            if (i0 + i * kJoinWaves < used)
            {
                const float factor = part_factor(top[i], largest);
                low += factor * a[i];
                high += factor * b[i];
                denominator += factor * total[i];
            }
    }
    sums[wave][lane] = low;
    sums[wave][lane + kWave] = high;
    if (lane == 0)
        totals[wave] = denominator;
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += kJoinWaves * kWave)
    {
        float numerator = 0.f, total = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWaves; ++w)
        {
            numerator += sums[w][c];
            total += totals[w];
        }
        *out_of(tl, query, head, pair, width, c) = total == 0.f ? 0.f : numerator / total;
    }
}

// The same for few splits of many rows: a wave for each row.
__global__ void __launch_bounds__(kJoinWaves* kWave) join_few_kernel(Cache cache, Rows rows, Query query, Split split,
                                                                     int tile_rows, int first_tile, int first_sequence)
{
    const int groups = (split.row_slots + kJoinWaves - 1) / kJoinWaves;
    const int slot = blockIdx.x % groups * kJoinWaves + threadIdx.x / kWave, head = blockIdx.x / groups;
    RowTile tl;
    if (!find_tile(rows, query, first_sequence + blockIdx.z, first_tile + (int) (gridDim.y - 1 - blockIdx.y), tile_rows,
                   tl))
        return;
    const int pair = tl.first + slot, used = splits_used(tl, split.span);
    if (pair > tl.last || used == 1)
        return;
    const int width = cache.head_width, lane = threadIdx.x % kWave;
    const int unit = ((int) blockIdx.z * (int) gridDim.y + (int) blockIdx.y) * cache.heads + head;
    const float* first = partial_row(split, unit, 0, slot, width);
    const size_t pitch = (size_t) split.row_slots * (width + 2);
    // Lane i holds split i's maximum and sum.
    const int own = min(lane, used - 1);
    const float top = first[own * pitch], sum = lane < used ? first[own * pitch + 1] : 0.f;
    const float largest = wave_max(lane < used ? top : -INFINITY); // (every lane takes part: not in a branch)
    const float factor = part_factor(top, largest);
    const float total = wave_sum(factor * sum);
    const int c0 = min(lane, width - 1), c1 = min(lane + kWave, width - 1);
    float low = 0.f, high = 0.f;
    constexpr int kAtOnce = 4;
    for (int i0 = 0; i0 < used; i0 += kAtOnce)
    {
        float a[kAtOnce], b[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
        {
            const float* part = first + min(i0 + i, used - 1) * pitch + 2;
            a[i] = part[c0];
            b[i] = part[c1];
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
        {
            if (i0 + i >= used)
                break;
            const float f = __shfl(factor, i0 + i);
            low += f * a[i];
            high += f * b[i];
        }
    }
    float* const out = out_of(tl, query, head, pair, width, 0);
    if (lane < width)
        out[lane] = total == 0.f ? 0.f : low / total;
    if (lane + kWave < width)
        out[lane + kWave] = total == 0.f ? 0.f : high / total;
}
static_assert(kFusedSplits <= kWave, "a lane for each split");

constexpr int kMostBlocks = 65535; // of a launch's y and z extents

void launch_tiles(hipStream_t stream, dim3 grid, int storage, const Cache& cache, const Rows& rows,
                  const Query& query, const Split& split, int tile_rows, int first_tile, int first_sequence)
{
    by_storage(storage, [&](auto type) {
        auto run = [&](auto width, auto full) {
            if constexpr (width() == 64)
                if (tile_rows == 32)
                {
                    tile_attention_kernel<type(), width(), full(), 2><<<grid, kTileWaves * kWave, 0, stream>>>(
                        cache, rows, query, split, first_tile, first_sequence);
                    return;
                }
            tile_attention_kernel<type(), width(), full(), 1>
                <<<grid, kTileWaves * kWave, 0, stream>>>(cache, rows, query, split, first_tile, first_sequence);
        };
        using Narrow = std::integral_constant<int, 64>;
        using Wide = std::integral_constant<int, 128>;
        cache.head_width == 64    ? run(Narrow {}, std::true_type {})
        : cache.head_width == 128 ? run(Wide {}, std::true_type {})
        : cache.head_width < 64   ? run(Narrow {}, std::false_type {})
                                  : run(Wide {}, std::false_type {});
    });
}
} // namespace

hipError_t attention(hipStream_t stream, const wsp_paged_cache& cache, const wsp_paged_rows& rows, const float* q,
                     int q_stride, int heads, bool causal, float scale, float* out, int out_stride,
                     const Scratch& scratch)
{
    if (rows.max_count == 0)
        return hipSuccess;
    const Query query {q, q_stride, heads, heads / cache.heads, causal, scale * 1.4426950408889634f, out, out_stride};
    const Plan plan = plan_attention(cache, rows, query.group, scratch.bytes / sizeof(float));
    const Split split {plan.splits, plan.span, plan.row_slots, static_cast<float*>(scratch.data),
                       plan.fused ? scratch.counters : nullptr};
    const Cache pool = device_cache(cache);
    const Rows packed = device_rows(cache, rows);
    for (int s = 0; s < rows.sequences; s += plan.slice)
        for (int t = 0; t < plan.tiles; t += kMostBlocks)
        {
            const dim3 grid(split.splits * cache.heads, std::min(plan.tiles - t, kMostBlocks),
                            std::min(rows.sequences - s, plan.slice));
            if (plan.tile_rows == kChunkRows)
                launch_chunks(stream, grid, cache.storage, pool, packed, query, split, t, s);
            else
                launch_tiles(stream, grid, cache.storage, pool, packed, query, split, plan.tile_rows, t, s);
            if (split.splits > kFusedSplits)
                join_kernel<<<dim3(cache.heads * split.row_slots, grid.y, grid.z), kJoinWaves * kWave, 0, stream>>>(
                    pool, packed, query, split, plan.tile_rows, t, s);
            else if (split.splits > 1 && !plan.fused)
                join_few_kernel<<<dim3(cache.heads * ((split.row_slots + kJoinWaves - 1) / kJoinWaves), grid.y, grid.z),
                                  kJoinWaves * kWave, 0, stream>>>(pool, packed, query, split, plan.tile_rows, t, s);
        }
    return hipGetLastError();
}
} // namespace wsp::paged
