// Attention of many rows over the pages of a cache of 16 or 8 bits: chunks of a
// prompt (include/wsp_hip.h, wsp_hip_paged_attention).
#include "paged_attention.h"

namespace wsp::paged
{
namespace
{
typedef float float16v __attribute__((ext_vector_type(16)));

// c + a·b over 16 k of 16-bit values of type OT, a 32 x 32 tile.
template <int OT>
__device__ __forceinline__ float16v mfma32(u32x4 a, u32x4 b, float16v c)
{
    if constexpr (OT == kF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                        0, 0, 0);
}

// The larger, and the sum, over the two halves of a wave.
__device__ __forceinline__ float halves_max(float v)
{
    const uint32_t half = __float_as_uint(v);
    const auto halves = __builtin_amdgcn_permlane32_swap(half, half, false, false);
    return fmaxf(__uint_as_float((uint32_t) halves[0]), __uint_as_float((uint32_t) halves[1]));
}
__device__ __forceinline__ float halves_sum(float v)
{
    const uint32_t half = __float_as_uint(v);
    const auto halves = __builtin_amdgcn_permlane32_swap(half, half, false, false);
    return __uint_as_float((uint32_t) halves[0]) + __uint_as_float((uint32_t) halves[1]);
}

// A barrier for LDS alone: loads from memory stay in flight across it.
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---------------------------------------------------------------------------
// Many rows: attention of a tile of 128 pairs (new row, head of the group), 32 a
// wave, over keys [split·span, +span) of one cached head, 64 at a time through LDS. The
// block converts and transposes what the storage holds once for its 128 pairs: keys as
// [key][channel], values as [channel][key], 16-bit operands of v_mfma_f32_32x32x16.
//
// S^T = K·Q^T leaves lane (n, h) with keys 8i + 4h + r (i, r < 4) of each 32 and
// pair n. Its values 8s .. 8s + 7 (s < 2) are the operand of the s-th product over
// 16 keys of O^T = V^T·P^T when that takes keys 4h .. 4h + 3 and 8 + 4h .. + 3 from
// lane half h, so the transposed values keep those eight in one 16-byte run and
// the weights cross no lanes.
//
// Queries and weights go in 16-bit parts, with the scalings of the kernel for few
// rows. E4M3 rows' powers of two are multiplied into the 16-bit operands, relative to a
// base (paged_attention.h; the keys' is their first one's). A tile with a key's power
// outside what they take keeps its keys as they are and multiplies their scores; one
// with such a value row goes as bf16 for the value products.
//
// While a tile is worked on the next is in flight to registers, and two blocks a CU
// fill each other's barriers; a wave at the matrix cores goes before one at vector
// work. Bound by both together: two chunks of 2048 rows over 16384 E4M3 positions (32
// query heads over eight, heads of 128) take 2.1 ms, 0.5 PFLOP/s of the algorithm and twice
// that in two-part products, of the 1.08 an 8192-cubed fp16 library product reaches; the
// matrix cores are busy 43% of the time, the vector units 45%, seldom at once (with a
// value row of zeros in every 64 positions 2.55 ms). (Eight waves a block, each over half the keys: 2.6 ms, with two tiles
// in LDS 3.6, its spills waiting for the loads in flight.) The accumulators are the
// matrix cores' own through all keys: 1.2·10^-6 off in that case, 4·10^-7 where every 32
// keys are summed apart, at 32 more vector instructions a tile.
// ---------------------------------------------------------------------------
constexpr int kChunkWaves = 4, kChunkKeys = 64;

// The 16-byte run of run c of eight keys of a channel's row: eight consecutive
// rows, and every fourth of 32, lie in different bank groups.
__device__ __forceinline__ int value_slot(int row, int c)
{
    return 8 * row + (c ^ (row & 7) ^ (row >> 3 & 3));
}

template <int W>
__device__ __forceinline__ int key_slot(int key, int c)
{
    return key * (W / 8) + (c ^ (key & 7));
}

// Eight E4M3 bytes times 2^power (as a float) as fp16.
__device__ __forceinline__ u32x4 e4m3_run(uint32_t low, uint32_t high, float power)
{
    return u32x4 {e4m3_to_halves<false>(low, power), e4m3_to_halves<true>(low, power),
                  e4m3_to_halves<false>(high, power), e4m3_to_halves<true>(high, power)};
}

// Waves a SIMD: three (E4M3 heads of 64, 512 rows over 2048 keys of 12 heads, 16 sequences:
// 219 us with two), two, or one, as many as do not make the registers spill into the loop.
template <int ST, int C, bool FULL>
constexpr int kChunkOccupancy = (ST == kBF16 && C >= 96) || (!FULL && C == 128) ? 1
                                : ST != kBF16 && FULL && C == 64                ? 3
                                                                                : 2;

// Heads lie in LDS as W channels (64 or 128), of which C are worked on (a multiple of
// 32); FULL: the heads are C wide.
template <int ST, int W, int C, bool FULL>
__global__ void __launch_bounds__(kChunkWaves* kWave, (kChunkOccupancy<ST, C, FULL>))
    chunk_attention_kernel(Cache cache, Rows rows, Query query, Split split, int first_tile, int first_sequence)
{
    constexpr int OT = operand_of<ST>, kParts = parts_of<OT>();
    constexpr float kBias = OT == kF16 ? 14.f : 0.f;
    constexpr int kThreads = kChunkWaves * kWave;
    constexpr int kKeyRuns = kChunkKeys * W / 8 / kThreads;      // runs of eight channels a thread loads
    constexpr int kKeyWords = 2 * bytes_of<ST>;                  // dwords of one as stored
    constexpr int kValueChannels = W / 32;                       // channels of eight keys a thread loads
    constexpr int kValueWords = (kValueChannels * bytes_of<ST> + 3) / 4;
    __shared__ u32x4 ks[kChunkKeys * W / 8];
    __shared__ u32x4 vs[W * kChunkKeys / 8];
    __shared__ __align__(16) int key_power[kChunkKeys];
    // The last tile (its first key + 1) with a non-finite value that some pair sees, and
    // the last E4M3 ones whose keys' and values' powers the operands do not take, and
    // with a value's past kLoudest.
    __shared__ int odd_tile, apart_tile, wide_tile, loud_tile;

    const int which = blockIdx.x % split.splits, head = blockIdx.x / split.splits;
    const int sequence = first_sequence + blockIdx.z;
    const int tile = first_tile + (int) (gridDim.y - 1 - blockIdx.y); // (the tiles that see most come first)
    RowTile tl;
    if (!find_tile(rows, query, sequence, tile, kChunkRows, tl))
        return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, n = lane % 32, h = lane / 32;
    const int width = FULL ? C : cache.head_width, row_bytes = width * bytes_of<ST>;
    const int page_mask = (1 << cache.page_shift) - 1;
    const int* table = rows.pages + (size_t) sequence * rows.table_width;
    const int used = splits_used(tl, split.span);
    if (which >= used)
        return;
    const int begin = which * split.span, end = tl.poisoned ? 0 : min(begin + split.span, tl.most);

    // This wave's pairs: lane (n, h) holds channels 16j + 8h .. + 7 of pair n.
    const int first = tl.first + 32 * wave, pair = first + n;
    const bool real = pair <= tl.last;
    const int seen = real ? min(keys_seen(query, tl, pair), end) : 0;
    const int wave_least = first <= tl.last ? min(keys_seen(query, tl, first), end) : 0;
    const int wave_most = first <= tl.last ? min(keys_seen(query, tl, min(first + 31, tl.last)), end) : 0;
    u32x4 qp[C / 16][kParts];
    int shift = 0; // the parts are the query's times 2^shift
    {
        const float* at = query.q + (size_t) (tl.first_row + (real ? pair : tl.first) / query.group) * query.q_stride
                          + (size_t) (head * query.group + (real ? pair : tl.first) % query.group) * width;
        float x[C / 16][8];
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < C / 16; ++j)
#pragma unroll
            for (int i = 0; i < 8; i += 4)
            {
                float4v run = {0.f, 0.f, 0.f, 0.f};
                if (real && (FULL || 16 * j + 8 * h < width))
                    run = *reinterpret_cast<const float4u*>(at + 16 * j + 8 * h + i);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    x[j][i + e] = run[e] * query.scale;
                    top = fmaxf(top, fabsf(x[j][i + e]));
                }
            }
        if constexpr (OT == kF16)
        {
            // 2^13 <= top·2^shift < 2^14 (a pair of zeros, or not finite: as it is)
            top = halves_max(top);
            shift = top > 0.f && top < INFINITY ? min(140 - (int) (__float_as_uint(top) >> 23), 126) : 0;
        }
#pragma unroll
        for (int j = 0; j < C / 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                uint32_t cut[3];
                if constexpr (OT == kF16)
                    cut_pair<OT>(ldexpf(x[j][2 * i], shift), ldexpf(x[j][2 * i + 1], shift), cut);
                else
                    cut_pair<OT>(x[j][2 * i], x[j][2 * i + 1], cut);
#pragma unroll
                for (int p = 0; p < kParts; ++p)
                    qp[j][p][i] = cut[p];
            }
    }

    // What a thread loads of a tile: key runs threadIdx.x + 256·i (run key_run of key
    // key_of + kKeysAtOnce·i), and of the eight keys of run `value_run` (16·wave +
    // 4h .. + 3 and 8 more on) the channels from value_channel on.
    constexpr int kKeysAtOnce = kThreads / (W / 8); // 16 or 32
    const int key_run = threadIdx.x % (W / 8), key_of = threadIdx.x / (W / 8);
    const int value_channel = threadIdx.x % 32 * kValueChannels, value_run = 2 * wave + h;
    // (Lanes past the row read its start: keys' runs there are staged as zeros, values'
    // channels there reach no output.)
    const bool key_real = (FULL && C == W) || 8 * key_run < width;
    const uint32_t key_offset = key_of % 16 * row_bytes + (key_real ? 8 * key_run : 0) * bytes_of<ST>;
    const uint32_t value_offset =
        4 * h * row_bytes + ((FULL && C == W) || value_channel < width ? value_channel : 0) * bytes_of<ST>;
    struct Raw
    {
        uint32_t k[kKeyRuns][kKeyWords];
        uint32_t v[8][kValueWords];
        uint32_t ke[ST == kE4M3 ? kKeyRuns : 1], ve[2]; // the exponents of those rows
    } raw;
    typedef int int4v __attribute__((ext_vector_type(4)));
    static_assert(kChunkKeys == 64, "four sixteens");
    int4v pages; // of each sixteen of the tile in flight (-1: none)

    auto load = [&](int k0) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
            pages[s] = k0 + 16 * s < end ? page_of(table, rows.table_width, cache.page_shift, cache.pages, k0 + 16 * s)
                                         : -1;
        // (Pages are the same for a whole wave, so these addresses are scalars.)
        auto row_of = [&](int page, int key) {
            return pool_row(max(page, 0), head, key & page_mask, cache.heads, cache.page_shift);
        };
#pragma unroll
        for (int i = 0; i < kKeyRuns; ++i)
        {
            const bool second = kKeysAtOnce == 32 && wave >= 2; // of the 32 keys of one i
            const int page = kKeysAtOnce == 16 ? pages[i] : i == 0 ? (second ? pages[1] : pages[0])
                                                                   : (second ? pages[3] : pages[2]);
            const size_t row = row_of(page, k0 + kKeysAtOnce * i + (second ? 16 : 0));
            load_words(static_cast<const char*>(cache.keys) + row * row_bytes + key_offset, raw.k[i]);
            if constexpr (ST == kE4M3)
                raw.ke[i] = *global(cache.key_exponents + row + (uint32_t) (key_of % 16));
        }
        const int page = wave == 0 ? pages[0] : wave == 1 ? pages[1] : wave == 2 ? pages[2] : pages[3];
        const size_t row = row_of(page, k0 + 16 * wave);
        const char* values = static_cast<const char*>(cache.values) + row * row_bytes;
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            const char* at = values + (8 * (i / 4) + i % 4) * row_bytes + value_offset;
            if constexpr (kValueChannels * bytes_of<ST> == 2)
                raw.v[i][0] = *global(reinterpret_cast<const uint16_t*>(at));
            else
                load_words(at, raw.v[i]);
        }
        if constexpr (ST == kE4M3)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                raw.ve[i] = *(const __attribute__((address_space(1))) u32u*) (cache.value_exponents + row + 8 * i
                                                                             + (uint32_t) (4 * h));
    };

    // E4M3: the powers that the operands leave out.
    int key_base = kExponentBias, value_base = kExponentBias;
    if (ST == kE4M3 && begin < end)
    {
        const int page = page_of(table, rows.table_width, cache.page_shift, cache.pages, begin);
        const size_t row = pool_row(max(page, 0), head, begin & page_mask, cache.heads, cache.page_shift);
        key_base = first_base(cache.key_exponents[row]);
        value_base = first_base(cache.value_exponents[row]);
    }
    // 2^(byte - base) as a float's bits, for bytes that a base takes.
    auto power_bits = [](uint32_t byte, int base) { return (byte + (uint32_t) (kExponentBias - base)) << 23; };
    auto value_byte = [&](int i) { return raw.ve[i / 4] >> (8 * (i % 4)) & 255u; };
    auto key_of_value = [&](int i) { return 16 * wave + 8 * (i / 4) + 4 * h + i % 4; };

    auto bad_pages = [&](int k0) { // a bit for each sixteen of the tile in flight
        int bad = 0;
#pragma unroll
        for (int s = 0; s < 4; ++s)
            bad |= pages[s] < 0 && k0 + 16 * s < end ? 1 << s : 0;
        return bad;
    };

    // Before the barrier behind which the tile goes to LDS: what its rows' powers ask for.
    auto look = [&](int k0) {
        if constexpr (ST == kE4M3)
        {
            int key_bytes[kKeyRuns], value_bytes[8];
#pragma unroll
            for (int i = 0; i < kKeyRuns; ++i)
                key_bytes[i] = (int) raw.ke[i];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                value_bytes[i] = (int) value_byte(i);
            if (k0 + kChunkKeys > end || bad_pages(k0) != 0)
            {
                // Rows that no pair sees may hold anything.
                const int bad = bad_pages(k0);
#pragma unroll
                for (int i = 0; i < kKeyRuns; ++i)
                {
                    const int key = key_of + kKeysAtOnce * i;
                    if (k0 + key >= end || (bad >> (key / 16) & 1) != 0)
                        key_bytes[i] = key_base;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k0 + key_of_value(i) >= end || (bad >> wave & 1) != 0)
                        value_bytes[i] = value_base;
            }
            int low = key_bytes[0], high = key_bytes[0];
#pragma unroll
            for (int i = 1; i < kKeyRuns; ++i)
            {
                low = min(low, key_bytes[i]);
                high = max(high, key_bytes[i]);
            }
            if (!base_takes(key_base, low, high))
                apart_tile = k0 + 1;
            low = high = value_bytes[0];
#pragma unroll
            for (int i = 1; i < 8; ++i)
            {
                low = min(low, value_bytes[i]);
                high = max(high, value_bytes[i]);
            }
            if (!base_takes(value_base, low, high))
            {
                wide_tile = k0 + 1;
                if (high > kLoudest)
                    loud_tile = k0 + 1;
            }
        }
    };

    // The raw tile to LDS.
    auto stage = [&](int k0, bool apart, auto type) __attribute__((always_inline)) {
        constexpr int VT = decltype(type)::value;
        if (ST == kE4M3 && apart && key_run == 0)
#pragma unroll
            for (int i = 0; i < kKeyRuns; ++i)
                key_power[key_of + kKeysAtOnce * i] = (int) raw.ke[i] - kExponentBias;
#pragma unroll
        for (int i = 0; i < kKeyRuns; ++i)
        {
            u32x4 run;
            if constexpr (ST == kE4M3)
                run = e4m3_run(raw.k[i][0], raw.k[i][1],
                               apart ? 1.f : __uint_as_float(power_bits(raw.ke[i], key_base)));
            else
                run = u32x4 {raw.k[i][0], raw.k[i][1], raw.k[i][2], raw.k[i][3]};
            if (!key_real)
                run = u32x4 {0, 0, 0, 0};
            ks[key_slot<W>(key_of + kKeysAtOnce * i, key_run)] = run;
        }
        // Values as pairs of channels, then pairs of keys of one channel.
        uint32_t pairs[8][kValueChannels / 2];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if constexpr (ST == kE4M3 && VT == kBF16)
            {
                const int power = (int) value_byte(i) - value_base;
                pairs[i][0] = e4m3_to_bf16<false>(raw.v[i][0], power);
                if constexpr (kValueChannels > 2)
                    pairs[i][1] = e4m3_to_bf16<true>(raw.v[i][0], power);
            }
            else if constexpr (ST == kE4M3)
            {
                const float power = __uint_as_float(power_bits(value_byte(i), value_base));
                pairs[i][0] = e4m3_to_halves<false>(raw.v[i][0], power);
                if constexpr (kValueChannels > 2)
                    pairs[i][1] = e4m3_to_halves<true>(raw.v[i][0], power);
            }
            else
#pragma unroll
                for (int c = 0; c < kValueChannels / 2; ++c)
                    pairs[i][c] = raw.v[i][c];
        // A weight of zero hides a value only while it is finite: values that no pair
        // sees count as zero, and non-finite ones among keys that some pairs see are
        // added behind the products, to those pairs alone.
        const int page = wave == 0 ? pages[0] : wave == 1 ? pages[1] : wave == 2 ? pages[2] : pages[3];
        if (k0 + kChunkKeys > min(tl.least, end) || page < 0)
        {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                const bool unseen = k0 + key_of_value(i) >= end || page < 0;
#pragma unroll
                for (int c = 0; c < kValueChannels / 2; ++c)
                {
                    const uint32_t kept = unseen ? 0u : finite_halves<VT>(pairs[i][c]);
                    odd = odd || (!unseen && kept != pairs[i][c]);
                    pairs[i][c] = kept;
                }
            }
            if (odd)
                odd_tile = k0 + 1;
        }
#pragma unroll
        for (int c = 0; c < kValueChannels; c += 2)
        {
            u32x4 low, high;
#pragma unroll
            for (int d = 0; d < 4; ++d)
            {
                low[d] = __builtin_amdgcn_perm(pairs[2 * d + 1][c / 2], pairs[2 * d][c / 2], 0x05040100);
                high[d] = __builtin_amdgcn_perm(pairs[2 * d + 1][c / 2], pairs[2 * d][c / 2], 0x07060302);
            }
            vs[value_slot(value_channel + c, value_run)] = low;
            vs[value_slot(value_channel + c + 1, value_run)] = high;
        }
    };

    float16v o[C / 32];
#pragma unroll
    for (int c = 0; c < C / 32; ++c)
        o[c] = float16v {};
    float m = -INFINITY, l = 0.f;
    if (threadIdx.x == 0)
        odd_tile = apart_tile = wide_tile = loud_tile = 0;
    __syncthreads();

    if (begin < end)
        load(begin);
    for (int k0 = begin; k0 < end; k0 += kChunkKeys)
    {
        look(k0);
        lds_barrier(); // (the tile before is read)
        const bool apart = ST == kE4M3 && apart_tile == k0 + 1, wide = ST == kE4M3 && wide_tile == k0 + 1;
        if (ST == kE4M3 && wide)
        {
            const int next = wide_base(value_base, loud_tile == k0 + 1);
            const float by = ldexpf(1.f, value_base - next);
#pragma unroll
            for (int c = 0; c < C / 32; ++c)
                o[c] *= by;
            value_base = next;
            stage(k0, apart, std::integral_constant<int, kBF16> {});
        }
        else
            stage(k0, apart, std::integral_constant<int, OT> {});
        const int bad = bad_pages(k0); // (the next tile's take their place)
        // (Held below infinity: a score of zero stays zero.)
        const float known = ldexpf(1.f, min(key_base - kExponentBias - shift, 127));
        lds_barrier();
        if (k0 + kChunkKeys < end)
            load(k0 + kChunkKeys);
        if (k0 >= wave_most) // (none of this wave's pairs sees a key)
            continue;

        const bool odd = odd_tile == k0 + 1;
        // 32 keys at a time: what is live fits the registers of two blocks a CU.
#pragma unroll 1
        for (int b = 0; b < 2; ++b)
        {
            const int from = k0 + 32 * b;
            if (from >= wave_most)
                break;
            __builtin_amdgcn_s_setprio(1);
            float16v s = {};
            u32x4 key[C / 16];
#pragma unroll
            for (int j = 0; j < C / 16; ++j)
                key[j] = ks[key_slot<W>(32 * b + n, 2 * j + h)];
#pragma unroll
            for (int j = 0; j < C / 16; ++j)
#pragma unroll
                for (int p = kParts - 1; p >= 0; --p)
                    s = mfma32<OT>(key[j], qp[j][p], s);
            __builtin_amdgcn_s_setprio(0);
            // Value 4i + r of s is key 8i + 4h + r of the 32. Scores in powers of two, but
            // for `scale`, which the multiply-add before the powers takes in.
            float scale = known;
            if (ST == kE4M3 && apart)
            {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    const int4v powers = *reinterpret_cast<const int4v*>(&key_power[32 * b + 8 * i + 4 * h]);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        s[4 * i + r] = ldexpf(s[4 * i + r], powers[r] - shift);
                }
                scale = 1.f;
            }
            const bool first_bad = (bad >> (2 * b) & 1) != 0, second_bad = (bad >> (2 * b + 1) & 1) != 0;
            if (from + 32 > wave_least || first_bad || second_bad)
            {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                {
                    if (i < 8 ? first_bad : second_bad)
                        s[i] = __builtin_nanf("");
                    s[i] = from + 8 * (i / 4) + 4 * h + i % 4 < seen ? s[i] : -INFINITY;
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                top = fmaxf(top, s[i]);
            // The maximum is rounded up to a whole power of two: what it rescales stays exact.
            const float m_new = fmaxf(m, ceilf(halves_max(top) * scale));
            const float finite = m_new == -INFINITY ? 0.f : m_new, base = finite - kBias;
            if (__any(m_new != m))
            {
                const float alpha = __builtin_amdgcn_exp2f(m - finite);
                l *= alpha;
#pragma unroll
                for (int c = 0; c < C / 32; ++c)
                    o[c] *= alpha;
                m = m_new;
            }
            u32x4 first_parts[2]; // of the weights
            auto add_rows = [&](auto type) __attribute__((always_inline)) {
                constexpr int VT = decltype(type)::value;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale, -base));
                float own[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    own[i % 4] += s[i];
                l += (own[0] + own[1]) + (own[2] + own[3]);
                u32x4 weights[2][parts_of<VT>()];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                    {
                        uint32_t cut[3];
                        cut_pair<VT>(s[8 * t + 2 * i], s[8 * t + 2 * i + 1], cut);
#pragma unroll
                        for (int p = 0; p < parts_of<VT>(); ++p)
                            weights[t][p][i] = cut[p];
                    }
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int t = 0; t < 2; ++t)
                {
                    u32x4 value[C / 32];
#pragma unroll
                    for (int c = 0; c < C / 32; ++c)
                        value[c] = vs[value_slot(32 * c + n, 4 * b + 2 * t + h)];
#pragma unroll
                    for (int p = parts_of<VT>() - 1; p >= 0; --p)
#pragma unroll
                        for (int c = 0; c < C / 32; ++c)
                            o[c] = mfma32<VT>(value[c], weights[t][p], o[c]);
                    if (ST != kE4M3)
                        first_parts[t] = weights[t][0];
                }
                __builtin_amdgcn_s_setprio(0);
            };
            if (ST == kE4M3 && wide)
                add_rows(std::integral_constant<int, kBF16> {});
            else
                add_rows(std::integral_constant<int, OT> {});
            if (odd) // (rare: infinities or NaN among the new rows' values)
            {
                uint32_t parts[8]; // (opaque: nothing of this is worked out before it is needed)
                if constexpr (ST != kE4M3)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                    {
                        parts[i] = first_parts[i / 4][i % 4];
                        asm("" : "+v"(parts[i]));
                    }
#pragma unroll 1
                for (int key = 0; key < 32; ++key)
                {
                    // Key 16t + 8i + 4h + r is value 4i + r of lane half h's weights t. (Only
                    // that a weight is not zero matters: the first part of it does. E4M3 has no
                    // infinities, and NaN is NaN by any weight.)
                    float weight = 1.f;
                    if constexpr (ST != kE4M3)
                    {
                        uint32_t held = 0;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (8 * (key / 16) + 4 * (key / 8 % 2) + key % 4 == i)
                                held = i % 2 == 0 ? parts[i / 2] << 16 : parts[i / 2] & 0xFFFF0000u;
                        weight = __uint_as_float(__shfl(held, n + 32 * (key / 4 % 2)));
                    }
                    const int position = from + key;
                    const int page = page_of(table, rows.table_width, cache.page_shift, cache.pages, position);
                    if (position >= seen || page < 0)
                        continue;
                    const size_t row = pool_row(page, head, position & page_mask, cache.heads, cache.page_shift);
#pragma unroll
                    for (int c = 0; c < C / 32; ++c)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                        {
                            const int channel = 32 * c + 8 * (i / 4) + 4 * h + i % 4;
                            const float value =
                                channel < width ? stored_value<ST>(cache.values, row * width + channel) : 0.f;
                            if (!isfinite(value))
                                o[c][i] += weight * value;
                        }
                }
            }
        }
    }

    // o[c][4i + r] is channel 32c + 8i + 4h + r of pair n; times the values' power.
    l = halves_sum(l) * (ST == kE4M3 ? ldexpf(1.f, -kSumShift) : 1.f);
    if (tl.poisoned)
        l = __builtin_nanf("");
    if (!real)
        return;
    const float power = ST == kE4M3 ? ldexpf(1.f, value_base - kExponentBias - kSumShift) : 1.f;
    const float by = used > 1 ? power : l == 0.f ? 0.f : power / l;
    const int unit_index = ((int) blockIdx.z * (int) gridDim.y + (int) blockIdx.y) * cache.heads + head;
    float* const part = partial_row(split, unit_index, which, pair - tl.first, width);
    float* const out = used > 1 ? part + 2 : out_of(tl, query, head, pair, width, 0);
    if (used > 1 && h == 0)
    {
        part[0] = m;
        part[1] = l;
    }
#pragma unroll
    for (int c = 0; c < C / 32; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (FULL || 32 * c + 8 * i + 4 * h < width)
                *reinterpret_cast<float4u*>(out + 32 * c + 8 * i + 4 * h) =
                    float4v {o[c][4 * i], o[c][4 * i + 1], o[c][4 * i + 2], o[c][4 * i + 3]} * by;
}
} // namespace

void launch_chunks(hipStream_t stream, dim3 grid, int storage, const Cache& cache, const Rows& rows,
                   const Query& query, const Split& split, int first_tile, int first_sequence)
{
    by_storage(storage, [&](auto type) {
        auto run = [&](auto width, auto channels, auto full) {
            if constexpr (type() != kF32)
                chunk_attention_kernel<type(), width(), channels(), full()><<<grid, kChunkWaves * kWave, 0, stream>>>(
                    cache, rows, query, split, first_tile, first_sequence);
        };
        using Narrow = std::integral_constant<int, 64>;
        using Middle = std::integral_constant<int, 96>;
        using Wide = std::integral_constant<int, 128>;
        cache.head_width == 64    ? run(Narrow {}, Narrow {}, std::true_type {})
        : cache.head_width == 128 ? run(Wide {}, Wide {}, std::true_type {})
        : cache.head_width < 64   ? run(Narrow {}, Narrow {}, std::false_type {})
        : cache.head_width <= 96  ? run(Wide {}, Middle {}, std::false_type {})
                                  : run(Wide {}, Wide {}, std::false_type {});
    });
}
} // namespace wsp::paged
