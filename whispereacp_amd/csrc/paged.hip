// The paged cache's rows: storing new ones and reading them back
// (include/wsp_hip.h, wsp_hip_paged_append and wsp_hip_paged_read). Every address
// of the pool comes from paged_plan.h's checked look-ups.
#include "paged.h"
#include "paged_device.h"

#include <algorithm>

namespace wsp::paged
{
namespace
{
constexpr int kBlock = 256, kWavesPerBlock = kBlock / kWave;
constexpr int kMinExponent = -80, kMaxExponent = 120;

// The power of two of an E4M3 row: the least k in range with amax <= 448·2^k
// (448 = 1.75·2^8).
__device__ __forceinline__ int row_exponent(float amax)
{
    const uint32_t bits = __float_as_uint(amax);
    const int k = (int) (bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
    return min(max(k, kMinExponent), kMaxExponent);
}

__device__ __forceinline__ float finite_magnitude(float v)
{
    const float a = fabsf(v);
    return a < INFINITY ? a : 0.f; // (false for NaN too)
}

// Four values as E4M3 bytes of v·2^-k; infinities and NaN become NaN.
__device__ __forceinline__ uint32_t to_e4m3(const float4v v, int k)
{
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        s[i] = isfinite(v[i]) ? ldexpf(v[i], -k) : __builtin_nanf("");
    int packed = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
    packed = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], packed, true);
    return (uint32_t) packed;
}

__device__ __forceinline__ float4v from_e4m3(uint32_t packed)
{
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8((int) packed, false);
    const auto high = __builtin_amdgcn_cvt_pk_f32_fp8((int) packed, true);
    return float4v {low[0], low[1], high[0], high[1]};
}

// Four consecutive stored values, `index` a multiple of four; E4M3 without its
// row's power of two.
template <int ST>
__device__ __forceinline__ float4v load_stored4(const void* pool, size_t index)
{
    if constexpr (ST == kF32)
        return *reinterpret_cast<const float4v*>(static_cast<const float*>(pool) + index);
    else if constexpr (ST == kF16)
    {
        const half4 h = *reinterpret_cast<const half4*>(static_cast<const _Float16*>(pool) + index);
        return float4v {(float) h[0], (float) h[1], (float) h[2], (float) h[3]};
    }
    else if constexpr (ST == kBF16)
    {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(pool) + index);
        return float4v {__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                        __uint_as_float(u.y & 0xFFFF0000u)};
    }
    else
        return from_e4m3(*reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(pool) + index));
}

template <int ST>
__device__ __forceinline__ void store_stored4(void* pool, size_t index, const float4v v, int k)
{
    if constexpr (ST == kF32)
        *reinterpret_cast<float4v*>(static_cast<float*>(pool) + index) = v;
    else if constexpr (ST == kF16)
    {
        const half4 h = {(_Float16) v[0], (_Float16) v[1], (_Float16) v[2], (_Float16) v[3]};
        *reinterpret_cast<half4*>(static_cast<_Float16*>(pool) + index) = h;
    }
    else if constexpr (ST == kBF16)
    {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        const bf16x4 h = {(__bf16) v[0], (__bf16) v[1], (__bf16) v[2], (__bf16) v[3]};
        *reinterpret_cast<bf16x4*>(static_cast<uint16_t*>(pool) + index) = h;
    }
    else
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(pool) + index) = to_e4m3(v, k);
}

// ---------------------------------------------------------------------------
// Append and read: a wave a packed row, LANES lanes (16 for heads up to 64 wide, 32
// for wider ones) a head, four values of its key and of its value each, and kTurns
// heads one after the other, all their loads in flight at once. The row's sequence,
// position and page are the same for the wave, so the search and the addresses are
// scalar. Append takes a head's largest magnitude over its lanes: a row is read once.
// Bound by memory: 64k rows of eight E4M3 heads of 128 read back in 131 us, 5.1 TB/s (as
// a large copy), up to 4096 rows of eight such sequences stored in 36, 4.4 TB/s; a step's
// few rows by the launch (3.5 us). (Lanes that searched and divided for themselves, one
// head each: 248 and 46 us.)
// ---------------------------------------------------------------------------
constexpr int kTurns = 4;

template <int LANES>
__device__ __forceinline__ float lanes_max(float v)
{
#pragma unroll
    for (int offset = LANES / 2; offset > 0; offset >>= 1)
        v = fmaxf(v, __shfl_xor(v, offset, LANES));
    return v;
}

// Where a packed row lies: its page (-1: none) and its place there.
struct Place
{
    int sequence, page, place;
    bool before; // its position is before its sequence
};

__device__ __forceinline__ Place place_of(const Cache& cache, const Rows& rows, int row)
{
    Place at {-1, -1, 0, false};
    if (row < 0 || row >= rows.rows)
        return at;
    at.sequence = sequence_of(rows.starts, rows.sequences, row);
    if (at.sequence < 0)
        return at;
    const long long position = position_of(rows.starts, rows.lengths, at.sequence, row);
    at.before = position < 0;
    if (!at.before)
    {
        at.page = page_at(cache, rows, at.sequence, (int) position);
        at.place = (int) position & ((1 << cache.page_shift) - 1);
    }
    return at;
}

template <int ST, int LANES>
__global__ void __launch_bounds__(kBlock)
    append_kernel(Cache cache, Rows rows, int first_row, const float* __restrict__ keys, int key_stride,
                  const float* __restrict__ values, int value_stride)
{
    const int row = first_row + (int) blockIdx.x * kWavesPerBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const Place at = place_of(cache, rows, row);
    if (at.page < 0)
        return;
    constexpr int kHeads = kWave / LANES; // a turn
    const int first = blockIdx.y * kHeads * kTurns + threadIdx.x % kWave / LANES, c = 4 * (threadIdx.x % LANES);
    const int width = cache.head_width;
    const bool inside = c < width;
    const float* const key_row = keys + (size_t) row * key_stride;
    const float* const value_row = values + (size_t) row * value_stride;
    float4v k[kTurns], v[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
    {
        const int head = first + kHeads * i;
        k[i] = v[i] = float4v {0.f, 0.f, 0.f, 0.f};
        if (inside && head < cache.heads)
        {
            k[i] = *reinterpret_cast<const float4u*>(key_row + (size_t) head * width + c);
            v[i] = *reinterpret_cast<const float4u*>(value_row + (size_t) head * width + c);
        }
    }
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
    {
        const int head = first + kHeads * i;
        const size_t slot = pool_row(at.page, head, at.place, cache.heads, cache.page_shift);
        int key_exponent = 0, value_exponent = 0;
        if constexpr (ST == kE4M3)
        {
            float key_max = 0.f, value_max = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                key_max = fmaxf(key_max, finite_magnitude(k[i][e]));
                value_max = fmaxf(value_max, finite_magnitude(v[i][e]));
            }
            key_exponent = row_exponent(lanes_max<LANES>(key_max));
            value_exponent = row_exponent(lanes_max<LANES>(value_max));
            if (c == 0 && head < cache.heads)
            {
                cache.key_exponents[slot] = (uint8_t) (key_exponent + kExponentBias);
                cache.value_exponents[slot] = (uint8_t) (value_exponent + kExponentBias);
            }
        }
        if (inside && head < cache.heads)
        {
            store_stored4<ST>(cache.keys, slot * width + c, k[i], key_exponent);
            store_stored4<ST>(cache.values, slot * width + c, v[i], value_exponent);
        }
    }
}

template <int ST, int LANES>
__global__ void __launch_bounds__(kBlock)
    read_kernel(Cache cache, Rows rows, int first_row, float* __restrict__ keys, int key_stride,
                float* __restrict__ values, int value_stride)
{
    const int row = first_row + (int) blockIdx.x * kWavesPerBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const Place at = place_of(cache, rows, row);
    if (at.sequence < 0)
        return;
    constexpr int kHeads = kWave / LANES; // a turn
    const int first = blockIdx.y * kHeads * kTurns + threadIdx.x % kWave / LANES, c = 4 * (threadIdx.x % LANES);
    const int width = cache.head_width;
    if (c >= width)
        return;
    float4v k[kTurns], v[kTurns];
    int key_exponents[kTurns], value_exponents[kTurns];
    const float other = at.before ? 0.f : __builtin_nanf(""); // where there is no page
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
    {
        const int head = first + kHeads * i;
        k[i] = v[i] = float4v {other, other, other, other};
        key_exponents[i] = value_exponents[i] = kExponentBias;
        if (at.page >= 0 && head < cache.heads)
        {
            const size_t slot = pool_row(at.page, head, at.place, cache.heads, cache.page_shift);
            k[i] = load_stored4<ST>(cache.keys, slot * width + c);
            v[i] = load_stored4<ST>(cache.values, slot * width + c);
            if constexpr (ST == kE4M3)
            {
                key_exponents[i] = cache.key_exponents[slot];
                value_exponents[i] = cache.value_exponents[slot];
            }
        }
    }
    float* const key_row = keys + (size_t) row * key_stride;
    float* const value_row = values + (size_t) row * value_stride;
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
    {
        const int head = first + kHeads * i;
        if (head >= cache.heads)
            return;
        if constexpr (ST == kE4M3)
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                k[i][e] = ldexpf(k[i][e], key_exponents[i] - kExponentBias);
                v[i][e] = ldexpf(v[i][e], value_exponents[i] - kExponentBias);
            }
        *reinterpret_cast<float4u*>(key_row + (size_t) head * width + c) = k[i];
        *reinterpret_cast<float4u*>(value_row + (size_t) head * width + c) = v[i];
    }
}

// f called with the storage and the lanes of a head as compile-time constants, the
// grid (rows, and the heads that a wave does not take) and the first row, as often as
// a launch's x extent takes.
constexpr int kMostRows = 1 << 24;

template <class F>
void by_lanes(const wsp_paged_cache& cache, const wsp_paged_rows& rows, F&& f)
{
    by_storage(cache.storage, [&](auto storage) {
        auto run = [&](auto lanes) {
            constexpr int kHeads = kTurns * kWave / decltype(lanes)::value;
            for (long long first = 0; first < rows.rows; first += kMostRows)
            {
                const int count = (int) std::min<long long>(rows.rows - first, kMostRows);
                f(storage, lanes,
                  dim3((count + kWavesPerBlock - 1) / kWavesPerBlock, (cache.heads + kHeads - 1) / kHeads), (int) first);
            }
        };
        cache.head_width <= 64 ? run(std::integral_constant<int, 16> {}) : run(std::integral_constant<int, 32> {});
    });
}
} // namespace

hipError_t append(hipStream_t stream, const wsp_paged_cache& cache, const wsp_paged_rows& rows, const float* keys,
                  int key_stride, const float* values, int value_stride)
{
    by_lanes(cache, rows, [&](auto storage, auto lanes, dim3 grid, int first) {
        append_kernel<storage(), lanes()><<<grid, kBlock, 0, stream>>>(
            device_cache(cache), device_rows(cache, rows), first, keys, key_stride, values, value_stride);
    });
    return hipGetLastError();
}

hipError_t read(hipStream_t stream, const wsp_paged_cache& cache, const wsp_paged_rows& rows, float* keys,
                int key_stride, float* values, int value_stride)
{
    by_lanes(cache, rows, [&](auto storage, auto lanes, dim3 grid, int first) {
        read_kernel<storage(), lanes()><<<grid, kBlock, 0, stream>>>(
            device_cache(cache), device_rows(cache, rows), first, keys, key_stride, values, value_stride);
    });
    return hipGetLastError();
}
} // namespace wsp::paged
