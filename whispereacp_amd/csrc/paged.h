// Host-side launchers of the paged cache's kernels (paged.hip,
// paged_attention.hip); arguments are checked by paged_capi.hip.
#pragma once

#include "../../include/wsp_hip.h"

#include <hip/hip_runtime.h>

namespace wsp::paged
{
// Memory for the attention's partial rows, and kSplitUnits counters that are zero
// between calls.
struct Scratch
{
    void* data;
    size_t bytes;
    unsigned int* counters;
};

hipError_t append(hipStream_t stream, const wsp_paged_cache& cache, const wsp_paged_rows& rows, const float* keys,
                  int key_stride, const float* values, int value_stride);
hipError_t read(hipStream_t stream, const wsp_paged_cache& cache, const wsp_paged_rows& rows, float* keys,
                int key_stride, float* values, int value_stride);
hipError_t attention(hipStream_t stream, const wsp_paged_cache& cache, const wsp_paged_rows& rows, const float* q,
                     int q_stride, int heads, bool causal, float scale, float* out, int out_stride,
                     const Scratch& scratch);
} // namespace wsp::paged
