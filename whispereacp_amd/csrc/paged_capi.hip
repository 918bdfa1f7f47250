// The C ABI of the paged cache (include/wsp_hip.h, wsp_hip_paged_*): argument
// checks, the context's device and its error string around paged.hip's kernels.
#include "capi_internal.h"
#include "paged.h"
#include "paged_plan.h"

using wsp::Context;

namespace
{
// The context's device made current while a call launches, whatever the
// caller's is.
class OnDevice
{
public:
    explicit OnDevice(int device)
    {
        status = hipGetDevice(&previous);
        if (status == hipSuccess && previous != device)
        {
            status = hipSetDevice(device);
            changed = status == hipSuccess;
        }
    }
    ~OnDevice()
    {
        if (changed)
            (void) hipSetDevice(previous);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;

    hipError_t status = hipSuccess;

private:
    int previous = 0;
    bool changed = false;
};

template <class Launch>
int run(Context* ctx, const wsp_paged_rows* rows, const char* what, Launch&& launch)
{
    if (rows->sequences == 0 || rows->rows == 0)
        return WSP_OK;
    const OnDevice device(ctx->device);
    const hipError_t e = device.status == hipSuccess ? launch() : device.status;
    return e == hipSuccess ? WSP_OK : wsp::context_hip(ctx, e, what);
}

int refused(Context* ctx, int status, const char* why)
{
    return wsp::context_fail(ctx, status, why);
}
} // namespace

extern "C" {

int wsp_hip_paged_append(wsp_hip_ctx* ctx, const wsp_paged_cache* cache, const wsp_paged_rows* rows,
                         const float* keys, int key_stride, const float* values, int value_stride)
{
    if (ctx == nullptr)
        return WSP_ERR_ARGUMENT;
    char why[256];
    int status = wsp::paged::refusal(cache, rows, why, sizeof(why));
    if (status == WSP_OK)
        status = wsp::paged::refusal_of_tensor(cache, rows, "key", keys, cache->heads, key_stride, why, sizeof(why));
    if (status == WSP_OK)
        status = wsp::paged::refusal_of_tensor(cache, rows, "value", values, cache->heads, value_stride, why,
                                               sizeof(why));
    if (status != WSP_OK)
        return refused(ctx, status, why);
    return run(ctx, rows, "paged append", [&] {
        return wsp::paged::append(ctx->stream, *cache, *rows, keys, key_stride, values, value_stride);
    });
}

int wsp_hip_paged_read(wsp_hip_ctx* ctx, const wsp_paged_cache* cache, const wsp_paged_rows* rows, float* keys,
                       int key_stride, float* values, int value_stride)
{
    if (ctx == nullptr)
        return WSP_ERR_ARGUMENT;
    char why[256];
    int status = wsp::paged::refusal(cache, rows, why, sizeof(why));
    if (status == WSP_OK)
        status = wsp::paged::refusal_of_tensor(cache, rows, "key", keys, cache->heads, key_stride, why, sizeof(why));
    if (status == WSP_OK)
        status = wsp::paged::refusal_of_tensor(cache, rows, "value", values, cache->heads, value_stride, why,
                                               sizeof(why));
    if (status != WSP_OK)
        return refused(ctx, status, why);
    return run(ctx, rows, "paged read", [&] {
        return wsp::paged::read(ctx->stream, *cache, *rows, keys, key_stride, values, value_stride);
    });
}

int wsp_hip_paged_attention(wsp_hip_ctx* ctx, const wsp_paged_cache* cache, const wsp_paged_rows* rows,
                            const float* q, int q_stride, int heads, int causal, float scale, float* out,
                            int out_stride)
{
    if (ctx == nullptr)
        return WSP_ERR_ARGUMENT;
    char why[256];
    int status = wsp::paged::refusal(cache, rows, why, sizeof(why));
    if (status == WSP_OK)
        status = wsp::paged::refusal_of_attention(cache, rows, heads, why, sizeof(why));
    if (status == WSP_OK)
        status = wsp::paged::refusal_of_tensor(cache, rows, "query", q, heads, q_stride, why, sizeof(why));
    if (status == WSP_OK)
        status = wsp::paged::refusal_of_tensor(cache, rows, "output", out, heads, out_stride, why, sizeof(why));
    if (status != WSP_OK)
        return refused(ctx, status, why);
    return run(ctx, rows, "paged attention", [&] {
        return wsp::paged::attention(ctx->stream, *cache, *rows, q, q_stride, heads, causal != 0, scale, out,
                                     out_stride, {ctx->parts, ctx->paged_bytes, ctx->paged_counters});
    });
}

} // extern "C"
