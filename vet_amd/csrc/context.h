// What the entry points share: the context, its timing scopes and checks of arguments.
#pragma once
#include <hip/hip_runtime.h>

#include <vector>

#include "common.h"

struct vetrast_ctx
{
    int device         = 0;
    int profiling      = 0;
    int last_hip_error = 0;
    struct Span
    {
        int scope;
        hipEvent_t start, stop;
    };
    std::vector<Span> spans;             // recorded since the last reset
    std::vector<hipEvent_t> free_events;  // recycled events
    float acc_ms[VETRAST_SCOPE_COUNT_]      = {};
    int32_t acc_launches[VETRAST_SCOPE_COUNT_] = {};
    char* lift_scratch = nullptr;  // this device's copy of the file-scope scratch array (vetrast_lift_error_static)
};

#define VET_HIP(ctx, expr)                               \
    do                                                   \
    {                                                    \
        hipError_t e_ = (expr);                          \
        if (e_ != hipSuccess)                            \
        {                                                \
            if (ctx) (ctx)->last_hip_error = (int)e_;    \
            return VETRAST_ERR_HIP;                      \
        }                                                \
    } while (0)

namespace vetrast
{
// Brackets the launches of one scope with events when profiling is on.
struct ScopeTimer
{
    vetrast_ctx* ctx;
    hipStream_t stream;
    int scope;
    hipEvent_t start = nullptr, stop = nullptr;
    bool on          = false;
    ScopeTimer(vetrast_ctx* c, hipStream_t s, int sc) : ctx(c), stream(s), scope(sc)
    {
        if (!ctx->profiling) return;
        start = take();
        stop  = take();
        if (!start || !stop) return;
        on = hipEventRecord(start, stream) == hipSuccess;
    }
    ~ScopeTimer()
    {
        if (!on) return;
        (void)hipEventRecord(stop, stream);
        ctx->spans.push_back({scope, start, stop});
    }
    hipEvent_t take()
    {
        if (!ctx->free_events.empty())
        {
            hipEvent_t e = ctx->free_events.back();
            ctx->free_events.pop_back();
            return e;
        }
        hipEvent_t e = nullptr;
        if (hipEventCreate(&e) != hipSuccess) return nullptr;
        return e;
    }
};

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool is_dtype(int32_t t) { return t == VETRAST_F32 || t == VETRAST_BF16 || t == VETRAST_F16; }
inline size_t dtype_bytes(int32_t t) { return t == VETRAST_F32 ? 4 : 2; }
constexpr int64_t kOptimMaxElements   = (int64_t)1 << 38;  // of a tensor, and of the places in flat arrays, whose blocks have numbers of 32 bits
}  // namespace vetrast
