// C ABI of the operators that leave entries out: argument checks and launches.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "context.h"
#include "dropout_kernels.h"

using namespace vetrast;

namespace
{
constexpr int64_t kDropoutAtOnce = (int64_t)1 << 33;  // elements of a launch: its threads are counted in 32 bits

template <int TYPE>
void launch_dropout(DropoutPass& l, hipStream_t stream)
{
    const dim3 grid((uint32_t)((l.n + kOptimChunk - 1) / kOptimChunk));
    if (l.residual) hipLaunchKernelGGL((dropout_kernel<TYPE, true>), grid, dim3(kBlock), 0, stream, l);
    else hipLaunchKernelGGL((dropout_kernel<TYPE, false>), grid, dim3(kBlock), 0, stream, l);
}

// Whether two stretches of memory share some of it without being the same one.
inline bool overlap(const void* a, const void* b, size_t bytes)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x != y && (x < y ? y - x : x - y) < bytes;
}
}  // namespace

extern "C" {

int vetrast_dropout(vetrast_ctx* ctx, const vetrast_dropout_args* a, void* stream_)
{
    if (!ctx || !a) return VETRAST_ERR_INVALID_ARG;
    if (a->n < 0 || a->n > kOptimMaxElements || !is_dtype(a->type) || !(a->p >= 0.0 && a->p <= 1.0)) return VETRAST_ERR_INVALID_ARG;
    if (!aligned_to(a->device_step, 8)) return VETRAST_ERR_INVALID_ARG;
    if (a->n == 0) return VETRAST_OK;
    const size_t each = dtype_bytes(a->type), bytes = (size_t)a->n * each;
    if (!a->x || !a->y || !aligned_to(a->x, each) || !aligned_to(a->y, each) || !aligned_to(a->residual, each)) return VETRAST_ERR_INVALID_ARG;
    if (overlap(a->x, a->y, bytes) || (a->residual && overlap(a->residual, a->y, bytes))) return VETRAST_ERR_INVALID_ARG;
    hipStream_t stream = (hipStream_t)stream_;
    DropoutPass l;
    l.bits  = dropout_bits(a->p, a->seed, a->step, a->device_step);
    l.scale = l.bits.threshold < 65536u ? (float)(65536.0 / (65536.0 - l.bits.threshold)) : 0.f;
    for (int64_t from = 0; from < a->n; from += kDropoutAtOnce)
    {
        l.x           = static_cast<const char*>(a->x) + (size_t)from * each;
        l.residual    = a->residual ? static_cast<const char*>(a->residual) + (size_t)from * each : nullptr;
        l.y           = static_cast<char*>(a->y) + (size_t)from * each;
        l.n           = (uint64_t)std::min(a->n - from, kDropoutAtOnce);
        l.first_block = (uint64_t)from / 8;
        if (a->type == VETRAST_F32) launch_dropout<VETRAST_F32>(l, stream);
        else if (a->type == VETRAST_BF16) launch_dropout<VETRAST_BF16>(l, stream);
        else launch_dropout<VETRAST_F16>(l, stream);
    }
    VET_HIP(ctx, hipGetLastError());
    return VETRAST_OK;
}

}  // extern "C"
