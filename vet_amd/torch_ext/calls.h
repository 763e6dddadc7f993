// What the tensor calls of this directory share: contexts, streams and what is asked of tensors.
#pragma once
#include <torch/torch.h>

#include <map>
#include <utility>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include "../../include/vetrast.h"

namespace vet_amd
{
inline void check(int st, const char* where)
{
    TORCH_CHECK(st == VETRAST_OK, "vetrast ", where, " failed: ", st, " (", vetrast_status_string(st), ")");
}

inline void* stream_on(const torch::Device& device)
{
    return (void*)c10::hip::getCurrentHIPStream(device.index()).stream();
}

inline bool capturing()
{
    return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

// What a host thread keeps. A context serves one host thread at a time and belongs to a device, a norm's workspace serves one stream of torch's.
struct Kept
{
    std::map<int, vetrast_ctx*> contexts;
    std::map<std::pair<int, void*>, torch::Tensor> workspaces;
    ~Kept()
    {
        for (auto& c : contexts) vetrast_destroy(c.second);
    }
};
inline Kept& kept()
{
    thread_local Kept k;
    return k;
}

// The caller has made `device` the current one.
inline vetrast_ctx* context_on(const torch::Device& device)
{
    vetrast_ctx*& ctx = kept().contexts[device.index()];
    if (!ctx) check(vetrast_create(&ctx), "create");
    return ctx;
}

inline int32_t type_of(const torch::Tensor& t, const char* what)
{
    switch (t.scalar_type())
    {
        case torch::kFloat32: return VETRAST_F32;
        case torch::kBFloat16: return VETRAST_BF16;
        case torch::kFloat16: return VETRAST_F16;
        default: TORCH_CHECK(false, what, " must be float32, bfloat16 or float16, not ", t.scalar_type());
    }
}

inline void check_on(const torch::Tensor& t, const torch::Device& device, const char* what)
{
    TORCH_CHECK(t.layout() == torch::kStrided && t.device() == device, what, " must be a strided tensor on ", device);
}

// The elements one behind the other in memory, whatever the order of dimensions.
inline bool dense(const torch::Tensor& t)
{
    return t.is_contiguous() || t.is_non_overlapping_and_dense();
}

inline bool same_order(const torch::Tensor& a, const torch::Tensor& b)
{
    return (a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides();
}
}  // namespace vet_amd
