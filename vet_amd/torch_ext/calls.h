// What the tensor calls of this directory share: contexts, streams and what is asked of tensors.
#pragma once
#include <torch/csrc/autograd/graph_task.h>
#include <torch/torch.h>

#include <map>
#include <unordered_map>
#include <unordered_set>
#include <utility>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
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

// A backward pass waits for the streams of the nodes that it comes to. In a capture each of them has to take part in it: torch otherwise records an
// event on a stream outside, and the process ends when the capture does. A leaf's node lives as long as any graph of that leaf, so one of an eager
// pass that still lives is what a captured pass would come to. What leads to `node` is looked at here, where an error can still be given; with `asked`
// (of the backward pass under way) only what that pass comes to.
using AskedNodes = std::unordered_map<torch::autograd::Node*, torch::autograd::GraphTask::ExecInfo>;
inline void check_captured_gradients(const std::shared_ptr<torch::autograd::Node>& node, const c10::Stream& here, const char* what,
                                     const AskedNodes* asked = nullptr)
{
    const auto captured = [&](const c10::Stream& stream) {
        if (stream == here) return true;
        const hipStream_t handle      = c10::hip::HIPStreamMasqueradingAsCUDA(stream).stream();
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        return handle != nullptr && hipStreamIsCapturing(handle, &status) == hipSuccess && status == hipStreamCaptureStatusActive;  // forked within the capture
    };
    std::vector<std::shared_ptr<torch::autograd::Node>> nodes{node};
    std::unordered_set<torch::autograd::Node*> seen;
    while (!nodes.empty())
    {
        const auto next = std::move(nodes.back());
        nodes.pop_back();
        if (!next || !seen.insert(next.get()).second) continue;
        if (asked && !asked->empty())  // (empty: all that there are)
        {
            const auto info = asked->find(next.get());
            if (info == asked->end() || !info->second.should_execute()) continue;
        }
        const auto stream = next->stream();
        TORCH_CHECK(!stream.has_value() || captured(*stream), what, ": an eager graph of a tensor that is differentiated in this captured call still lives (on another stream): ",
                    "drop it before the capture, or detach");
        for (const auto& edge : next->next_edges()) nodes.push_back(edge.function);
    }
}
inline void check_captured_gradients(const torch::Tensor& t, const char* what)
{
    if (!t.requires_grad()) return;
    check_captured_gradients(t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t),
                             c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).unwrap(), what);
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
