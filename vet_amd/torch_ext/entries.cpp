// See entries.h.
#include "entries.h"

#include <cstring>
#include <unordered_set>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "calls.h"

namespace vet_amd
{
namespace
{
// The tensor's elements in the order of memory that `like` has.
torch::Tensor in_order_of(const torch::Tensor& t, at::IntArrayRef strides)
{
    if (t.strides() == strides) return t;
    return torch::empty_strided(t.sizes(), strides, t.options()).copy_(t);
}

torch::Tensor dropout_call(const torch::Tensor& x, const torch::Tensor& residual, const torch::Tensor& device_step, double p, uint64_t seed, uint64_t step)
{
    c10::DeviceGuard guard(x.device());
    torch::NoGradGuard no_grad;
    const torch::Tensor in = dense(x) ? x : x.contiguous();
    torch::Tensor y        = torch::empty_strided(in.sizes(), in.strides(), in.options());
    if (y.numel() == 0) return y;
    torch::Tensor added;
    vetrast_dropout_args a;
    std::memset(&a, 0, sizeof(a));
    if (residual.defined())
    {
        added      = in_order_of(residual, in.strides());
        a.residual = added.data_ptr();
    }
    a.x    = in.data_ptr();
    a.y    = y.data_ptr();
    a.n    = in.numel();
    a.type = type_of(in, "dropout: x");
    a.p    = p;
    a.seed = seed;
    a.step = step;
    if (device_step.defined()) a.device_step = device_step.data_ptr<int64_t>();
    check(vetrast_dropout(context_on(x.device()), &a, stream_on(x.device())), "dropout");
    return y;
}

// A backward pass ends with a wait for the streams of the nodes that it came to. In a capture each of them has to be the one that is
// captured: torch otherwise records an event on a stream outside the capture, and the process ends when the capture does. A leaf's node
// lives as long as any graph of that leaf, so one of an eager pass that still lives is what a captured pass would come to. What leads to
// `t` is looked at here, where an error can still be given.
void check_captured_gradients(const torch::Tensor& t, const char* what)
{
    if (!t.defined() || !t.requires_grad()) return;
    const c10::Stream here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).unwrap();
    std::vector<std::shared_ptr<torch::autograd::Node>> nodes{t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t)};
    std::unordered_set<torch::autograd::Node*> seen;
    while (!nodes.empty())
    {
        const auto node = std::move(nodes.back());
        nodes.pop_back();
        if (!node || !seen.insert(node.get()).second) continue;
        const auto stream = node->stream();
        TORCH_CHECK(!stream.has_value() || *stream == here, what, ": an eager graph of a tensor that is differentiated in this captured call still lives (on another stream): ",
                    "drop it before the capture, or detach");
        for (const auto& edge : node->next_edges()) nodes.push_back(edge.function);
    }
}

struct DropoutFunction : public torch::autograd::Function<DropoutFunction>
{
    using Maybe = std::optional<torch::Tensor>;
    static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x, const Maybe& residual, const Maybe& device_step, double p,
                                 int64_t seed, int64_t step)
    {
        const torch::Tensor counted    = device_step.value_or(torch::Tensor());
        torch::Tensor y                = dropout_call(x, residual.value_or(torch::Tensor()), counted, p, (uint64_t)seed, (uint64_t)step);
        ctx->saved_data["residual"]    = residual.has_value();
        ctx->saved_data["p"]           = p;
        ctx->saved_data["seed"]        = seed;
        ctx->saved_data["step"]        = step;
        ctx->saved_data["strides"]     = y.strides().vec();
        ctx->save_for_backward({counted});  // noticed there if somebody has written it meanwhile
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list gradients)
    {
        const torch::Tensor& dy = gradients[0];
        torch::autograd::variable_list r(6);
        if (!dy.defined()) return r;
        if (ctx->needs_input_grad(0))
        {
            const torch::Tensor counted = ctx->get_saved_variables()[0];
            const auto strides          = ctx->saved_data["strides"].toIntVector();
            // (the differentiable call, so that the gradient has one itself)
            r[0] = Dropout(in_order_of(dy, strides), ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                           (uint64_t)ctx->saved_data["step"].toInt(), std::nullopt, counted.defined() ? Maybe(counted) : std::nullopt);
        }
        if (ctx->saved_data["residual"].toBool()) r[1] = dy;
        return r;
    }
};
}  // namespace

torch::Tensor Dropout(const torch::Tensor& x, double p, uint64_t seed, uint64_t step, const std::optional<torch::Tensor>& residual,
                      const std::optional<torch::Tensor>& device_step)
{
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout: p lies in [0, 1], not ", p);
    TORCH_CHECK(x.defined() && x.is_cuda() && x.layout() == torch::kStrided, "dropout: x must be a strided tensor on the GPU");
    type_of(x, "dropout: x");
    torch::Tensor added, counted;
    if (residual.has_value() && residual->defined())
    {
        added = *residual;
        check_on(added, x.device(), "dropout: residual");
        TORCH_CHECK(added.scalar_type() == x.scalar_type() && added.sizes() == x.sizes(), "dropout: the residual must have the type and shape of x");
    }
    if (device_step.has_value() && device_step->defined())
    {
        counted = *device_step;
        check_on(counted, x.device(), "dropout: device_step");
        TORCH_CHECK(counted.scalar_type() == torch::kInt64 && counted.numel() == 1, "dropout: device_step is one int64");
    }
    if (torch::GradMode::is_enabled() && (x.requires_grad() || (added.defined() && added.requires_grad())))
    {
        if (capturing())
        {
            check_captured_gradients(x, "dropout");
            check_captured_gradients(added, "dropout");
        }
        const auto maybe = [](const torch::Tensor& t) { return t.defined() ? std::optional(t) : std::nullopt; };
        return DropoutFunction::apply(x, maybe(added), maybe(counted), p, (int64_t)seed, (int64_t)step);
    }
    return dropout_call(x, added, counted, p, seed, step);
}
}  // namespace vet_amd
