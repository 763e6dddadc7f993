// See entries.h.
#include "entries.h"

#include <cstring>
#include <limits>

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

// (A view that negates what lies in memory is made a tensor of its own here and below; kernels read memory.)
torch::Tensor Dropout(const torch::Tensor& given, double p, uint64_t seed, uint64_t step, const std::optional<torch::Tensor>& residual,
                      const std::optional<torch::Tensor>& device_step)
{
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout: p lies in [0, 1], not ", p);
    TORCH_CHECK(given.defined() && given.is_cuda() && given.layout() == torch::kStrided, "dropout: x must be a strided tensor on the GPU");
    const torch::Tensor x = given.resolve_neg();
    type_of(x, "dropout: x");
    torch::Tensor added, counted;
    if (residual.has_value() && residual->defined())
    {
        added = *residual;
        check_on(added, x.device(), "dropout: residual");
        TORCH_CHECK(added.scalar_type() == x.scalar_type() && added.sizes() == x.sizes(), "dropout: the residual must have the type and shape of x");
        added = added.resolve_neg();
    }
    if (device_step.has_value() && device_step->defined())
    {
        counted = *device_step;
        check_on(counted, x.device(), "dropout: device_step");
        TORCH_CHECK(counted.scalar_type() == torch::kInt64 && counted.numel() == 1, "dropout: device_step is one int64");
        TORCH_CHECK(!counted.is_neg(), "dropout: device_step is read where it lies and cannot be a negative view");
    }
    if (torch::GradMode::is_enabled() && (x.requires_grad() || (added.defined() && added.requires_grad())))
    {
        if (capturing())
        {
            check_captured_gradients(x, "dropout");
            if (added.defined()) check_captured_gradients(added, "dropout");
        }
        const auto maybe = [](const torch::Tensor& t) { return t.defined() ? std::optional(t) : std::nullopt; };
        return DropoutFunction::apply(x, maybe(added), maybe(counted), p, (int64_t)seed, (int64_t)step);
    }
    return dropout_call(x, added, counted, p, seed, step);
}

std::tuple<torch::Tensor, torch::Tensor> SelectKept(const torch::Tensor& given, int64_t budget, int64_t recent, const std::optional<torch::Tensor>& length)
{
    constexpr int64_t kMost = (int64_t)1 << 30, kRows = std::numeric_limits<int32_t>::max();
    TORCH_CHECK(budget >= 0 && budget <= kMost, "select_kept: a budget lies in [0, 2^30], not at ", budget);
    TORCH_CHECK(recent >= 0 && recent <= budget, "select_kept: recent lies in [0, budget], not at ", recent);
    TORCH_CHECK(given.defined() && given.is_cuda() && given.layout() == torch::kStrided && given.scalar_type() == torch::kFloat32,
                "select_kept: score must be a float32 tensor on the GPU");
    TORCH_CHECK(given.dim() == 1 || given.dim() == 2, "select_kept: score is [N] or [rows, N]");
    TORCH_CHECK(given.size(-1) <= kMost && (given.dim() == 1 || given.size(0) <= kRows), "select_kept: a row has at most 2^30 scores, and rows are counted in 32 bits");
    c10::DeviceGuard guard(given.device());
    torch::NoGradGuard no_grad;
    const torch::Tensor score = given.resolve_neg();
    const bool one      = score.dim() == 1;
    const int64_t rows  = one ? 1 : score.size(0), n = score.size(-1);
    // rows may lie further apart, their scores not, and they must not be one row seen many times
    torch::Tensor in = n > 1 && (score.stride(-1) != 1 || (!one && rows > 1 && score.stride(0) < n)) ? score.contiguous() : score;
    if (n == 1 && !one && rows > 1 && in.stride(0) < 1) in = in.contiguous();
    const auto ints     = score.options().dtype(torch::kInt32).requires_grad(false);
    torch::Tensor index = one ? torch::empty({budget}, ints) : torch::empty({rows, budget}, ints), count = torch::empty({rows}, ints);
    torch::Tensor lengths;
    if (length.has_value() && length->defined())
    {
        check_on(*length, score.device(), "select_kept: length");
        TORCH_CHECK(length->scalar_type() == torch::kInt32 && length->numel() == rows, "select_kept: length is int32, one for each row");
        lengths = length->resolve_neg().contiguous();
    }
    const size_t bytes      = vetrast_select_kept_workspace_bytes((int32_t)rows, (int32_t)n);
    torch::Tensor workspace = torch::empty({(int64_t)bytes}, ints.dtype(torch::kUInt8));
    vetrast_select_args a;
    std::memset(&a, 0, sizeof(a));
    a.score           = in.data_ptr<float>();
    a.row_stride      = one || rows <= 1 || n == 0 ? n : in.stride(0);
    a.length          = lengths.defined() ? lengths.data_ptr<int32_t>() : nullptr;
    a.index           = index.data_ptr<int32_t>();
    a.count           = count.data_ptr<int32_t>();
    a.rows            = (int32_t)rows;
    a.n               = (int32_t)n;
    a.budget          = (int32_t)budget;
    a.recent          = (int32_t)recent;
    a.workspace       = bytes ? workspace.data_ptr() : nullptr;
    a.workspace_bytes = bytes;
    check(vetrast_select_kept(context_on(score.device()), &a, stream_on(score.device())), "select_kept");
    return {index, count};
}

namespace
{
// A tensor's entries along `dim` as vetrast_keep_tensor has them, without a copy: what lies behind the dimension contiguous, what lies
// in front of it evenly apart.
bool rows_of(const torch::Tensor& t, int64_t dim, int64_t each, vetrast_keep_tensor& k)
{
    int64_t inner = 1;
    for (int64_t d = t.dim() - 1; d > dim; --d)
    {
        if (t.size(d) != 1 && t.stride(d) != inner) return false;
        inner *= t.size(d);
    }
    int64_t outers = 1, apart = 0;
    for (int64_t d = dim - 1; d >= 0; --d)
    {
        if (t.size(d) == 1) continue;
        if (outers == 1) apart = t.stride(d);
        else if (t.stride(d) != apart * outers) return false;
        outers *= t.size(d);
    }
    k.src             = t.data_ptr();
    k.outers          = outers;
    k.n               = t.size(dim);
    k.row_bytes       = inner * each;
    k.src_outer_bytes = apart * each;
    k.src_row_bytes   = t.size(dim) > 1 ? t.stride(dim) * each : k.row_bytes;
    return true;
}
}  // namespace

std::vector<torch::Tensor> KeepRows(const std::vector<torch::Tensor>& tensors, const torch::Tensor& index, const std::vector<int64_t>& dims)
{
    TORCH_CHECK(index.defined() && index.is_cuda() && index.layout() == torch::kStrided && index.scalar_type() == torch::kInt32 && (index.dim() == 1 || index.dim() == 2),
                "keep_rows: index must be an int32 tensor [K] or [rows, K] on the GPU");
    TORCH_CHECK(tensors.size() == dims.size(), "keep_rows: ", tensors.size(), " tensors, but dimensions of ", dims.size());
    const torch::Device device = index.device();
    c10::DeviceGuard guard(device);
    torch::NoGradGuard no_grad;
    const bool one           = index.dim() == 1;
    const int64_t kept       = index.size(-1), rows = one ? 1 : index.size(0);
    constexpr int64_t kMost  = std::numeric_limits<int32_t>::max();
    TORCH_CHECK(kept <= kMost && rows <= kMost && (int64_t)tensors.size() <= kMost, "keep_rows: indices, their rows and tensors are counted in 32 bits");
    const bool apart         = (kept <= 1 || index.stride(-1) == 1) && (one || rows <= 1 || index.stride(0) >= kept);
    const torch::Tensor at   = apart ? index.resolve_neg() : index.contiguous();
    std::vector<torch::Tensor> out, gathered;
    std::vector<vetrast_keep_tensor> list;
    for (size_t k = 0; k < tensors.size(); ++k)
    {
        const torch::Tensor& t = tensors[k];
        TORCH_CHECK(t.defined(), "keep_rows: tensor ", k, " is undefined");
        check_on(t, device, "keep_rows: tensors");
        TORCH_CHECK(!t.is_conj() && !t.is_neg(), "keep_rows: a tensor that is a conjugate or negative view must be made one of its own first");
        const int64_t dim = dims[k] < 0 ? dims[k] + t.dim() : dims[k];
        TORCH_CHECK(dim >= (one ? 0 : 1) && dim < t.dim(), "keep_rows: tensor ", k, " has no entries along dimension ", dims[k],
                    one ? "" : " (the first is that of the rows of indices)");
        TORCH_CHECK(one || t.size(0) == rows, "keep_rows: tensor ", k, " has ", one ? 0 : t.size(0), " rows, the indices have ", rows);
        auto sizes = t.sizes().vec();
        sizes[dim] = kept;
        out.push_back(torch::empty(sizes, t.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous)));
        if (out.back().numel() == 0) continue;
        vetrast_keep_tensor e;
        if (!rows_of(t, dim, (int64_t)t.element_size(), e))
        {
            gathered.push_back(t.contiguous());
            rows_of(gathered.back(), dim, (int64_t)t.element_size(), e);
        }
        e.dst = out.back().data_ptr();
        list.push_back(e);
    }
    if (list.empty()) return out;
    vetrast_keep_args a;
    std::memset(&a, 0, sizeof(a));
    a.tensors          = list.data();
    a.num_tensors      = (int32_t)list.size();
    a.index_rows       = (int32_t)rows;
    a.kept             = (int32_t)kept;
    a.index_row_stride = one || rows <= 1 ? kept : at.stride(0);
    a.index            = at.data_ptr<int32_t>();
    check(vetrast_keep_rows(context_on(device), &a, stream_on(device)), "keep_rows");
    return out;
}
}  // namespace vet_amd
