// See adamw.h.
#include "adamw.h"

#include <cstring>
#include <limits>
#include <map>
#include <utility>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

namespace vet_amd
{
namespace
{
constexpr int64_t kBlock = VETRAST_MOMENT_BLOCK;

void check(int st, const char* where)
{
    TORCH_CHECK(st == VETRAST_OK, "vetrast ", where, " failed: ", st, " (", vetrast_status_string(st), ")");
}

void* stream_on(const torch::Device& device)
{
    return (void*)c10::hip::getCurrentHIPStream(device.index()).stream();
}

bool capturing()
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
Kept& kept()
{
    thread_local Kept k;
    return k;
}

// The caller has made `device` the current one.
vetrast_ctx* context_on(const torch::Device& device)
{
    vetrast_ctx*& ctx = kept().contexts[device.index()];
    if (!ctx) check(vetrast_create(&ctx), "create");
    return ctx;
}

// Zeroed memory for vetrast_gradient_norm, which leaves it zeroed where that counts. A captured call has its own, cleared in the graph, and
// so has one on a stream that is not of torch's pool (its id is its handle): such a stream may be destroyed while its norm still runs,
// and another that gets its handle would count in the same memory.
torch::Tensor norm_workspace(const torch::Device& device, size_t bytes)
{
    const auto options = torch::TensorOptions(device).dtype(torch::kUInt8);
    const auto stream  = c10::hip::getCurrentHIPStream(device.index());
    void* handle       = (void*)stream.stream();
    const bool foreign = handle != nullptr && (intptr_t)stream.id() == reinterpret_cast<intptr_t>(handle);
    if (foreign || capturing()) return torch::zeros({(int64_t)bytes}, options);
    torch::Tensor& w = kept().workspaces[{device.index(), handle}];
    if (!w.defined() || w.numel() < (int64_t)bytes) w = torch::zeros({(int64_t)bytes}, options);
    return w;
}

int32_t type_of(const torch::Tensor& t, const char* what)
{
    switch (t.scalar_type())
    {
        case torch::kFloat32: return VETRAST_F32;
        case torch::kBFloat16: return VETRAST_BF16;
        case torch::kFloat16: return VETRAST_F16;
        default: TORCH_CHECK(false, what, " must be float32, bfloat16 or float16, not ", t.scalar_type());
    }
}

void check_on(const torch::Tensor& t, const torch::Device& device, const char* what)
{
    TORCH_CHECK(t.layout() == torch::kStrided && t.device() == device, what, " must be a strided tensor on ", device);
}

// The elements one behind the other in memory, whatever the order of dimensions.
bool dense(const torch::Tensor& t)
{
    return t.is_contiguous() || t.is_non_overlapping_and_dense();
}

int64_t whole_blocks(int64_t n)
{
    return (n + kBlock - 1) / kBlock * kBlock;
}

bool same_order(const torch::Tensor& a, const torch::Tensor& b)
{
    return (a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides();
}

// Whether two orders of memory are one: strides of dimensions of one element say nothing.
bool same_memory(at::IntArrayRef sizes, at::IntArrayRef a, at::IntArrayRef b)
{
    for (size_t d = 0; d < sizes.size(); ++d)
        if (sizes[d] != 1 && a[d] != b[d]) return false;
    return true;
}

// Moments of a list of tensors, placed one behind the other in flat arrays; `total`: elements of these.
std::vector<vetrast_moment_tensor> moment_list(const TensorPointers& ms, const TensorPointers& vs, const torch::Device& device, int64_t& total)
{
    TORCH_CHECK(ms.size() == vs.size(), "as many first moments as second ones are needed, not ", ms.size(), " and ", vs.size());
    std::vector<vetrast_moment_tensor> list(ms.size());
    total = 0;
    for (size_t k = 0; k < ms.size(); ++k)
    {
        const torch::Tensor &m = *ms[k], &v = *vs[k];
        check_on(m, device, "moments");
        check_on(v, device, "moments");
        TORCH_CHECK(m.scalar_type() == torch::kFloat32 && v.scalar_type() == torch::kFloat32 && dense(m) && dense(v), "moments must be dense float32 tensors");
        TORCH_CHECK(m.sizes() == v.sizes() && same_order(m, v), "both moments of a tensor must have one shape and order");
        list[k] = {m.data_ptr<float>(), v.data_ptr<float>(), m.numel(), total};
        total += whole_blocks(list[k].n);
    }
    return list;
}

TensorPointers pointers(const std::vector<torch::Tensor>& list)
{
    TensorPointers r;
    for (auto& t : list) r.push_back(&t);
    return r;
}

vetrast_moments_args moments_args(const std::vector<vetrast_moment_tensor>& list, const torch::Tensor& m, const torch::Tensor& v, const torch::Tensor& scale)
{
    return {list.data(), (int32_t)list.size(), 0, m.data_ptr<uint8_t>(), v.data_ptr<uint8_t>(), scale.data_ptr<uint8_t>()};
}
}  // namespace

AdamW::AdamW(std::vector<Group> groups, Options options) : options_(options)
{
    TORCH_CHECK(options.moment_bits == 32 || options.moment_bits == 8, "AdamW: moment_bits is 32 or 8, not ", options.moment_bits);
    TORCH_CHECK(options.beta1 >= 0 && options.beta1 < 1 && options.beta2 >= 0 && options.beta2 < 1, "AdamW: betas lie in [0, 1)");
    // as vetrast_adamw_step has it
    TORCH_CHECK((float)options.eps >= std::numeric_limits<float>::min() && (float)options.eps <= std::numeric_limits<float>::max(),
                "AdamW: eps must be a finite float32 of at least 2^-126, not ", options.eps);
    TORCH_CHECK(groups.size() <= VETRAST_ADAMW_MAX_GROUPS, "AdamW: at most ", VETRAST_ADAMW_MAX_GROUPS, " groups");
    for (auto& g : groups)
    {
        for (auto& p : g.params)
        {
            TORCH_CHECK(p.defined() && p.is_cuda(), "AdamW: parameters must be tensors on the GPU");
            if (slots_.empty()) device_ = p.device();
            for (auto& s : slots_) TORCH_CHECK(!s.param.is_same(p), "AdamW: a parameter is in the list twice");
            Slot s;
            s.param = p;
            s.group = (int)lr_.size();
            s.type  = type_of(p, "AdamW: parameters");
            slots_.push_back(std::move(s));
        }
        lr_.push_back(g.lr);
        weight_decay_.push_back(g.weight_decay);
    }
    TORCH_CHECK(!slots_.empty(), "AdamW: no parameters");
    c10::DeviceGuard guard(device_);
    context_on(device_);  // here and not in a step that may be captured
    lay_out();
    if (options_.capturable)
    {
        const int64_t bytes = (int64_t)vetrast_adamw_device_state_bytes((int32_t)lr_.size());
        device_state_       = torch::zeros({bytes}, torch::TensorOptions(device_).dtype(torch::kUInt8));
        device_step         = device_state_.narrow(0, 0, 8).view(torch::kInt64);
        lr_factor           = device_state_.narrow(0, 8, 4).view(torch::kFloat32);
        lr_factor.fill_(1.0);
    }
}

void AdamW::fill_master(const Slot& s, torch::Tensor& to)
{
    // in the parameter's order of memory
    to.narrow(0, s.first, s.n).copy_(s.param.detach().as_strided({s.n}, {1}));
}

// Room in the flat state for every parameter as it is now. What a parameter of unchanged size had moves along. Nothing of the object
// changes before everything that may throw is done (a parameter that is refused, memory that runs out while both states are there):
// places and lengths are what the kernels go by, and always those of the arrays that are there.
void AdamW::lay_out()
{
    torch::NoGradGuard no_grad;
    std::vector<Slot> slots = slots_;
    std::vector<int64_t> from(slots.size(), -1);
    int64_t at = 0;
    for (size_t k = 0; k < slots.size(); ++k)
    {
        Slot& s = slots[k];
        check_on(s.param, device_, "AdamW: parameters");
        TORCH_CHECK(dense(s.param), "AdamW: parameters must be dense, without gaps or overlaps");
        if (s.n == s.param.numel()) from[k] = s.first;
        else
        {
            s.step = 0;
            take_order(s);
        }
        s.n     = s.param.numel();
        s.first = at;
        at += whole_blocks(s.n);
    }
    const auto bytes  = torch::TensorOptions(device_).dtype(torch::kUInt8);
    const auto floats = torch::TensorOptions(device_).dtype(torch::kFloat32);
    const bool eight  = options_.moment_bits == 8;
    torch::Tensor m   = torch::zeros({at}, eight ? bytes : floats);
    torch::Tensor v   = torch::zeros({at}, eight ? bytes : floats);
    torch::Tensor scales, masters;
    if (eight) scales = torch::zeros({at / kBlock, 2}, bytes);
    if (options_.master_weights) masters = torch::zeros({at}, floats);
    for (size_t k = 0; k < slots.size(); ++k)
    {
        const Slot& s   = slots[k];
        const int64_t n = whole_blocks(s.n);
        if (from[k] >= 0 && n > 0)
        {
            m.narrow(0, s.first, n).copy_(exp_avg.narrow(0, from[k], n));
            v.narrow(0, s.first, n).copy_(exp_avg_sq.narrow(0, from[k], n));
            if (eight) scales.narrow(0, s.first / kBlock, n / kBlock).copy_(block_scale.narrow(0, from[k] / kBlock, n / kBlock));
            if (masters.defined()) masters.narrow(0, s.first, n).copy_(master.narrow(0, from[k], n));
        }
        else if (masters.defined()) fill_master(s, masters);
    }
    slots_.swap(slots);
    exp_avg     = std::move(m);
    exp_avg_sq  = std::move(v);
    block_scale = std::move(scales);
    master      = std::move(masters);
    elements_   = at;
}

// The arrays were allocated on one stream, and a caller may go on with another, after a wait for the first. When they are freed, here or
// with the object, their memory must not be given out before what that other stream does with it has ended.
void AdamW::use_on_stream()
{
    if (capturing()) return;  // a graph's memory is its owner's to keep
    const c10::Stream stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device_.index()).unwrap();
    if (stream_ == stream) return;
    for (torch::Tensor* t : {&exp_avg, &exp_avg_sq, &block_scale, &master, &device_state_})
        if (t->defined() && t->numel() > 0) t->record_stream(stream);
    stream_ = stream;
}

// The kernels go by the layout, not by the arrays' lengths, and the arrays are open to the caller.
void AdamW::check_state() const
{
    const auto fits = [&](const torch::Tensor& t, bool there, torch::ScalarType type, int64_t n) {
        return there ? t.defined() && t.device() == device_ && t.scalar_type() == type && t.is_contiguous() && t.numel() == n : !t.defined();
    };
    const bool eight = options_.moment_bits == 8;
    const auto type  = eight ? torch::kUInt8 : torch::kFloat32;
    TORCH_CHECK(fits(exp_avg, true, type, elements_) && fits(exp_avg_sq, true, type, elements_) && fits(block_scale, eight, torch::kUInt8, elements_ / kBlock * 2) &&
                    fits(master, options_.master_weights, torch::kFloat32, elements_),
                "AdamW: a state tensor is not the one that was laid out: copy into it, and leave its size and type as they are");
}

void AdamW::take_order(Slot& s)
{
    s.sizes   = s.param.sizes().vec();
    s.strides = s.param.strides().vec();
    s.rows    = s.param.is_contiguous();
}

// What the state of a parameter has in the order of memory that the parameter had, in the order that it has now (a network that was
// turned to channels last, say). An element keeps its index. All is made aside first, as copies in place need no memory.
void AdamW::reorder(Slot& s)
{
    const auto turned = [&](const torch::Tensor& flat) {
        torch::Tensor to = torch::empty_strided(s.sizes, s.param.strides(), flat.options());
        return to.copy_(flat.as_strided(s.sizes, s.strides)).as_strided({s.n}, {1});
    };
    const auto place     = [&](const torch::Tensor& array) { return array.narrow(0, s.first, s.n); };
    torch::Tensor masters = master.defined() ? turned(place(master)) : master;
    if (options_.moment_bits == 32)
    {
        const torch::Tensor m = turned(place(exp_avg)), v = turned(place(exp_avg_sq));
        place(exp_avg).copy_(m);
        place(exp_avg_sq).copy_(v);
    }
    else
    {
        // blocks get other elements, so codes are made anew, rounded to nearest; a lost block's elements lose the blocks that they come to
        const auto floats = torch::TensorOptions(device_).dtype(torch::kFloat32);
        torch::Tensor m = torch::empty({s.n}, floats), v = torch::empty({s.n}, floats);
        const auto convert = [&](decltype(vetrast_pack_moments)& call, const char* where) {
            const std::vector<vetrast_moment_tensor> list{{m.data_ptr<float>(), v.data_ptr<float>(), s.n, s.first}};
            const vetrast_moments_args a = moments_args(list, exp_avg, exp_avg_sq, block_scale);
            check(call(context_on(device_), &a, stream_on(device_)), where);
        };
        convert(vetrast_unpack_moments, "unpack_moments");
        m = turned(m);
        v = turned(v);
        convert(vetrast_pack_moments, "pack_moments");
    }
    if (masters.defined()) place(master).copy_(masters);
}

// The state follows a parameter of unchanged size to another order in memory.
void AdamW::follow_orders()
{
    for (auto& s : slots_)
    {
        const torch::Tensor& p = s.param;
        if (p.sizes() == s.sizes && p.strides() == s.strides) continue;
        if (p.numel() != s.n || !dense(p)) continue;  // laid out anew or refused where it is stepped
        if (!(p.is_contiguous() && s.rows) && !(p.sizes() == s.sizes && same_memory(s.sizes, p.strides(), s.strides)))
        {
            if (p.sizes() != s.sizes && !p.grad().defined()) continue;  // nothing is stepped, and with a gradient it is refused
            TORCH_CHECK(p.sizes() == s.sizes, "AdamW: a parameter has changed its shape and the order of its elements in memory, it needs an optimiser of its own");
            TORCH_CHECK(!capturing(), "AdamW: a parameter has changed its order in memory, take a step before the one that is captured");
            reorder(s);
        }
        take_order(s);
    }
}

// A new layout if a parameter has changed its size, and what it holds in the parameters' order.
void AdamW::follow_parameters()
{
    bool moved = false;
    for (auto& s : slots_) moved |= s.param.numel() != s.n;
    if (moved)
    {
        TORCH_CHECK(!options_.capturable, "AdamW: parameters cannot change their size with capturable");
        TORCH_CHECK(!capturing(), "AdamW: a parameter has changed its size, its state cannot be laid out in a captured call");  // in the graph's own memory
        lay_out();
    }
    follow_orders();
}

void AdamW::step(bool zero_grad, const std::optional<torch::Tensor>& grad_scale)
{
    torch::NoGradGuard no_grad;
    c10::DeviceGuard guard(device_);
    TORCH_CHECK(options_.capturable || !capturing(), "AdamW: a step that is captured in a graph needs capturable, which keeps the step count on the device");
    check_state();
    use_on_stream();
    follow_parameters();
    const bool eight = options_.moment_bits == 8;
    tensors_.clear();
    groups_.clear();
    if (options_.capturable)
        for (size_t g = 0; g < lr_.size(); ++g) groups_.push_back({lr_[g], weight_decay_[g], 0});
    group_of_.assign(lr_.size(), -1);
    std::vector<torch::Tensor> reordered;  // gradients that were copied into their parameter's order
    for (auto& s : slots_)
    {
        const torch::Tensor& p    = s.param;
        const torch::Tensor& grad = p.grad();
        if (!grad.defined()) continue;
        check_on(p, device_, "AdamW: parameters");
        check_on(grad, device_, "AdamW: gradients");
        const int32_t type = type_of(p, "AdamW: parameters");
        TORCH_CHECK(type == s.type, "AdamW: a parameter has changed its type");
        TORCH_CHECK(grad.scalar_type() == p.scalar_type() && grad.sizes() == p.sizes(), "AdamW: a gradient must have its parameter's type and shape");
        TORCH_CHECK(dense(p), "AdamW: parameters must be dense, without gaps or overlaps");
        void* gradient = nullptr;
        if (same_order(p, grad)) gradient = grad.data_ptr();
        else
        {
            // what clears it below is another tensor, which a replay would not read
            TORCH_CHECK(!zero_grad || dense(grad) || !capturing(), "AdamW: a gradient with gaps or overlaps cannot be cleared in a captured step");
            reordered.push_back(torch::empty_like(p).copy_(grad));
            gradient = reordered.back().data_ptr();
        }
        int64_t& place  = group_of_[s.group];
        const auto fits = [&](int64_t k) { return groups_[k].lr == lr_[s.group] && groups_[k].weight_decay == weight_decay_[s.group] && groups_[k].step == s.step + 1; };
        if (options_.capturable) place = s.group;
        else if (place < 0 || !fits(place))
        {
            // parameters of a group that started later are a group of their own here
            place = 0;
            while (place < (int64_t)groups_.size() && !fits(place)) ++place;
            if (place == (int64_t)groups_.size()) groups_.push_back({lr_[s.group], weight_decay_[s.group], s.step + 1});
        }
        tensors_.push_back({p.data_ptr(), gradient, s.n, s.first, type, type, (int32_t)place, 0});
    }
    TORCH_CHECK(groups_.size() <= VETRAST_ADAMW_MAX_GROUPS, "AdamW: ", groups_.size(), " groups, as parameters of one count, rate and decay each are one, and at most ",
                VETRAST_ADAMW_MAX_GROUPS, " are possible");
    vetrast_adamw_args a;
    std::memset(&a, 0, sizeof(a));
    a.tensors             = tensors_.data();
    a.groups              = groups_.data();
    a.num_tensors         = (int32_t)tensors_.size();
    a.num_groups          = (int32_t)groups_.size();
    a.exp_avg             = exp_avg.data_ptr();
    a.exp_avg_sq          = exp_avg_sq.data_ptr();
    a.block_scale         = eight ? block_scale.data_ptr<uint8_t>() : nullptr;
    a.master              = master.defined() ? master.data_ptr<float>() : nullptr;
    a.beta1               = options_.beta1;
    a.beta2               = options_.beta2;
    a.eps                 = options_.eps;
    a.moment_bits         = options_.moment_bits;
    a.stochastic_rounding = options_.stochastic_rounding ? 1 : 0;
    a.seed                = options_.seed;
    a.zero_grad           = zero_grad ? 1 : 0;
    a.device_state        = device_state_.defined() ? device_state_.data_ptr() : nullptr;
    if (grad_scale.has_value() && grad_scale->defined())
    {
        const torch::Tensor& x = *grad_scale;
        check_on(x, device_, "AdamW: grad_scale");
        TORCH_CHECK(x.scalar_type() == torch::kFloat32 && x.is_contiguous() && (x.numel() == 1 || x.numel() == 2),
                    "AdamW: grad_scale is one float32, or the two that grad_norm returns");
        a.grad_scale = x.data_ptr<float>() + x.numel() - 1;
    }
    check(vetrast_adamw_step(context_on(device_), &a, stream_on(device_)), "adamw_step");
    for (auto& s : slots_)
    {
        const torch::Tensor& grad = s.param.grad();
        if (!grad.defined()) continue;
        s.step += 1;
        // the kernel wrote through raw pointers: tell everyone who keys on the version counters
        if (!s.param.is_inference()) s.param.unsafeGetTensorImpl()->bump_version();
        if (!zero_grad) continue;
        if (same_order(s.param, grad))
        {
            if (!grad.is_inference()) grad.unsafeGetTensorImpl()->bump_version();
        }
        else if (dense(grad)) s.param.mutable_grad().zero_();  // the kernel cleared its copy
        else s.param.mutable_grad() = torch::zeros_like(s.param);
    }
}

void AdamW::zero_grad()
{
    torch::NoGradGuard no_grad;
    for (auto& s : slots_)
        if (s.param.grad().defined()) s.param.mutable_grad().zero_();
}

torch::Tensor AdamW::grad_norm(double max_norm, double scale)
{
    TensorPointers grads;
    grads.reserve(slots_.size());
    for (auto& s : slots_) grads.push_back(&s.param.grad());
    return GradNorm(grads, max_norm, scale);
}

void AdamW::set_lr(int64_t group, double lr)
{
    TORCH_CHECK(group >= 0 && group < (int64_t)lr_.size(), "AdamW: no group ", group);
    lr_[group] = lr;
}

std::vector<int64_t> AdamW::steps() const
{
    std::vector<int64_t> r;
    const int64_t all = options_.capturable ? device_step.item<int64_t>() : 0;
    for (auto& s : slots_) r.push_back(options_.capturable ? all : s.step);
    return r;
}

void AdamW::set_step(int64_t step)
{
    set_step(std::vector<int64_t>(slots_.size(), step));
}

void AdamW::check_counts(const std::vector<int64_t>& steps) const
{
    TORCH_CHECK(steps.size() == slots_.size(), "AdamW: ", slots_.size(), " parameters, but counts of ", steps.size());
    for (int64_t n : steps)
    {
        TORCH_CHECK(n >= 0, "AdamW: steps are counted from 0");
        TORCH_CHECK(!options_.capturable || n == steps[0], "AdamW: with capturable all parameters have one count");
    }
}

void AdamW::set_step(const std::vector<int64_t>& steps)
{
    check_counts(steps);
    if (options_.capturable)
    {
        c10::DeviceGuard guard(device_);
        use_on_stream();
        device_step.fill_(steps[0]);
    }
    for (size_t k = 0; k < slots_.size(); ++k) slots_[k].step = steps[k];
}

std::vector<std::pair<int64_t, int64_t>> AdamW::layout() const
{
    std::vector<std::pair<int64_t, int64_t>> r;
    for (auto& s : slots_) r.push_back({s.first, s.n});
    return r;
}

std::tuple<torch::Tensor, torch::Tensor> AdamW::moments()
{
    torch::NoGradGuard no_grad;
    c10::DeviceGuard guard(device_);
    check_state();
    use_on_stream();
    follow_orders();
    if (options_.moment_bits == 32) return {exp_avg, exp_avg_sq};
    return UnpackMoments(exp_avg, exp_avg_sq, block_scale);
}

void AdamW::load_moments(const std::vector<torch::Tensor>& exp_avgs, const std::vector<torch::Tensor>& exp_avg_sqs, int64_t step)
{
    load_moments(exp_avgs, exp_avg_sqs, std::vector<int64_t>(slots_.size(), step));
}

void AdamW::load_moments(const std::vector<torch::Tensor>& exp_avgs, const std::vector<torch::Tensor>& exp_avg_sqs, const std::vector<int64_t>& steps)
{
    torch::NoGradGuard no_grad;
    c10::DeviceGuard guard(device_);
    TORCH_CHECK(exp_avgs.size() == slots_.size(), "AdamW: ", slots_.size(), " parameters, but moments of ", exp_avgs.size());
    TORCH_CHECK(exp_avg_sqs.size() == slots_.size(), "AdamW: as many second moments as first ones are needed, not ", exp_avg_sqs.size());
    check_counts(steps);
    check_state();
    use_on_stream();
    follow_parameters();
    std::vector<torch::Tensor> kept[2];
    for (size_t k = 0; k < slots_.size(); ++k)
        for (int which = 0; which < 2; ++which)
        {
            const torch::Tensor &p = slots_[k].param, &x = which ? exp_avg_sqs[k] : exp_avgs[k];
            TORCH_CHECK(dense(p), "AdamW: parameters must be dense, without gaps or overlaps");
            check_on(x, device_, "AdamW: moments");
            TORCH_CHECK(x.scalar_type() == torch::kFloat32, "AdamW: moments must be float32 tensors");
            TORCH_CHECK(x.sizes() == p.sizes() || (x.dim() == 1 && x.numel() == slots_[k].n), "AdamW: parameter ", k, " and its moments differ in shape");
            if (x.sizes() == p.sizes() && !same_order(x, p)) kept[which].push_back(torch::empty_like(p, x.options()).copy_(x));
            else kept[which].push_back(dense(x) ? x : x.contiguous());
        }
    int64_t total                           = 0;
    std::vector<vetrast_moment_tensor> list = moment_list(pointers(kept[0]), pointers(kept[1]), device_, total);
    set_step(steps);
    if (options_.moment_bits == 8)
    {
        const vetrast_moments_args a = moments_args(list, exp_avg, exp_avg_sq, block_scale);
        check(vetrast_pack_moments(context_on(device_), &a, stream_on(device_)), "pack_moments");
        return;
    }
    for (size_t k = 0; k < list.size(); ++k)
    {
        exp_avg.narrow(0, slots_[k].first, slots_[k].n).copy_(kept[0][k].as_strided({slots_[k].n}, {1}));
        exp_avg_sq.narrow(0, slots_[k].first, slots_[k].n).copy_(kept[1][k].as_strided({slots_[k].n}, {1}));
    }
}

void AdamW::reload_master()
{
    torch::NoGradGuard no_grad;
    if (!options_.master_weights) return;
    c10::DeviceGuard guard(device_);
    check_state();
    use_on_stream();
    for (auto& s : slots_)
        TORCH_CHECK(s.param.numel() == s.n && dense(s.param), "AdamW: a parameter has changed its size; step() notices that by itself");
    follow_orders();
    for (auto& s : slots_) fill_master(s, master);
}

torch::Tensor GradNorm(const TensorPointers& gradients, double max_norm, double scale)
{
    std::vector<vetrast_gradient> list;
    std::vector<torch::Tensor> gathered;  // of gradients with gaps
    list.reserve(gradients.size());
    std::optional<torch::Device> device;
    c10::OptionalDeviceGuard guard;
    for (const torch::Tensor* gradient : gradients)
    {
        const torch::Tensor& g = *gradient;
        if (!g.defined()) continue;
        if (!device)
        {
            TORCH_CHECK(g.is_cuda(), "grad_norm: gradients must be tensors on the GPU");
            device = g.device();
            guard.reset_device(*device);
        }
        check_on(g, *device, "grad_norm: gradients");
        const int32_t type = type_of(g, "grad_norm: gradients");
        const void* data   = g.data_ptr();
        if (!dense(g))
        {
            gathered.push_back(g.contiguous());
            data = gathered.back().data_ptr();
        }
        list.push_back({data, g.numel(), type, 0});
    }
    TORCH_CHECK(device, "grad_norm: no gradients");
    vetrast_gradient_norm_args a;
    std::memset(&a, 0, sizeof(a));
    a.gradients             = list.data();
    a.num_gradients         = (int32_t)list.size();
    a.max_norm              = max_norm;
    a.scale                 = scale;
    a.workspace_bytes       = vetrast_gradient_norm_workspace_bytes(list.data(), a.num_gradients);
    torch::Tensor workspace = norm_workspace(*device, a.workspace_bytes);
    torch::Tensor out       = torch::empty({2}, torch::TensorOptions(*device).dtype(torch::kFloat32));
    a.workspace             = workspace.data_ptr();
    a.out                   = out.data_ptr<float>();
    check(vetrast_gradient_norm(context_on(*device), &a, stream_on(*device)), "gradient_norm");
    return out;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> PackMoments(const TensorPointers& exp_avgs, const TensorPointers& exp_avg_sqs)
{
    TORCH_CHECK(!exp_avgs.empty() && exp_avgs[0]->is_cuda(), "pack_moments: a list of tensors on the GPU is needed");
    const torch::Device device = exp_avgs[0]->device();
    c10::DeviceGuard guard(device);
    int64_t total = 0;
    const std::vector<vetrast_moment_tensor> list = moment_list(exp_avgs, exp_avg_sqs, device, total);
    const auto bytes    = torch::TensorOptions(device).dtype(torch::kUInt8);
    torch::Tensor m     = torch::empty({total}, bytes), v = torch::empty({total}, bytes);
    torch::Tensor scale = torch::empty({total / kBlock, 2}, bytes);
    const vetrast_moments_args a = moments_args(list, m, v, scale);
    check(vetrast_pack_moments(context_on(device), &a, stream_on(device)), "pack_moments");
    return {m, v, scale};
}

std::tuple<torch::Tensor, torch::Tensor> UnpackMoments(const torch::Tensor& exp_avg, const torch::Tensor& exp_avg_sq, const torch::Tensor& block_scale)
{
    TORCH_CHECK(exp_avg.is_cuda(), "unpack_moments: tensors on the GPU are needed");
    const torch::Device device = exp_avg.device();
    c10::DeviceGuard guard(device);
    for (const torch::Tensor* t : {&exp_avg, &exp_avg_sq, &block_scale})
    {
        check_on(*t, device, "unpack_moments: codes and scales");
        TORCH_CHECK(t->scalar_type() == torch::kUInt8 && t->is_contiguous(), "unpack_moments: codes and scales are contiguous uint8 tensors");
    }
    const int64_t n = exp_avg.numel();
    TORCH_CHECK(n % kBlock == 0 && exp_avg_sq.numel() == n && block_scale.numel() == n / kBlock * 2,
                "unpack_moments: whole blocks of ", kBlock, " codes with two scales each are needed");
    const auto floats = torch::TensorOptions(device).dtype(torch::kFloat32);
    torch::Tensor m = torch::empty({n}, floats), v = torch::empty({n}, floats);
    if (n == 0) return {m, v};
    const std::vector<vetrast_moment_tensor> list{{m.data_ptr<float>(), v.data_ptr<float>(), n, 0}};
    // flat arrays begin at multiples of 16 bytes; a part of one, such as the scales of one parameter, may not
    const auto placed = [](const torch::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(); };
    const torch::Tensor mc = placed(exp_avg), vc = placed(exp_avg_sq), scale = placed(block_scale);
    const vetrast_moments_args a = moments_args(list, mc, vc, scale);
    check(vetrast_unpack_moments(context_on(device), &a, stream_on(device)), "unpack_moments");
    return {m, v};
}
}  // namespace vet_amd
