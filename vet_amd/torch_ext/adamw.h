// AdamW over lists of tensors for libtorch callers: everything a training step has gradients for, stepped together. All arithmetic
// happens behind vetrast_adamw_step, vetrast_gradient_norm and vetrast_pack_moments / vetrast_unpack_moments (include/vetrast.h).
#pragma once
#include <torch/torch.h>

#include <optional>
#include <tuple>
#include <vector>

#include "../../include/vetrast.h"

namespace vet_amd
{
// The reference steps its texture with MyAdam (src/lib/models/my_adam.cpp) and its network with torch::optim::Adam, a dozen
// elementwise launches a tensor; this class takes both kinds of tensors, in one launch for up to 160 of them.
// An object serves one host thread and one stream at a time.
class AdamW
{
   public:
    struct Group
    {
        std::vector<torch::Tensor> params;
        double lr           = 1e-3;
        double weight_decay = 0.0;
    };
    struct Options
    {
        double beta1 = 0.9, beta2 = 0.999, eps = 1e-8;
        int moment_bits          = 32;     // 8: codes with two scale bytes for every 128 elements
        bool master_weights      = false;  // 16-bit parameters have float32 masters here, which are what the step updates
        bool stochastic_rounding = false;  // bf16 parameters without masters are rounded by random bits
        uint64_t seed            = 0;      // of the random bits, also those that round 8-bit moments
        bool capturable          = false;  // the step count lies on the device, steps may be captured in a graph
    };
    // Parameters: dense tensors on one GPU (any order of dimensions), float32, bfloat16 or float16, no two of which share memory;
    // their gradients are found in .grad() at every step (these may share memory only while steps do not clear them). Masters are read from the parameters here, moments are zero.
    AdamW(std::vector<Group> groups, Options options);

    // One step on every parameter that has a gradient. grad_scale: float32 on the GPU, one element or the two that GradNorm
    // returns (the last counts); where it is not finite, parameters, moments and the device's step count stay as they are (a count
    // on the host goes up all the same: it does not see the device).
    // A parameter whose number of elements has changed starts anew, as MyAdam does. The state of one that has changed its order in memory
    // follows it: an element keeps its index. 8-bit moments are rounded to nearest once more by that.
    // Parameters of one group that have different counts are several groups to the kernels: VETRAST_ADAMW_MAX_GROUPS in all.
    void step(bool zero_grad = false, const std::optional<torch::Tensor>& grad_scale = std::nullopt);
    void zero_grad();
    // GradNorm of the parameters' gradients.
    torch::Tensor grad_norm(double max_norm = 0.0, double scale = 1.0);

    void set_lr(int64_t group, double lr);
    // Steps done by every parameter; with capturable, all have the device's count (this waits for the device).
    std::vector<int64_t> steps() const;
    // One count for all, or one a parameter as steps() gives them: those that began later have smaller ones.
    void set_step(int64_t step);
    void set_step(const std::vector<int64_t>& steps);
    // First element and number of elements of every parameter in the flat state tensors.
    std::vector<std::pair<int64_t, int64_t>> layout() const;
    // Both moments as flat float32 tensors laid out like the state (the state itself where it is float32), in the order of memory that
    // the parameters have now.
    std::tuple<torch::Tensor, torch::Tensor> moments();
    // Takes over float32 moments, two tensors a parameter, from a run with either kind of state: of the parameter's shape, or flat in
    // the order of its memory. Counts as for set_step.
    void load_moments(const std::vector<torch::Tensor>& exp_avgs, const std::vector<torch::Tensor>& exp_avg_sqs, int64_t step);
    void load_moments(const std::vector<torch::Tensor>& exp_avgs, const std::vector<torch::Tensor>& exp_avg_sqs, const std::vector<int64_t>& steps);
    // Parameters shrink to the entries `index` (int32 [K], as SelectKept gives them; one below 0 or beyond the end leaves zeros) along dims[k], and
    // their moments and masters with them: a scene that loses points trains on. Their gradients are dropped, counts stay, and the other parameters
    // keep their state. params: contiguous parameters of this optimiser. 8-bit moments are rounded to nearest once more. Not with capturable, whose captured
    // steps would go on with what was there. Graphs of these parameters from before can no longer be differentiated. Nothing changes if it throws.
    void keep_rows(const std::vector<torch::Tensor>& params, const torch::Tensor& index, const std::vector<int64_t>& dims);
    // Masters are read from the parameters again (after a checkpoint was loaded into these).
    void reload_master();

    // The state, flat: every parameter starts at a multiple of VETRAST_MOMENT_BLOCK elements, and has its own in the order of memory that
    // it had at the last call of step, moments, load_moments or reload_master. exp_avg and exp_avg_sq are float32,
    // or uint8 codes with block_scale uint8 [blocks, 2]; master is float32 or undefined. They are other tensors after a step or
    // load_moments that found a parameter of another size.
    torch::Tensor exp_avg, exp_avg_sq, block_scale, master;
    // With capturable: steps done (int64 [1]) and a factor on every group's learning rate (float32 [1]); both may be written.
    torch::Tensor device_step, lr_factor;

   private:
    struct Slot
    {
        torch::Tensor param;
        int group     = 0;
        int32_t type  = 0;
        int64_t first = 0, n = -1, step = 0;
        std::vector<int64_t> sizes, strides;  // of the parameter when its state was put in order
        bool rows = true;                     // it was contiguous
    };
    void lay_out();
    static void take_order(Slot& s);
    void reorder(Slot& s);
    void follow_orders();
    void follow_parameters();
    void use_on_stream();
    void check_state() const;
    void check_counts(const std::vector<int64_t>& steps) const;
    static void fill_master(const Slot& s, torch::Tensor& to);
    std::vector<Slot> slots_;
    std::vector<double> lr_, weight_decay_;
    Options options_;
    torch::Device device_ = torch::kCPU;
    torch::Tensor device_state_;
    std::optional<c10::Stream> stream_;  // that the arrays are known to be used on
    int64_t elements_ = 0;  // of the flat state
    std::vector<vetrast_adamw_tensor> tensors_;  // of the call under way
    std::vector<vetrast_adamw_group> groups_;
    std::vector<int64_t> group_of_;
};

// Lists of tensors that somebody else holds (a Python list of a hundred is half of a call's time when it is copied).
using TensorPointers = std::vector<const torch::Tensor*>;

// vetrast_gradient_norm over tensors on one GPU (undefined ones are left out): float32 [2], the norm of `scale` times the gradients and
// the factor that brings it to at most max_norm (<= 0: `scale`).
torch::Tensor GradNorm(const TensorPointers& gradients, double max_norm = 0.0, double scale = 1.0);

// Moments of a list of tensors as codes and scales, in flat tensors laid out as AdamW keeps them, and such flat tensors back as float32.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> PackMoments(const TensorPointers& exp_avgs, const TensorPointers& exp_avg_sqs);
std::tuple<torch::Tensor, torch::Tensor> UnpackMoments(const torch::Tensor& exp_avg, const torch::Tensor& exp_avg_sq, const torch::Tensor& block_scale);
}  // namespace vet_amd
