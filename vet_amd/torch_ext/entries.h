// Operators that leave entries out, for libtorch callers: at random for one step (dropout without a stored mask). All arithmetic happens
// behind vetrast_dropout (include/vetrast.h).
#pragma once
#include <torch/torch.h>

#include <optional>

#include "../../include/vetrast.h"

namespace vet_amd
{
// x with a share p of its elements left out and the others scaled by 1 / (1 - p), p rounded to a multiple of 2^-16; plus a residual of x's
// shape and type. Differentiable (any number of times) in both. float32, bfloat16 or float16 on the GPU, any order of dimensions: the mask
// is a function of seed, step and an element's place in memory (a tensor with gaps is made contiguous first), and nothing is kept for the
// backward pass. Give every layer a seed of its own and count steps.
// device_step: int64 [1] on the GPU, added to `step` (AdamW::device_step, say), for steps that are captured in a graph. The backward
// pass reads it again: it must not be written between the two.
torch::Tensor Dropout(const torch::Tensor& x, double p, uint64_t seed, uint64_t step = 0, const std::optional<torch::Tensor>& residual = std::nullopt,
                      const std::optional<torch::Tensor>& device_step = std::nullopt);
}  // namespace vet_amd
