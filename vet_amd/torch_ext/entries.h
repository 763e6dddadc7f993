// Operators that leave entries out, for libtorch callers: at random for one step (dropout without a stored mask), or for good, those
// that gave least (eviction). All arithmetic happens behind vetrast_dropout, vetrast_select_kept and vetrast_keep_rows
// (include/vetrast.h).
#pragma once
#include <torch/torch.h>

#include <optional>
#include <tuple>
#include <vector>

#include "../../include/vetrast.h"

namespace vet_amd
{
// x with a share p of its elements left out and the others scaled by 1 / (1 - p), p rounded to a multiple of 2^-16; plus a residual of x's
// shape and type. Differentiable (any number of times) in both. float32, bfloat16 or float16 on the GPU, any order of dimensions: the mask
// is a function of seed, step and an element's place in memory (a tensor with gaps is made contiguous first), and nothing is kept for the
// backward pass. Give every layer a seed of its own and count steps.
// device_step: int64 [1] on the GPU, added to `step` (AdamW::device_step, say), for steps that are captured in a graph. The backward
// pass reads it again: it must not be written between the two, which is noticed and refused unless a replayed graph has done it.
torch::Tensor Dropout(const torch::Tensor& x, double p, uint64_t seed, uint64_t step = 0, const std::optional<torch::Tensor>& residual = std::nullopt,
                      const std::optional<torch::Tensor>& device_step = std::nullopt);

// Which entries a budget keeps: the last `recent` of a row whatever their scores, else those with the highest scores, of equal ones
// those in front; a NaN is below everything. score: float32 [N] or [rows, N] on the GPU; length: int32 [rows], entries of a row (the others are not
// read). Gives int32 indices [budget] or [rows, budget] in ascending order with -1 behind the last one, and int32 [rows] of how many there
// are. Nothing waits for the device.
std::tuple<torch::Tensor, torch::Tensor> SelectKept(const torch::Tensor& score, int64_t budget, int64_t recent = 0,
                                                    const std::optional<torch::Tensor>& length = std::nullopt);

// The rows that go with such indices, of a list of tensors of any type: tensor k's entries along dimension dims[k]. With indices [rows, K] a tensor's
// first dimension is the rows'. An index below 0 or beyond the end leaves zeros. The results are contiguous and have no history.
std::vector<torch::Tensor> KeepRows(const std::vector<torch::Tensor>& tensors, const torch::Tensor& index, const std::vector<int64_t>& dims);
}  // namespace vet_amd
