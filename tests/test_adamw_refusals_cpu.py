"""What torch_ops.AdamW refuses before it looks at its parameters, so without a GPU."""
import pytest
import torch

from vet_amd import torch_ops


@pytest.mark.parametrize("eps", [0.0, -1e-8, 1e-60, 1e-40, 2.0 ** -127, float("inf"), 1e39, float("nan")])
def test_an_eps_that_no_step_takes_is_refused(eps):
    with pytest.raises(RuntimeError, match="eps"):
        torch_ops.AdamW([([torch.zeros(3)], 0.1)], eps=eps)


@pytest.mark.parametrize("eps", [2.0 ** -126, 1e-15, 1e-8, 1.0, 3e38])
def test_an_eps_that_steps_take_is_not(eps):
    with pytest.raises(RuntimeError, match="on the GPU"):  # the next thing that is looked at
        torch_ops.AdamW([([torch.zeros(3)], 0.1)], eps=eps)
