"""A step that is counted on the device and goes on between a forward pass and its backward pass would give the gradient of another mask: it is
noticed, also where an optimiser's own kernel counts."""
import numpy as np
import pytest
import torch

from tests import entries_model as em
from tests.test_gpu_point_dropout import leaves, shim
from vet_amd import synthetic, torch_ops

pytestmark = pytest.mark.gpu


def optimiser():
    """One whose count says nothing about the tensors that are differentiated."""
    other = torch.zeros(8, device="cuda", requires_grad=True)
    other.grad = torch.ones_like(other)
    return torch_ops.AdamW([([other], 0.1)], capturable=True)


def test_a_step_of_the_optimiser_is_noticed():
    opt = optimiser()
    x = torch.randn(3000, device="cuda", requires_grad=True)
    y = torch_ops.dropout(x, 0.3, seed=2, device_step=opt.device_step)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    # as it is meant to be used: the step behind the backward pass
    for k in range(1, 4):
        x.grad = None
        torch_ops.dropout(x, 0.3, seed=2, device_step=opt.device_step).sum().backward()
        opt.step()
        factor, _ = em.dropout(np.ones(3000), 0.3, 2, k)
        assert np.abs(x.grad.cpu().numpy() - factor).max() <= 2.0 ** -23 * 2


def test_a_step_of_the_optimiser_is_noticed_by_a_render():
    opt = optimiser()
    scene = synthetic.tiny_scene(num_points=500)
    inputs = leaves(scene)
    outs = shim(scene, inputs, dropout=0.25, dropout_seed=1, dropout_device_step=opt.device_step)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        sum(o.sum() for o in outs).backward()


def test_the_rates_factor_is_no_count():
    """It lies beside the count, and says nothing about masks."""
    opt = optimiser()
    x = torch.randn(3000, device="cuda", requires_grad=True)
    y = torch_ops.dropout(x, 0.3, seed=2, device_step=opt.device_step)
    opt.lr_factor.fill_(0.5)
    y.sum().backward()
    factor, _ = em.dropout(np.ones(3000), 0.3, 2, 0)
    assert np.abs(x.grad.cpu().numpy() - factor).max() <= 2.0 ** -23 * 2
    y = torch_ops.dropout(x, 0.3, seed=2, device_step=opt.device_step)
    opt.set_step(7)
    assert opt.steps() == [7] and opt.lr_factor.item() == 0.5
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        assert optimiser().steps() == [0]
