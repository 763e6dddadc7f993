"""Tensors whose elements stand in memory with the other sign (the imaginary parts of a conjugate, say) count as what they are, or are refused where
memory itself is read or written from call to call."""
import pytest
import torch

from tests.test_gpu_point_weights import shim
from vet_amd import synthetic, torch_ops

pytestmark = pytest.mark.gpu


def negative(t):
    """t's values in a view that negates what lies in memory."""
    view = torch._neg_view(-t)
    assert view.is_neg() and torch.equal(view, t)
    return view


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dropout(dtype):
    x, r, dy = (torch.randn(1000, device="cuda").to(dtype) for _ in range(3))
    want = torch_ops.dropout(x, 0.3, seed=1, step=2, residual=r)
    assert torch.equal(torch_ops.dropout(negative(x), 0.3, seed=1, step=2, residual=r), want)
    assert torch.equal(torch_ops.dropout(x, 0.3, seed=1, step=2, residual=negative(r)), want)
    leaf, plain = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    y = torch_ops.dropout(torch._neg_view(-leaf), 0.3, seed=1, step=2, residual=r)
    assert torch.equal(y, want)
    (g,) = torch.autograd.grad(y, leaf, negative(dy))
    (h,) = torch.autograd.grad(torch_ops.dropout(plain, 0.3, seed=1, step=2, residual=r), plain, dy)
    assert torch.equal(g, h)
    (one,) = (torch_ops.dropout(negative(x[:1]), 0.0, seed=1),)
    assert torch.equal(one, x[:1])


def test_selection_and_rows():
    score = torch.randn(3, 500, device="cuda")
    index, count = torch_ops.select_kept(score, 40, recent=5)
    got = torch_ops.select_kept(negative(score), 40, recent=5)
    assert torch.equal(got[0], index) and torch.equal(got[1], count)
    length = torch.tensor([500, 20, 300], dtype=torch.int32, device="cuda")
    index, count = torch_ops.select_kept(score, 40, length=length)
    got = torch_ops.select_kept(score, 40, length=negative(length))
    assert torch.equal(got[0], index) and torch.equal(got[1], count)
    x = torch.randn(3, 500, 2, device="cuda")
    assert torch.equal(torch_ops.keep_rows([x], negative(index), [1])[0], torch_ops.keep_rows([x], index, [1])[0])


def test_memory_that_calls_read_or_write_in_place_is_refused():
    x, count = torch.randn(64, device="cuda"), torch.ones(1, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="negative view"):
        torch_ops.dropout(x, 0.5, seed=1, device_step=negative(count))
    scene = synthetic.tiny_scene(num_points=500)
    with pytest.raises(RuntimeError, match="point_weight"):
        shim(scene, negative(torch.ones(500, device="cuda")))
    with pytest.raises(RuntimeError, match="dropout_device_step"):
        shim(scene, None, train=True, dropout=0.25, dropout_seed=1, dropout_device_step=negative(count))
