"""AdamW.keep_rows gives parameters other elements: what autograd records from then on is of the new ones, whatever still lives of
the old ones."""
import pytest
import torch

from vet_amd import torch_ops

pytestmark = pytest.mark.gpu


def some(n, kept):
    """Indices of all n entries in another order, or of some of them."""
    return torch.arange(n - 1, -1, -1, device="cuda", dtype=torch.int32)[:kept]


def test_training_goes_on_while_a_graph_from_before_lives():
    torch.manual_seed(2)
    p = torch.randn(60, 4, device="cuda", requires_grad=True)
    opt = torch_ops.AdamW([([p], 0.1)])
    seen = []
    p.register_hook(lambda g: seen.append(g.shape))
    p.register_post_accumulate_grad_hook(lambda t: seen.append(t.grad.shape))
    before = (p * p).sum()
    before.backward()
    opt.step()
    opt.keep_rows([p], some(60, 41), [0])
    seen.clear()
    loss = (p * p).sum()
    loss.backward()
    assert torch.equal(p.grad, 2 * p.detach()) and seen == [(41, 4), (41, 4)]
    assert torch.isfinite(before)
    opt.step()
