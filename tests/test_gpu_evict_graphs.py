"""AdamW.keep_rows gives parameters other elements: what autograd has recorded of the old ones is refused, and what it records from then on is
of the new ones, whatever still lives."""
import numpy as np
import pytest
import torch

from tests.test_gpu_torch_ext import _views
from vet_amd import synthetic, torch_ops

pytestmark = pytest.mark.gpu


def some(n, kept):
    """Indices of all n entries in another order, or of some of them."""
    return torch.arange(n - 1, -1, -1, device="cuda", dtype=torch.int32)[:kept]


def render(scene):
    """A scene's leaves and a call that renders them as they are then and sums up the pixels."""
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    texture, confidence, position = (cu(a).requires_grad_(True) for a in (scene.texture, scene.confidence.reshape(1, -1), scene.position))
    rest = [cu(scene.background), torch.zeros((scene.poses_se3.shape[0], 6), dtype=torch.float64, device="cuda"), cu(scene.intrinsics), cu(scene.poses_se3)]

    def call():
        outs = torch_ops.blend_point_cloud(texture, rest[0], position, rest[1], rest[2], confidence, rest[3], None, _views(scene), scene.num_layers, train=True,
                                           use_environment_map=0, need_point_gradient=1, drop_out_points_by_radius=0, debug_max_list_length=scene.max_list_length)
        return sum(o.sum() for o in outs)

    return texture, confidence, position, call


@pytest.mark.parametrize("kept", [60, 41])
def test_a_graph_from_before_is_refused(kept):
    """With as many entries in another order the shapes say nothing."""
    torch.manual_seed(1)
    p, q = (torch.randn(60, 4, device="cuda", requires_grad=True) for _ in range(2))
    opt = torch_ops.AdamW([([p, q], 0.1)])
    loss, other = (p * p).sum(), (q * q).sum()
    version = p._version
    opt.keep_rows([p], some(60, kept), [0])
    assert p._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    other.backward()  # a parameter that was left alone
    assert torch.equal(q.grad, 2 * q.detach())


@pytest.mark.parametrize("kept", [900, 650])
def test_a_render_from_before_is_refused(kept):
    """Its workspace has places for the old number of points."""
    scene = synthetic.tiny_scene(num_points=900, seed=4)
    texture, confidence, position, call = render(scene)
    opt = torch_ops.AdamW([([texture, confidence, position], 0.01)])
    loss = call()
    opt.keep_rows([texture, confidence, position], some(900, kept), [1, 1, 0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    call().backward()
    opt.step()
    assert texture.grad.shape == (4, kept) and position.grad.shape == (kept, 4) and all(torch.isfinite(t).all() for t in (texture, confidence, position))


@pytest.mark.parametrize("points, channels", [(650, 4), (900, 3), (1200, 4)])
def test_a_render_whose_tensors_were_exchanged_is_refused(points, channels):
    """As a program may do it by itself; torch does not see it."""
    scene = synthetic.tiny_scene(num_points=900, seed=5)
    other = synthetic.tiny_scene(num_points=points, channels=channels, seed=6)
    texture, confidence, position, call = render(scene)
    loss = call()
    for t, a in ((texture, other.texture), (confidence, other.confidence.reshape(1, -1)), (position, other.position)):
        t.data = torch.from_numpy(a).cuda()
    with pytest.raises(RuntimeError, match="rendered with 900 points of 4 channels"):
        loss.backward()


@pytest.mark.parametrize("kept", [60, 41])
def test_a_graph_that_has_saved_nothing_is_refused_too(kept):
    p = torch.randn(60, 4, device="cuda", requires_grad=True)
    opt = torch_ops.AdamW([([p], 0.1)])
    w = torch.randn(60, 4, device="cuda")
    loss = (p * w).sum()
    opt.keep_rows([p], some(60, kept), [0])
    with pytest.raises(RuntimeError, match="other entries"):
        loss.backward()
    assert p.grad is None
    (p * w[:kept]).sum().backward()
    assert torch.equal(p.grad, w[:kept])


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


def test_in_inference_mode():
    """An eviction needs no gradients; what it leaves is trained on."""
    torch.manual_seed(3)
    start = torch.randn(60, 4, device="cuda")
    results = []
    for mode in (torch.no_grad, torch.inference_mode):
        p, q = start.clone().requires_grad_(True), torch.ones(5, device="cuda", requires_grad=True)
        opt = torch_ops.AdamW([([p, q], 0.1)])
        for k in range(3):
            opt.zero_grad()
            ((p * p).sum() + (q * q).sum()).backward()
            opt.step()
            if k == 1:
                with mode():
                    opt.keep_rows([p], some(60, 41), [0])
                assert not p.is_inference() and not opt.exp_avg.is_inference() and p.is_leaf and p.requires_grad
        opt.load_moments([torch.zeros_like(p), torch.zeros_like(q)], [torch.zeros_like(p), torch.zeros_like(q)], 0)
        results.append(p.detach())
    assert torch.equal(*results)


def test_on_another_stream_than_the_parameters_own():
    """The old entries are read there, and their memory is not given out before that."""
    n = 1 << 20
    p = torch.randn(n, 4, device="cuda", requires_grad=True)
    opt = torch_ops.AdamW([([p], 0.1)])
    p.grad = torch.ones_like(p)
    index = some(n, n // 2 + 1)
    want = p.detach().index_select(0, index.long())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(50_000_000)
        opt.keep_rows([p], index, [0])
    taken = [torch.full((n, 4), float("nan"), device="cuda") for _ in range(4)]  # what an allocation at once would get
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(p.detach(), want) and torch.isnan(taken[0]).all()
