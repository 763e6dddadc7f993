"""Drop-out of points without a mask in memory: a call renders, and differentiates, bit by bit what it does with the mask that the
definition gives (vetrast_dropout's random bits, element view * N + point)."""
import numpy as np
import pytest
import torch

from tests import entries_model as em
from tests.test_gpu_torch_ext import _views
from vet_amd import abi, synthetic, torch_ops
from vet_amd.rasterizer import DeviceScene, make_params

pytestmark = pytest.mark.gpu


def mask(views, n, p, seed, step):
    return (em.dropout_bits(views * n, seed, step) < em.threshold(p)).reshape(views, n).astype(np.float32)


def same_as_with_a_mask(rasterizer, scene, params, p, seed, step, device_step=None, order=None):
    dev = DeviceScene(scene)
    got = rasterizer.forward(dev, params, point_dropout=p, dropout_seed=seed, dropout_step=step, dropout_device_step=device_step, point_order=order)
    scene.dropout = mask(len(scene.views), scene.num_points, p, seed, step + (int(device_step) if device_step is not None else 0))
    want = rasterizer.forward(DeviceScene(scene), params, point_order=order)
    for b in range(len(scene.views)):
        lists = [(r.offsets(b), r.fragments(b), r.kept(b)) for r in (got, want)]
        blended = [np.arange(o[-1]) - np.repeat(o[:-1], np.diff(o)) < np.repeat(k, np.diff(o)) for o, _, k in lists]  # behind a cut anything goes
        assert np.array_equal(lists[0][0], lists[1][0])
        assert np.array_equal(lists[0][1][blended[0]], lists[1][1][blended[1]])
    assert all(torch.equal(a, b) for a, b in zip(got.out, want.out))
    upstream = [torch.from_numpy(g).cuda() for g in scene.grad_out()]
    a, b = (rasterizer.backward(r, upstream, want_cameras=True) for r in (got, want))
    for key in ("texture", "confidence", "background", "points", "point_count", "pose", "intrinsics"):
        assert torch.equal(a[key], b[key]) or (scene.index is not None and key in ("texture", "confidence")), key
        assert torch.allclose(a[key], b[key], rtol=1e-5, atol=1e-6 * float(b[key].abs().max()))  # rows behind an index are added in any order
    weights = [rasterizer.point_weights(r, torch.empty(scene.num_points, device="cuda"), 0.0) for r in (got, want)]
    assert torch.equal(*weights) and (weights[0] > 0).any()
    scene.dropout = None


@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("views", [1, 2, 4, 7])
@pytest.mark.parametrize("distortion", [0, 1])
def test_modes_and_views(mode, views, distortion, rasterizer):
    scene = synthetic.tiny_scene(num_points=2501, w=64, h=48, num_layers=3, K=8, seed=10 * mode + views, num_views=views, channels=1 + (views + mode) % 4)
    params = make_params(scene, need_point_gradient=1, render_mode=mode, allow_distortion=distortion)
    same_as_with_a_mask(rasterizer, scene, params, 0.25, 2 ** 63 + 5, 2 ** 40 + views)


@pytest.mark.parametrize("p", [2.0 ** -18, 2.0 ** -16, 0.9])
def test_probabilities(p, rasterizer):
    scene = synthetic.tiny_scene(num_points=4000, K=8, seed=3)
    same_as_with_a_mask(rasterizer, scene, make_params(scene, need_point_gradient=1), p, 1, 1)


def test_everything_left_out(rasterizer):
    scene = synthetic.tiny_scene(num_points=1000, K=8, seed=4, num_views=2)
    res = rasterizer.forward(DeviceScene(scene), make_params(scene), point_dropout=1.0)
    assert all(res.offsets(b)[-1] == 0 for b in range(2))
    got = rasterizer.backward(res, [torch.ones_like(o) for o in res.out])
    assert not got["texture"].any() and not got["confidence"].any() and not got["points"].any()


def test_with_an_order_an_index_and_the_step_on_the_device(rasterizer):
    scene = synthetic.tiny_scene(num_points=3001, K=8, seed=5, num_views=2)
    order = torch.randperm(3001, device="cuda", dtype=torch.int32)
    count = torch.full((1,), 12, dtype=torch.int64, device="cuda")
    params = make_params(scene, need_point_gradient=1, drop_out_points_by_radius=1)
    same_as_with_a_mask(rasterizer, scene, params, 0.4, 9, 30, device_step=count, order=order)
    scene.index = np.random.default_rng(1).integers(0, 700, 3001).astype(np.int32)
    same_as_with_a_mask(rasterizer, scene, params, 0.4, 9, 30)


def test_crowded_bins_and_large_clouds(rasterizer):
    scene = synthetic.config2(num_points=200_000, seed=2, w=640, h=360)
    same_as_with_a_mask(rasterizer, scene, make_params(scene, need_point_gradient=1), 0.25, 4, 4)


# ---- through the shim ----------------------------------------------------------------------------------------------------------

def leaves(scene):
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return [cu(scene.texture).requires_grad_(True), cu(scene.background), cu(scene.position),
            torch.zeros((scene.poses_se3.shape[0], 6), dtype=torch.float64, device="cuda"), cu(scene.intrinsics),
            cu(scene.confidence.reshape(1, -1)).requires_grad_(True), cu(scene.poses_se3)]


def shim(scene, inputs, train=True, **kw):
    return torch_ops.blend_point_cloud(*inputs, None, _views(scene), scene.num_layers, train=train, use_environment_map=0, need_point_gradient=0,
                                       drop_out_points_by_radius=0, debug_max_list_length=scene.max_list_length,
                                       quirk_background_confidence_leak=0, size_bins_from_history=0, **kw)


def with_mask(rasterizer, scene, p, seed, step):
    scene.dropout = mask(len(scene.views), scene.num_points, p, seed, step)
    res = rasterizer.forward(DeviceScene(scene), make_params(scene))
    grads = rasterizer.backward(res, [torch.ones_like(o) for o in res.out], want_points=False)
    scene.dropout = None
    return res.out, grads


def test_a_training_step(rasterizer):
    scene = synthetic.tiny_scene(num_points=3000, K=8, seed=6, num_views=3)
    inputs = leaves(scene)
    for step in (1, 2):
        outs = shim(scene, inputs, dropout=0.25, dropout_seed=77, dropout_step=step)
        got = torch.autograd.grad(sum(o.sum() for o in outs), [inputs[0], inputs[5]])
        want, grads = with_mask(rasterizer, scene, 0.25, 77, step)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert torch.equal(got[0], grads["texture"]) and torch.equal(got[1].view(-1), grads["confidence"])
    # not in an evaluation, and a mask of torch's generator without a seed
    plain = shim(scene, inputs, train=False)
    assert all(torch.equal(a, b) for a, b in zip(plain, shim(scene, inputs, train=False, dropout=0.25, dropout_seed=77)))
    torch.manual_seed(3)
    a = shim(scene, inputs, dropout=0.25)
    torch.manual_seed(3)
    b = shim(scene, inputs, dropout=0.25)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and not torch.equal(a[0], plain[0])


def test_refusals_of_the_shim():
    scene = synthetic.tiny_scene(num_points=500)
    inputs = leaves(scene)
    for bad in (torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(RuntimeError, match="dropout_device_step"):
            shim(scene, inputs, dropout=0.25, dropout_seed=1, dropout_device_step=bad)
    with pytest.raises(RuntimeError):
        shim(scene, inputs, dropout=1.5, dropout_seed=1)
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    outs = shim(scene, inputs, dropout=0.25, dropout_seed=1, dropout_device_step=count)
    count += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        sum(o.sum() for o in outs).backward()


def test_captured_steps_count_by_themselves(rasterizer):
    """A captured training step whose drop-out goes by the count that the captured optimiser step keeps on the device."""
    scene = synthetic.tiny_scene(num_points=2000, K=8, seed=7)
    inputs = leaves(scene)
    opt = torch_ops.AdamW([([inputs[0]], 0.0)], capturable=True)  # a rate of zero: the scene stays
    stream = torch.cuda.Stream()

    def step():
        outs = shim(scene, inputs, dropout=0.5, dropout_seed=5, dropout_device_step=opt.device_step, allow_distortion=1)
        inputs[0].grad = torch.autograd.grad(sum(o.sum() for o in outs), inputs[0])[0]
        grad = inputs[0].grad.clone()
        opt.step()
        return [o.detach() for o in outs], grad

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    inputs[0].grad = None
    with torch.cuda.graph(graph, stream=stream):
        outs, grad = step()
    for k in range(3, 6):
        assert opt.steps() == [k]
        graph.replay()
        torch.cuda.synchronize()
        want, grads = with_mask(rasterizer, scene, 0.5, 5, k)
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(grad, grads["texture"])
        torch.randn(100_000, device="cuda").sort()
