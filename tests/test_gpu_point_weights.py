"""What every point gave to the pixels of a render, against the definition in 64 bits on the lists that the render left, and against the
gradient that the sum of all pixels has with respect to the descriptors.

Bounds. All terms are positive, so relative errors do not grow in sums: a transmittance behind k fragments has 2 k roundings of float32, alpha
up to 4 (weight of the corner; with an activation the confidence is the float32 that the render has), their product one, and a sum of m terms m. A
bucket's mean in FUZZY_BLEND has as many roundings as fragments, and two more. Below 2^-126, deep in long lists, a rounding is off by up to 2^-150
whatever the value; no factor behind it is above 1, so a term is off by at most its roundings times that, and a sum by that times its terms,
of which there are no more than roundings counted here."""
import numpy as np
import pytest
import torch

from tests.test_gpu_torch_ext import _views
from vet_amd import abi, synthetic, torch_ops
from vet_amd.rasterizer import DeviceScene, make_params

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24


def definition(res, scene, params, confidence=None):
    """Sums in 64 bits and the largest number of roundings behind one."""
    mode, K = int(params.render_mode), int(params.debug_max_list_length)
    n = scene.num_points
    conf = (scene.confidence if confidence is None else confidence).astype(np.float64)
    total, roundings, terms = np.zeros(n), 0, np.zeros(n, np.int64)
    for b in range(len(scene.views)):
        offsets, keys, kept = res.offsets(b), res.fragments(b), res.kept(b)
        bases = res.layer_bases()
        if mode == abi.RENDER_BILINEAR_BLEND:
            at = res._view_array(res.layout.projected_base, res.layout.projected_stride, b, torch.float32, 2 * n).cpu().numpy().reshape(n, 2)
        for l in range(scene.num_layers):
            for q in np.nonzero(kept[bases[l]:bases[l + 1]])[0] + bases[l]:
                key = keys[offsets[q]:offsets[q] + kept[q]]
                ids, depth = (key & np.uint64(0xFFFFFFFF)).astype(np.int64), (key >> np.uint64(32)).astype(np.uint32).view(np.float32)
                share = np.ones(len(key))
                if mode == abi.RENDER_BILINEAR_BLEND:
                    ids, corner = ids >> 2, ids & 3
                    uv = at[ids].astype(np.float64) / 2 ** l
                    off = uv - np.floor(uv)
                    share = np.where(corner & 1, off[:, 0], 1 - off[:, 0]) * np.where(corner & 2, off[:, 1], 1 - off[:, 1])
                alpha = share * conf[ids if scene.index is None else scene.index[ids]]
                if mode == abi.RENDER_FUZZY_BLEND:
                    m = int((depth - depth[0] < np.float32(params.depth_accept_blend)).sum())
                    mean = alpha[:m].mean()
                    front = np.concatenate([[1.0], np.cumprod(1 - np.concatenate([[mean], alpha[m:]]))])
                    w = np.concatenate([np.full(m, mean / m), front[1:-1] * alpha[m:]])
                    roundings = max(roundings, m + 2)
                else:
                    w = np.concatenate([[1.0], np.cumprod(1 - alpha)[:-1]]) * alpha
                np.add.at(total, ids, w)
                np.add.at(terms, ids, 1)
                roundings = max(roundings, 2 * len(key) + 6)
    return total, roundings + terms


def close(got, want, roundings, before=0.0, decay=1.0):
    got = got.double().cpu().numpy()
    want = want + decay * before
    assert np.all(np.abs(got - want) <= 1.01 * STEP * (roundings + 3) * np.abs(want) + 2.0 ** -150 * roundings.astype(np.float64) ** 2)


def cases():
    tiny = synthetic.tiny_scene
    yield "one view", tiny(num_points=2000, K=8, seed=1), {}
    yield "no cut", tiny(num_points=2000, K=-1, seed=2), {}
    yield "long lists", tiny(num_points=20_000, K=-1, seed=3), {}
    yield "two views, one channel", tiny(num_points=1500, K=4, seed=4, num_views=2, channels=1), {}
    yield "rounds of views", tiny(num_points=900, w=61, h=45, num_layers=4, K=5, seed=5, num_views=6), {}
    yield "seen in part", tiny(num_points=1500, w=96, h=64, num_layers=3, K=8, seed=6, num_views=3), dict(expected_fragments=[100.0, 100.0, 100.0])
    yield "radius", tiny(num_points=3000, K=8, seed=7), dict(drop_out_points_by_radius=1)
    yield "one point", tiny(num_points=1, K=4, seed=8), {}
    shared = tiny(num_points=1200, K=6, seed=9, num_views=2)
    rng = np.random.default_rng(9)
    shared.index = rng.integers(0, 400, 1200).astype(np.int32)
    shared.dropout = (rng.random((2, 1200)) < 0.3).astype(np.float32)
    yield "shared rows and a mask", shared, {}
    yield "viewer", tiny(num_points=1500, K=8, seed=10), dict(viewer_only=1, stability_cutoff_value=0.5)


@pytest.mark.parametrize("mode", [1, 2, 3])
def test_the_definition(mode, rasterizer):
    for label, scene, over in cases():
        print("[case]", label, "mode", mode, flush=True)
        params = make_params(scene, render_mode=mode, **over)
        res = rasterizer.forward(DeviceScene(scene), params)
        want, roundings = definition(res, scene, params)
        start = torch.rand(scene.num_points, device="cuda")
        close(rasterizer.point_weights(res, start.clone(), 0.75), want, roundings, start.double().cpu().numpy(), 0.75)
        got = rasterizer.point_weights(res, torch.full_like(start, float("nan")), 0.0)
        close(got, want, roundings)
        # no order of atomics in it
        assert torch.equal(got, rasterizer.point_weights(res, torch.empty_like(start), 0.0))
        assert want.sum() > 0 or scene.num_points == 1


@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("K, views", [(8, 1), (8, 5), (-1, 1)])
def test_many_points(mode, K, views, rasterizer):
    """So many that the call clears a place for each of them instead of finding their pixels again."""
    scene = synthetic.tiny_scene(num_points=140_000, w=96, h=64, num_layers=2, K=K, seed=11, num_views=views)
    scene.dropout = (np.random.default_rng(11).random((views, 140_000)) < 0.2).astype(np.float32)
    params = make_params(scene, render_mode=mode)
    res = rasterizer.forward(DeviceScene(scene), params)
    want, roundings = definition(res, scene, params)
    start = torch.rand(scene.num_points, device="cuda")
    close(rasterizer.point_weights(res, start.clone(), 0.75), want, roundings, start.double().cpu().numpy(), 0.75)
    got = rasterizer.point_weights(res, torch.full_like(start, float("nan")), 0.0)
    close(got, want, roundings)
    assert torch.equal(got, rasterizer.point_weights(res, torch.empty_like(start), 0.0))


@pytest.mark.parametrize("mode", [1, 3])
def test_it_is_a_gradient(mode, rasterizer):
    """The sum of all pixels of a channel has these sums as its gradient with respect to that channel's descriptors, which the backward pass
    forms from the same lists by another route; and it leaves the backward pass as it was."""
    scene = synthetic.config2(num_points=60_000, seed=5, w=480, h=270)
    params = make_params(scene, render_mode=mode)
    dev = DeviceScene(scene)
    res = rasterizer.forward(dev, params)
    ones = [torch.ones_like(o) for o in res.out]
    want = rasterizer.backward(res, ones)
    got = rasterizer.point_weights(res, torch.empty(scene.num_points, device="cuda"), 0.0)
    g = want["texture"][0].double()
    assert got.sum() > 1000
    # a product with the upstream gradient and sums over the layers in both; 16 fragments a list in front
    assert ((got.double() - g).abs() <= 60 * STEP * g.abs()).all()
    again = rasterizer.backward(res, ones)
    for key in ("texture", "confidence", "points", "background"):
        assert torch.equal(want[key], again[key])


def test_raw_confidences(rasterizer):
    scene = synthetic.tiny_scene(num_points=2000, K=8, seed=21)
    scene.confidence = (0.2 * np.random.default_rng(1).standard_normal(2000)).astype(np.float32)
    params = make_params(scene, confidence_activation=1, confidence_scale=10.0)
    dev = DeviceScene(scene)
    res = rasterizer.forward(dev, params)
    got = rasterizer.point_weights(res, torch.empty(2000, device="cuda"), 0.0)
    confidence = rasterizer.pack_descriptors(dev, params)[:, 4].cpu().numpy()
    want, roundings = definition(res, scene, params, confidence)
    close(got, want, roundings)


def test_kept_descriptors_and_orders(rasterizer):
    scene = synthetic.tiny_scene(num_points=3000, K=8, seed=22)
    params, dev = make_params(scene), DeviceScene(scene)
    want = rasterizer.point_weights(rasterizer.forward(dev, params), torch.empty(3000, device="cuda"), 0.0)
    order = torch.randperm(3000, device="cuda", dtype=torch.int32)
    res = rasterizer.forward(dev, params, point_order=order, packed=rasterizer.pack_descriptors(dev, params))
    assert torch.equal(want, rasterizer.point_weights(res, torch.empty(3000, device="cuda"), 0.0))


def test_refusals(rasterizer):
    scene = synthetic.tiny_scene()
    res = rasterizer.forward(DeviceScene(scene), make_params(scene), save_for_backward=False)
    with pytest.raises(abi.VetrastError):
        rasterizer.point_weights(res, torch.zeros(scene.num_points, device="cuda"))


def test_no_points(rasterizer):
    scene = synthetic.tiny_scene()
    scene.position, scene.texture, scene.confidence = scene.position[:0], scene.texture[:, :0], scene.confidence[:0]
    dev = DeviceScene(scene)
    some = torch.zeros(256, device="cuda")
    dev.ptr = lambda name, ptr=dev.ptr: ptr(name) or (some.data_ptr() if name in ("position", "texture", "confidence") else None)
    res = rasterizer.forward(dev, make_params(scene))
    rasterizer.point_weights(res, torch.empty(0, device="cuda"))


# ---- through the shim ----------------------------------------------------------------------------------------------------------

def shim(scene, weight, texture=None, **kw):
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    tangents = torch.zeros((scene.poses_se3.shape[0], 6), dtype=torch.float64, device="cuda")
    return torch_ops.blend_point_cloud(cu(scene.texture) if texture is None else texture, cu(scene.background), cu(scene.position), tangents, cu(scene.intrinsics),
                                       cu(scene.confidence.reshape(1, -1)), cu(scene.poses_se3), None, _views(scene), scene.num_layers,
                                       use_environment_map=0, drop_out_points_by_radius=0, debug_max_list_length=scene.max_list_length,
                                       point_weight=weight, **kw)


@pytest.mark.parametrize("mode", [1, 2, 3])
def test_a_render_accumulates(mode, rasterizer):
    scene = synthetic.tiny_scene(num_points=4000, K=8, seed=31, num_views=2)
    dev, params = DeviceScene(scene), make_params(scene, render_mode=mode)
    one = rasterizer.point_weights(rasterizer.forward(dev, params), torch.zeros(4000, device="cuda"), 0.0)
    plain = shim(scene, None, render_mode=mode)
    weight = torch.zeros(4000, device="cuda")
    for k in range(3):  # without a backward pass
        version = weight._version
        outs = shim(scene, weight, render_mode=mode, point_weight_decay=0.5)
        assert weight._version > version and all(torch.equal(a, b) for a, b in zip(outs, plain))
    assert torch.allclose(weight, 1.75 * one, rtol=4 * 2.0 ** -23, atol=0)
    # and with one, whose gradients are what they were
    texture = torch.from_numpy(scene.texture).cuda().requires_grad_(True)
    sum(o.square().sum() for o in shim(scene, None, texture, train=True, render_mode=mode)).backward()
    want, texture.grad = texture.grad, None
    weight.zero_()
    outs = shim(scene, weight, texture, train=True, render_mode=mode)
    assert torch.equal(weight, one)
    sum(o.square().sum() for o in outs).backward()
    assert torch.equal(texture.grad, want)


def test_refusals_of_the_shim():
    scene = synthetic.tiny_scene(num_points=500)
    for bad in (torch.zeros(499, device="cuda"), torch.zeros(500, device="cuda").double(), torch.zeros(500), torch.zeros(1000, device="cuda")[::2],
                torch.zeros(500, device="cuda", requires_grad=True)):
        with pytest.raises(RuntimeError, match="point_weight"):
            shim(scene, bad)


def test_captured():
    scene = synthetic.tiny_scene(num_points=3000, K=8, seed=41)
    texture, weight = torch.from_numpy(scene.texture).cuda(), torch.zeros(3000, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    inputs = [cu(scene.background), cu(scene.position), torch.zeros((1, 6), dtype=torch.float64, device="cuda"), cu(scene.intrinsics),
              cu(scene.confidence.reshape(1, -1)), cu(scene.poses_se3)]

    def call():
        torch_ops.blend_point_cloud(texture, *inputs, None, _views(scene), scene.num_layers, use_environment_map=0, drop_out_points_by_radius=0,
                                    debug_max_list_length=8, point_weight=weight, size_bins_from_history=0, allow_distortion=1)

    with torch.no_grad(), torch.cuda.stream(stream):
        for _ in range(3):
            call()
    torch.cuda.current_stream().wait_stream(stream)
    one = weight / 3
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph, stream=stream):
        call()
    weight.zero_()
    for k in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(weight, k * one, rtol=8 * 2.0 ** -23, atol=0)
        torch.randn(100_000, device="cuda").sort()
