"""A point without a fragment gives nothing, whatever its confidence, and that does not depend on how many points there are: calls clear a place
for every point of a large cloud, and look for the pixels of a small one's."""
import numpy as np
import pytest
import torch

from vet_amd import synthetic
from vet_amd.rasterizer import DeviceScene, make_params

pytestmark = pytest.mark.gpu

SMALL, LARGE = 3000, 140_000


def padded(scene, n, confidence):
    """The scene with n - N points behind the camera."""
    more = n - scene.num_points
    behind = np.tile(np.array([[0.0, 0.0, -50.0, 0.1]], np.float32), (more, 1))
    return synthetic.Scene(scene.name, np.concatenate([scene.position, behind]), np.concatenate([scene.texture, np.ones((4, more), np.float32)], 1),
                           np.concatenate([scene.confidence, np.resize(confidence, more).astype(np.float32)]), scene.background, scene.poses_se3, scene.intrinsics,
                           scene.views, scene.num_layers, scene.max_list_length, scene.seed)


def weights(rasterizer, scene, mode, decay):
    start = torch.full((scene.num_points,), 2.0, device="cuda")
    res = rasterizer.forward(DeviceScene(scene), make_params(scene, render_mode=mode))
    return rasterizer.point_weights(res, start, decay).cpu().numpy()


@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("views", [1, 3])
def test_points_that_no_view_sees(mode, views, rasterizer):
    scene = synthetic.tiny_scene(num_points=SMALL, K=8, seed=51, num_views=views)
    strange = np.array([np.nan, np.inf, -np.inf, 0.5])
    for n in (SMALL + 100, LARGE):
        for decay in (0.0, 0.5):
            got = weights(rasterizer, padded(scene, n, strange), mode, decay)
            assert np.all(got[SMALL:] == 2 * decay) and np.all(np.isfinite(got[:SMALL])), (n, decay)


@pytest.mark.parametrize("mode", [1, 2])
def test_strange_confidences_of_points_that_are_seen(mode, rasterizer):
    """What they leave in the lists is the same for a small and a large cloud: an opaque point in front of a NaN, a NaN whose bits are all ones."""
    scene = synthetic.tiny_scene(num_points=SMALL, K=8, seed=52)
    conf = scene.confidence.copy()
    conf[::7], conf[1::29], conf[2::31], conf[3::37] = 1.0, np.nan, np.inf, np.array([0xFFFFFFFF], np.uint32).view(np.float32)
    scene.confidence = conf
    small, large = (weights(rasterizer, padded(scene, n, np.array([0.5])), mode, 0.0)[:SMALL] for n in (SMALL + 100, LARGE))
    assert np.isnan(small).any() and (small > 0).any() and (small == 0).any()
    assert np.array_equal(small, large, equal_nan=True)
