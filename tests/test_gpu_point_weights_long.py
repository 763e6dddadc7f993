"""Weights over a pass of hundreds of renders are float32 from call to call: each call rounds the old value times the decay, and the sum. All terms are
positive, so n calls are off by 2 n roundings of 2^-24 at most, relative to the value."""
import numpy as np
import pytest
import torch

from vet_amd import synthetic
from vet_amd.rasterizer import DeviceScene, make_params

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("decay", [1.0, 0.9])
def test_hundreds_of_renders(decay, rasterizer):
    scene = synthetic.tiny_scene(num_points=3000, K=8, seed=61)
    res = rasterizer.forward(DeviceScene(scene), make_params(scene))
    one = rasterizer.point_weights(res, torch.empty(3000, device="cuda"), 0.0).double().cpu().numpy()
    weight = torch.zeros(3000, device="cuda")
    n, kept, want = 400, float(np.float32(decay)), np.zeros(3000)
    for _ in range(n):
        rasterizer.point_weights(res, weight, decay)
        want = kept * want + one
    assert want.max() > 1 and np.all(np.abs(weight.double().cpu().numpy() - want) <= 1.01 * 2 * n * 2.0 ** -24 * want)
