"""Buffers that the calls of vet_amd/rasterizer.py write to are looked at before."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_buffers_of_norms(rasterizer):
    g = torch.ones(1000, device="cuda")
    whole = torch.full((8,), 3.0, device="cuda")
    need = 1 << 16
    for out in (whole[:1], whole[::4], whole.double(), torch.zeros(2), whole[:0]):
        with pytest.raises(AssertionError):
            rasterizer.gradient_norm([g], out=out)
    for workspace in (torch.zeros(need, device="cuda"), torch.zeros(need, dtype=torch.uint8), torch.zeros(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(AssertionError):
            rasterizer.gradient_norm([g], workspace=workspace)
    with pytest.raises(RuntimeError):
        rasterizer.gradient_norm([g], workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    rasterizer.gradient_norm([g], out=whole[2:4], workspace=torch.zeros(need, dtype=torch.uint8, device="cuda"))
    assert whole[2].item() == pytest.approx(1000 ** 0.5) and whole.cpu().tolist()[:2] == [3.0, 3.0] and (whole[4:] == 3).all()


def test_buffers_of_steps(rasterizer):
    p, g, m, v = (torch.ones(128, device="cuda") for _ in range(4))
    bytes_ = rasterizer.lib.vetrast_adamw_device_state_bytes(1)
    for kw in (dict(grad_scale=torch.ones(0, device="cuda")), dict(grad_scale=torch.ones(2, device="cuda")),
               dict(device_state=torch.zeros(bytes_, device="cuda")[:1]), dict(device_state=torch.zeros(bytes_, device="cuda")),
               dict(device_state=torch.zeros(2 * bytes_, dtype=torch.uint8, device="cuda")[::2]),
               dict(device_state=torch.zeros(bytes_ - 1, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(AssertionError):
            rasterizer.adamw_step([(p, g, 0, 0)], [(0.1, 0.0, 1)], m, v, **kw)
    assert (p == 1).all() and (m == 1).all() and (v == 1).all()
    state = torch.zeros(bytes_, dtype=torch.uint8, device="cuda")
    rasterizer.adamw_step([(p, g, 0, 0)], [(0.1, 0.0, 1)], m, v, grad_scale=torch.ones(1, device="cuda"), device_state=state)
    assert state[:8].view(torch.int64).item() == 1 and (p == 1).all()  # a rate of zero, as its factor in the state is
