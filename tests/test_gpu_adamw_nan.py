"""Gradients that are NaN of any sign and payload, as memory filled with ones reads: a block of 8-bit moments that meets one is lost as a
whole, and no other element is touched."""
import numpy as np
import pytest
import torch

from tests import optim_model as om
from tests.test_gpu_adamw import B, Batch, F, H, numbers

pytestmark = pytest.mark.gpu

PATTERNS = {F: [0xFFFFFFFF, 0xFFF00000, 0xFFEFFF00, 0xFFEFFEFF, 0xFFC00000, 0x7FFFFFFF, 0x7FC00000], B: [0xFFFF, 0xFFF0, 0xFFC0, 0x7FFF], H: [0xFFFF, 0xFF00, 0xFE00, 0x7FFF]}


@pytest.mark.parametrize("stochastic", [False, True])
@pytest.mark.parametrize("n", [128 * 5 + 9, 900_009], ids=["small", "large"])
@pytest.mark.parametrize("param,grad,master", [(F, F, False), (B, B, False), (B, B, True), (H, H, False), (B, F, False), (F, B, False), (F, H, False)],
                         ids=lambda t: str(t).replace("torch.", ""))
def test_a_block_is_lost_to_any_nan(param, grad, master, n, stochastic, rasterizer):
    for pattern in PATTERNS[grad]:
        batch = Batch(np.random.default_rng(21), [(n, param, grad, 0)], 8, master)
        i = batch.items[0]
        bad, place = [3, 300, n - 1], np.arange(n)
        width = torch.iinfo(torch.int32 if grad == F else torch.int16)
        i["grad"].t.view(torch.int32 if grad == F else torch.int16)[bad] = pattern if pattern <= width.max else pattern - (1 << width.bits)
        assert torch.isnan(i["grad"].t[bad]).all()
        struck, lost = np.isin(place, bad), np.isin(place // 128, [k // 128 for k in bad])
        for step, unfit in ((4, struck), (5, lost)):  # the second step reads what the first left
            batch.step(rasterizer, [(0.01, 0.0, step)], stochastic_rounding=stochastic)
            m, v = (x[:n] for x in om.decode(*(batch.of(i, x).cpu().numpy() for x in (batch.m, batch.v, batch.scale))))
            assert np.array_equal(np.isnan(m), lost) and np.array_equal(np.isnan(v), lost), (hex(pattern), step)
            assert np.array_equal(np.isnan(numbers(i["param"].t)), unfit), (hex(pattern), step)
            batch.check()
            i["grad"].t.fill_(0.5)
