"""What the optimiser for libtorch callers (torch_ops.AdamW) does with its state when parameters, streams or the caller change around it."""
import numpy as np
import pytest
import torch

from tests import optim_model as om
from tests.test_gpu_adamw_torch import numbers, parameter, states
from vet_amd import torch_ops

pytestmark = pytest.mark.gpu


def grow(p, shape, seed):
    p.data = torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(p.dtype).cuda()
    p.grad = None
    p.grad = torch.ones_like(p)


def held(opt):
    """Everything the optimiser holds: arrays with their addresses, layout, counts."""
    return [t.data_ptr() for t in states(opt)], [t.clone() for t in states(opt)], opt.layout(), opt.steps()


def same(a, b):
    return a[0] == b[0] and all(torch.equal(x, y) for x, y in zip(a[1], b[1], strict=True)) and a[2:] == b[2:]


# ---- a change of size that fails ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_change_of_size_leaves_the_state(bits):
    """The first parameter grows while the second cannot be stepped: an error, and nothing has moved; once the second can, the step is the
    one that a run without the error takes."""
    shapes = [(3, 500), (40, 6), (129,)]
    ps, qs = ([parameter(s, torch.bfloat16, 70 + k) for k, s in enumerate(shapes)] for _ in range(2))
    a, b = (torch_ops.AdamW([(x, 0.01, 0.1)], moment_bits=bits, master_weights=True, seed=3) for x in (ps, qs))
    for _ in range(2):
        a.step()
        b.step()
    grow(ps[0], (4, 1700), 1)
    grow(qs[0], (4, 1700), 1)
    was, whole, before = ps[1].data, torch.zeros(40, 12, dtype=torch.bfloat16, device="cuda"), held(a)
    values = [p.detach().clone() for p in ps]
    ms = [torch.zeros(p.shape, device="cuda") for p in ps]
    ps[1].data = whole[:, ::2]
    for call in (a.step, a.step, lambda: a.load_moments(ms, ms, 5), a.step):
        with pytest.raises(RuntimeError, match="dense"):
            call()
        assert same(before, held(a)) and torch.equal(ps[0], values[0]) and torch.equal(ps[2], values[2]) and not whole.any()
    ps[1].data = was
    a.step()
    b.step()
    assert a.layout() == b.layout() == [(0, 6800), (6912, 240), (7168, 129)] and a.steps() == b.steps() == [1, 3, 3]
    assert all(torch.equal(x, y) for x, y in zip(ps + states(a), qs + states(b), strict=True))


@pytest.mark.parametrize("bits", [32, 8])
def test_memory_that_runs_out_leaves_the_state(bits):
    """Old and new state exist side by side when points are added, which is where memory ends first."""
    ps = [parameter((4, 1000), seed=80), parameter((300,), seed=81)]
    opt = torch_ops.AdamW([(ps, 0.01)], moment_bits=bits)
    opt.step()
    grow(ps[0], (4, 4_000_000), 2)
    grow(ps[1], (300,), 3)
    before, small = held(opt), ps[1].detach().clone()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (1 << 20)) / total)
    try:
        for _ in range(2):
            with pytest.raises(torch.OutOfMemoryError):
                opt.step()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert same(before, held(opt)) and torch.equal(ps[1], small)
    want, *_, tol, _, _ = om.step64(numbers(ps[0]), np.ones(ps[0].shape), np.zeros(ps[0].shape), np.zeros(ps[0].shape), 1, 0.01)
    opt.step()
    assert opt.layout() == [(0, 16_000_000), (16_000_000, 300)] and opt.steps() == [1, 2]
    assert (np.abs(numbers(ps[0]) - want) <= tol).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_tensors_of_another_size_are_refused(bits):
    p = parameter((1000,), torch.bfloat16, 82)
    opt = torch_ops.AdamW([([p], 0.01)], moment_bits=bits, master_weights=True)
    zeros = [torch.zeros(1000, device="cuda")]
    for t in states(opt):
        n, was = t.shape, p.detach().clone()
        t.resize_(0)
        for call in (opt.step, lambda: opt.load_moments(zeros, zeros, 1), opt.reload_master):
            with pytest.raises(RuntimeError, match="laid out"):
                call()
        assert torch.equal(p, was) and opt.steps() == [0]
        t.resize_(n)
    opt.step()
    assert opt.steps() == [1]
