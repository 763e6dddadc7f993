"""Dropout without a stored mask against its definition in 64 bits: the C interface over types, sizes, probabilities and addresses, and the
differentiable call of the shim over orders of memory, streams and graphs.

Bounds: the factor, the product and the sum with the residual are rounded to float32 (2^-24 each, relative to what they give), the result
once to its type (half a step; in float16 at least 2^-25, half of its smallest step)."""
import numpy as np
import pytest
import torch

from tests import entries_model as em
from vet_amd import abi, torch_ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def name(dtype):
    return str(dtype).split(".")[1]


def check(y, x, p, seed, step, residual=None):
    """y, x, residual: flat tensors in the order of memory."""
    ref, out = em.dropout(x.double().cpu().numpy(), p, seed, step, None if residual is None else residual.double().cpu().numpy())
    got, added = y.double().cpu().numpy(), 0.0 if residual is None else residual.double().cpu().numpy()
    bound = em.HALF_STEP[name(y.dtype)] * np.abs(ref) + 2.0 ** -23 * np.abs(ref - added) + 2.0 ** -24 * np.abs(ref)
    bound = 1.001 * bound + (2.0 ** -25 if y.dtype == torch.float16 else 2.0 ** -133)
    assert np.all(np.abs(got - ref) <= bound)
    if residual is None:
        assert np.all(got[out] == 0)
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 511, 2047, 2048, 2049, 6145, 100_003])
def test_sizes(rasterizer, dtype, n):
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, generator=gen, device="cuda").to(dtype)
    r = torch.randn(n, generator=gen, device="cuda").to(dtype)
    for p, seed, step in ((0.1, 3, 0), (0.5, 2 ** 64 - 1, 2 ** 64 - 2), (0.997, 1 << 40, 1 << 33)):
        check(rasterizer.dropout(x, p, seed, step), x, p, seed, step)
        check(rasterizer.dropout(x, p, seed, step, residual=r), x, p, seed, step, r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [1, 3])
def test_addresses(rasterizer, dtype, shift):
    """Tensors that begin at any element of their type; their neighbours in memory stay."""
    n = 5003
    big = [torch.randn(n + 8, device="cuda").to(dtype) for _ in range(3)]
    x, r, y = (b[shift + k:shift + k + n] for k, b in enumerate(big))
    before = big[2].clone()
    rasterizer.dropout(x, 0.3, 11, 5, residual=r, out=y)
    check(y, x, 0.3, 11, 5, r)
    at = shift + 2
    assert torch.equal(big[2][:at], before[:at]) and torch.equal(big[2][at + n:], before[at + n:])


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -17, 2.0 ** -16, 0.25, 1 - 2.0 ** -16, 1 - 2.0 ** -17, 1.0])
def test_probabilities(rasterizer, p):
    x = torch.randn(70_001, device="cuda")
    y = rasterizer.dropout(x, p, 5, 9)
    out = check(y, x, p, 5, 9)
    if em.threshold(p) == 0:
        assert torch.equal(x, y)
    if em.threshold(p) == 65536:
        assert out.all()


def test_shares(rasterizer):
    """The share that is left out is p within five standard deviations, for every place in a group of eight and for pairs of neighbours,
    seeds and steps as for a coin that was thrown anew."""
    n, p = 1 << 20, 0.25
    x = torch.ones(n, device="cuda")
    out = [rasterizer.dropout(x, p, seed, step) == 0 for seed, step in ((1, 1), (2, 1), (1, 2), (1 + (1 << 32), 1), (1, 1 + (1 << 32)))]
    for o in out:
        assert abs(o.double().mean().item() - p) < 5 * (p * (1 - p) / n) ** 0.5
        part = o.view(-1, 8).double().mean(0)
        assert (part - p).abs().max().item() < 5 * (p * (1 - p) / (n / 8)) ** 0.5
    both = p * p
    for k in (1, 2, 7, 8, 64):
        assert abs((out[0][k:] & out[0][:-k]).double().mean().item() - both) < 5 * (both / n) ** 0.5
    for o in out[1:]:
        assert abs((out[0] & o).double().mean().item() - both) < 5 * (both * (1 - both) / n) ** 0.5


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_left_out_leaves_nothing_behind(rasterizer, dtype):
    x = torch.full((4096,), float("nan"), device="cuda", dtype=dtype)
    x[::2] = float("inf")
    out = torch.from_numpy(em.dropout_bits(4096, 21, 4) < em.threshold(0.4)).cuda()
    y = rasterizer.dropout(x, 0.4, 21, 4)
    assert (y[out] == 0).all() and y[~out][1::2].shape and not torch.isfinite(y[~out]).any()
    r = torch.randn(4096, device="cuda").to(dtype)
    assert torch.equal(rasterizer.dropout(x, 0.4, 21, 4, residual=r)[out], r[out])


def test_in_place(rasterizer):
    x, r = torch.randn(9001, device="cuda"), torch.randn(9001, device="cuda")
    want = rasterizer.dropout(x, 0.2, 8, 1, residual=r)
    onto_x, onto_r = x.clone(), r.clone()
    rasterizer.dropout(onto_x, 0.2, 8, 1, residual=r, out=onto_x)
    rasterizer.dropout(x, 0.2, 8, 1, residual=onto_r, out=onto_r)
    assert torch.equal(onto_x, want) and torch.equal(onto_r, want)


def test_places_beyond_33_bits(rasterizer):
    """More elements than a launch takes, in place; looked at where launches meet and at the end."""
    n = (1 << 33) + 5 * 2048 + 13
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    rasterizer.dropout(x, 0.25, 77, 6, out=x)
    for first in (0, (1 << 32) - 1000, (1 << 33) - 4003, n - 3001):
        some = x[first:first + min(8000, n - first)]
        out = em.dropout_bits(some.numel(), 77, 6, first) < em.threshold(0.25)
        assert np.array_equal(some.float().cpu().numpy() == 0, out)


# ---- the shim --------------------------------------------------------------------------------------------------------------

def layouts(dtype):
    x = torch.randn(3, 5, 14, 11, device="cuda").to(dtype)
    yield "rows", x
    yield "channels last", x.contiguous(memory_format=torch.channels_last)
    yield "turned", x.permute(2, 0, 3, 1)
    yield "gaps", x[:, ::2, 1:]
    yield "one for all", x[:, :1].expand(3, 4, 14, 11)
    yield "a number", x[0, 0, 0, 0].clone()
    yield "none", x[:0]


def dense_order(x):
    """x's elements in the order of memory that the call gives its result, flat."""
    kept = x if x.is_contiguous() or torch._prims_common.is_non_overlapping_and_dense(x) else x.contiguous()
    return torch.as_strided(kept, (kept.numel(),), (1,), kept.storage_offset()), kept.stride()


@pytest.mark.parametrize("dtype", TYPES)
def test_orders_of_memory_and_gradients(dtype):
    for label, x in layouts(dtype):
        print("[case]", label, flush=True)
        x = x.detach().requires_grad_(True)
        r = torch.randn_like(x, memory_format=torch.contiguous_format).requires_grad_(True)
        y = torch_ops.dropout(x, 0.3, seed=9, step=2, residual=r)
        flat, strides = dense_order(x.detach())
        assert y.dtype == dtype and y.shape == x.shape and y.stride() == strides
        dy = torch.randn_like(y, memory_format=torch.contiguous_format)  # an order of its own
        gx, gr = torch.autograd.grad(y, [x, r], dy)
        if x.numel() == 0:
            continue
        in_order = lambda t: torch.as_strided(torch.empty_strided(x.shape, strides, dtype=dtype, device="cuda").copy_(t), (x.numel(),), (1,))
        check(in_order(y.detach()), flat, 0.3, 9, 2, in_order(r.detach()))
        check(in_order(gx), in_order(dy), 0.3, 9, 2)
        assert torch.equal(gr, dy)


def test_gradients_against_differences():
    """The call is linear in x up to rounding: the gradient's product with a direction is what a step along it changes."""
    x, d, dy = (torch.randn(4099, device="cuda", dtype=torch.float32) for _ in range(3))
    x.requires_grad_(True)
    y = torch_ops.dropout(x, 0.45, seed=3, step=1)
    (g,) = torch.autograd.grad(y, x, dy)
    moved = torch_ops.dropout(x.detach() + 0.5 * d, 0.45, seed=3, step=1)
    change = ((moved.double() - y.detach().double()) * dy.double()).sum().item()
    size = ((moved.abs() + y.detach().abs()).double() * dy.abs().double()).sum().item()
    assert abs(change - 0.5 * (g.double() * d.double()).sum().item()) <= 4 * 2.0 ** -24 * size


def test_gradients_of_shared_and_broadcast_inputs():
    x = torch.randn(1, 7, 1, device="cuda", requires_grad=True)
    y = torch_ops.dropout(x.expand(5, 7, 3), 0.5, seed=1, step=1, residual=x.expand(5, 7, 3))
    (g,) = torch.autograd.grad(y.sum(), x)
    factor, _ = em.dropout(np.ones(105), 0.5, 1, 1)
    assert np.array_equal(g.view(-1).cpu().numpy(), (factor.reshape(5, 7, 3) + 1).sum((0, 2)))
    # the same tensor as input and residual
    z = torch.randn(64, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(torch_ops.dropout(z, 0.5, seed=1, step=1, residual=z).sum(), z)
    assert np.array_equal(g.cpu().numpy(), em.dropout(np.ones(64), 0.5, 1, 1)[0] + 1)


def test_the_gradient_has_a_gradient():
    x = torch.randn(513, device="cuda", requires_grad=True)
    dy = torch.randn(513, device="cuda", requires_grad=True)
    y = torch_ops.dropout(x, 0.5, seed=6, step=3)
    (gx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    (again,) = torch.autograd.grad(gx, dy, torch.ones_like(gx))
    assert np.array_equal(again.cpu().numpy(), em.dropout(np.ones(513), 0.5, 6, 3)[0])


def test_only_what_is_asked_for():
    x, r = torch.randn(100, device="cuda"), torch.randn(100, device="cuda", requires_grad=True)
    y = torch_ops.dropout(x, 0.5, seed=1, residual=r)
    (g,) = torch.autograd.grad(y.sum(), r)
    assert (g == 1).all()
    with torch.no_grad():
        assert not torch_ops.dropout(x, 0.5, seed=1, residual=r).requires_grad


def test_refusals_of_the_shim():
    x = torch.randn(8, device="cuda")
    for bad, match in ((dict(residual=torch.randn(9, device="cuda")), "shape"), (dict(residual=torch.randn(8, device="cuda").half()), "type"),
                       (dict(residual=torch.randn(8)), "on cuda"), (dict(device_step=torch.zeros(2, dtype=torch.int64, device="cuda")), "one int64"),
                       (dict(device_step=torch.zeros(1, device="cuda")), "one int64"), (dict(device_step=torch.zeros(1, dtype=torch.int64)), "on cuda")):
        with pytest.raises(RuntimeError, match=match):
            torch_ops.dropout(x, 0.5, seed=1, **bad)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        torch_ops.dropout(x.double(), 0.5, seed=1)
    with pytest.raises(abi.VetrastError):
        from vet_amd.rasterizer import Rasterizer
        Rasterizer().dropout(x, 2.0, 1)


def test_the_step_on_the_device():
    count = torch.full((1,), 40, dtype=torch.int64, device="cuda")
    x = torch.randn(3000, device="cuda", requires_grad=True)
    y = torch_ops.dropout(x, 0.3, seed=2, step=2, device_step=count)
    check(y.detach(), x.detach(), 0.3, 2, 42)
    count += 1  # noticed, instead of a gradient with another mask
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_captured_forward_and_backward():
    """Replays count on the device; each is checked, with work of the program and waits between them."""
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    x = torch.randn(5000, device="cuda", requires_grad=True)
    stream = torch.cuda.Stream()

    def step():
        y = torch_ops.dropout(x, 0.3, seed=4, device_step=count, residual=x)
        (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
        return y, g

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y, g = step()
        count += 1
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        check(y.detach(), x.detach(), 0.3, 4, k, x.detach())
        factor, _ = em.dropout(np.ones(5000), 0.3, 4, k)
        assert np.abs(g.cpu().numpy() - factor - 1).max() <= 4 * 2.0 ** -24 * 2.5
        torch.randn(100_000, device="cuda").sort()


@pytest.mark.parametrize("between", [False, True])
def test_a_capture_beside_a_living_graph_of_the_same_leaf_is_refused(between):
    """torch's backward pass would wait there for a stream outside the capture, which ends the process."""
    x = torch.randn(512, device="cuda", requires_grad=True)
    living = torch_ops.dropout(x, 0.3, seed=4, step=1)
    out = torch.empty(512, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        with pytest.raises(RuntimeError, match="still lives"):
            torch_ops.dropout(2 * x if between else x, 0.3, seed=4, step=2)
        out.copy_(torch_ops.dropout(x.detach(), 0.3, seed=4, step=2))
    graph.replay()
    torch.cuda.synchronize()
    check(out, x.detach(), 0.3, 4, 2)
    living.sum().backward()
    assert x.grad is not None


def test_another_stream():
    x = torch.randn(1 << 22, device="cuda")
    want = torch_ops.dropout(x, 0.1, seed=1, step=1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        z = x * 1.0
        got = torch_ops.dropout(z, 0.1, seed=1, step=1)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
