"""The optimiser for libtorch callers (torch_ops.AdamW, grad_norm, pack_moments, unpack_moments): what it does with parameters as
programs have them, its refusals, captured steps, and a run of everything together behind the rasterizer."""
import threading

import numpy as np
import pytest
import torch

from tests import optim_model as om
from vet_amd import synthetic, torch_ops
from tests.test_gpu_torch_ext import _views

pytestmark = pytest.mark.gpu


def parameter(shape, dtype=torch.float32, seed=0, gradient=True):
    gen = torch.Generator().manual_seed(seed)
    p = (torch.randn(shape, generator=gen) * 0.1).to(dtype).cuda().requires_grad_(True)
    if gradient:
        p.grad = (torch.randn(shape, generator=gen) * 0.01).to(dtype).cuda()
    return p


def numbers(t):
    return t.detach().cpu().double().numpy()


def states(opt):
    return [t for t in (opt.exp_avg, opt.exp_avg_sq, opt.block_scale, opt.master) if t is not None]


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_follow_the_definition(bits):
    ps = [parameter((5, 700), seed=1), parameter((3,), seed=2), parameter((129,), seed=3), parameter((64, 64), seed=4, gradient=False)]
    opt = torch_ops.AdamW([(ps[:2], 0.01, 0.1), (ps[2:], 0.003, 0.0)], moment_bits=bits, seed=21)
    lay = opt.layout()
    assert lay == [(0, 3500), (3584, 3), (3712, 129), (3968, 4096)]
    last = ps[3].detach().clone()
    for step in range(1, 5):
        before = [numbers(p) for p in ps]
        m0, v0 = (numbers(t) for t in opt.moments())
        opt.set_lr(1, 0.003 * step)
        opt.step()
        for k, p in enumerate(ps[:3]):
            f, n = lay[k]
            want, m, v, tol, tol_m, tol_v = om.step64(before[k].reshape(-1), numbers(p.grad).reshape(-1), m0[f:f + n], v0[f:f + n], step,
                                                      *((0.01, 0.1) if k < 2 else (0.003 * step, 0.0)))
            assert (np.abs(numbers(p).reshape(-1) - want) <= tol).all()
            if bits == 32:
                assert (np.abs(numbers(opt.exp_avg)[f:f + n] - m) <= tol_m).all()
            p.grad.mul_(-0.7)
    assert opt.steps() == [4, 4, 4, 0] and torch.equal(ps[3], last)
    # one that starts later counts for itself
    before, g = numbers(ps[3]), torch.full_like(ps[3], 0.5)
    ps[3].grad = g
    opt.step(zero_grad=True)
    assert opt.steps() == [5, 5, 5, 1] and not any(p.grad.any() for p in ps)
    want, _, _, tol, *_ = om.step64(before, numbers(torch.full_like(g, 0.5)), np.zeros_like(before), np.zeros_like(before), 1, 0.012)
    assert (np.abs(numbers(ps[3]) - want) <= tol).all()
    opt.zero_grad()


@pytest.mark.parametrize("bits", [32, 8])
def test_any_dense_order_of_dimensions(bits):
    """A channels-last or transposed parameter steps like its contiguous twin, whatever the gradient's strides are. The moments
    follow the parameter's memory."""
    base = parameter((6, 5, 3, 4), seed=5)
    g = torch.randn((6, 5, 3, 4), generator=torch.Generator().manual_seed(6)).cuda()
    kinds = [lambda t: t.clone(), lambda t: t.clone(memory_format=torch.channels_last), lambda t: t.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0)]
    for own in kinds:
        for other in kinds:
            p, q = own(base.detach()).requires_grad_(True), base.detach().clone().requires_grad_(True)
            p.grad, q.grad = other(g), g.clone()
            a, b = (torch_ops.AdamW([([x], 0.01, 0.0)], moment_bits=bits) for x in (p, q))
            a.step(zero_grad=True)
            b.step(zero_grad=True)
            assert torch.equal(p, q) and not p.grad.any() and not q.grad.any()
            a.set_step(0)
    # a gradient that lies in one number, and one with gaps
    p, q = (base.detach().clone().requires_grad_(True) for _ in range(2))
    p.grad, q.grad = torch.full((1,), 0.25, device="cuda").expand(6, 5, 3, 4), torch.full((6, 5, 3, 4), 0.25, device="cuda")
    a, b = (torch_ops.AdamW([([x], 0.01, 0.0)], moment_bits=bits) for x in (p, q))
    a.step(zero_grad=True)
    b.step(zero_grad=True)
    assert torch.equal(p, q) and p.grad.shape == p.shape and not p.grad.any()
    p.grad = torch.zeros(6, 5, 3, 8, device="cuda")[..., ::2]
    p.grad += 0.5
    q.grad.fill_(0.5)
    assert torch.equal(a.grad_norm(), b.grad_norm())
    a.step(zero_grad=True)
    b.step()
    assert torch.equal(p, q) and not p.grad.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_master_weights(dtype):
    ps = [parameter((300, 7), dtype, 7), parameter((11,), dtype, 8), parameter((5,), torch.float32, 9)]
    opt = torch_ops.AdamW([(ps, 1e-4, 0.1)], master_weights=True)
    for (f, n), p in zip(opt.layout(), ps):
        assert torch.equal(opt.master[f:f + n], p.detach().float().reshape(-1))
    exact = [numbers(p).reshape(-1) for p in ps]
    m, v = [np.zeros(p.numel()) for p in ps], [np.zeros(p.numel()) for p in ps]
    total = [0.0] * 3
    for step in range(1, 31):
        opt.step()
        for k, p in enumerate(ps):
            exact[k], m[k], v[k], tol, *_ = om.step64(exact[k], numbers(p.grad).reshape(-1), m[k], v[k], step, 1e-4, 0.1)
            total[k] = total[k] + tol
    for k, ((f, n), p) in enumerate(zip(opt.layout(), ps)):
        held = p if p.dtype == torch.float32 else opt.master[f:f + n]
        # moments drift with their own roundings, at most thirty steps' worth in the quotient
        assert (np.abs(numbers(held).reshape(-1) - exact[k]) <= total[k] * 2 + 30 * 30 * 8 * om.U * 1e-4).all()
        if p.dtype != torch.float32:
            assert torch.equal(p.detach().reshape(-1), opt.master[f:f + n].to(dtype))
    with torch.no_grad():
        ps[0].zero_()
    opt.reload_master()
    assert not opt.master[:2100].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_that_changes_its_size_starts_anew(bits):
    """What adding points does: the others keep their moments and counts."""
    ps = [parameter((4, 1000), seed=10), parameter((1, 1000), seed=11), parameter((4,), seed=12)]
    twins = [p.detach().clone().requires_grad_(True) for p in ps]
    for p, q in zip(ps, twins):
        q.grad = p.grad.clone()
    opt, ref = (torch_ops.AdamW([([x[0]], 0.01, 0.0), (x[1:], 0.01, 0.0)], moment_bits=bits, seed=4) for x in (ps, twins))
    for o in (opt, ref):
        o.step()
        o.step()
    more = torch.randn(4, 1500, generator=torch.Generator().manual_seed(1)).cuda()
    ps[0].data = more.clone()
    ps[0].grad = torch.ones_like(more)
    opt.step()
    ref.step()
    assert opt.steps() == [1, 3, 3] and opt.layout()[1] == (6016, 1000)
    want, *_, tol_p, _, _ = om.step64(numbers(more), np.ones((4, 1500)), np.zeros((4, 1500)), np.zeros((4, 1500)), 1, 0.01)
    assert (np.abs(numbers(ps[0]) - want) <= tol_p).all()
    if bits == 32:
        for k in (1, 2):
            assert torch.equal(ps[k], twins[k])
    else:  # other random bits from here on, as the elements have other numbers; this step did not read them yet
        for k in (1, 2):
            assert torch.equal(ps[k], twins[k])


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_load_for_parameters_that_changed_their_size(bits):
    """Before any step has seen the new size: the state is laid out for it."""
    ps = [parameter((4, 100), torch.bfloat16, 60), parameter((30,), torch.bfloat16, 61)]
    opt = torch_ops.AdamW([(ps, 0.01)], moment_bits=bits, master_weights=True)
    opt.step()
    kept = opt.master[512:542].clone()
    ps[0].data = torch.randn(4, 1500, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    ms = [torch.full((4, 1500), 0.25, device="cuda"), torch.full((30,), -1.0, device="cuda")]
    opt.load_moments(ms, [m * m for m in ms], 7)
    assert opt.layout() == [(0, 6000), (6016, 30)] and opt.steps() == [7, 7]
    assert torch.equal(opt.master[:6000], ps[0].detach().float().reshape(-1)) and torch.equal(opt.master[6016:6046], kept)
    m, v = opt.moments()
    for (f, n), x in zip(opt.layout(), ms):  # a power of two is within half a code of itself, and the offset another 2^-15 of it
        assert (abs(m[f:f + n] - x.reshape(-1)) <= abs(x.reshape(-1)) / 16).all() and (abs(v[f:f + n] - x.reshape(-1) ** 2) <= x.reshape(-1) ** 2 / 16).all()
    fixed = torch_ops.AdamW([(ps, 0.01)], moment_bits=bits, capturable=True)
    ps[1].data = torch.zeros(31, dtype=torch.bfloat16, device="cuda")
    ms[1] = torch.zeros(31, device="cuda")
    with pytest.raises(RuntimeError, match="change their size"):
        fixed.load_moments(ms, ms, 1)


def test_moments_move_between_widths():
    ps = [parameter((4, 777), seed=13), parameter((777,), seed=14)]
    full = torch_ops.AdamW([(ps, 0.01, 0.0)])
    for _ in range(3):
        full.step()
    parts = [tuple(t[f:f + n].clone() for t in full.moments()) for f, n in full.layout()]
    ms, vs = [m for m, _ in parts], [v for _, v in parts]
    small = torch_ops.AdamW([(ps, 0.01, 0.0)], moment_bits=8)
    small.load_moments(ms, vs, 3)
    assert small.steps() == [3, 3]
    mc, vc, scale = torch_ops.pack_moments(ms, vs)
    assert torch.equal(mc, small.exp_avg) and torch.equal(vc, small.exp_avg_sq) and torch.equal(scale, small.block_scale)
    m, v = small.moments()
    back = torch_ops.AdamW([(ps, 0.01, 0.0)])
    back.load_moments([m[f:f + n] for f, n in small.layout()], [v[f:f + n] for f, n in small.layout()], 3)
    assert torch.equal(back.exp_avg, m) and torch.equal(back.exp_avg_sq, v)
    unit = np.exp2(numbers(scale) - 127.0)
    for k, (a, b) in enumerate(((m, full.exp_avg), (v, full.exp_avg_sq))):
        a, b, u = numbers(a), numbers(b), np.repeat(unit[:, k], 128)
        assert (np.abs(a - b) <= (np.abs(b) + u) / 16 * 1.0001 + (u / 8 if k else 0)).all()
    assert all(t.numel() == 0 for t in torch_ops.pack_moments([torch.zeros(0, device="cuda")], [torch.zeros(0, device="cuda")]))
    assert all(t.numel() == 0 for t in torch_ops.unpack_moments(*torch_ops.pack_moments([torch.zeros(0, device="cuda")], [torch.zeros(0, device="cuda")])))


def test_moments_follow_the_parameters_order():
    """Loaded in any order of dimensions, they mean the same elements; flat ones are in the order of memory."""
    base = torch.randn(4, 3, 5, 6, generator=torch.Generator().manual_seed(3)).cuda()
    p = base.clone(memory_format=torch.channels_last).requires_grad_(True)
    p.grad = torch.zeros_like(p)
    m, v = torch.randn_like(base).contiguous(), torch.rand_like(base).contiguous()
    for bits in (32, 8):
        forms = []
        for x, y in ((m, v), (m.clone(memory_format=torch.channels_last), v), (m.transpose(0, 3).contiguous().transpose(0, 3), v),
                     (m.permute(0, 2, 3, 1).reshape(-1), v.permute(0, 2, 3, 1).reshape(-1))):
            opt = torch_ops.AdamW([([p], 0.01)], moment_bits=bits)
            opt.load_moments([x], [y], 5)
            forms.append(opt.moments())
        assert all(torch.equal(a[0], forms[0][0]) and torch.equal(a[1], forms[0][1]) for a in forms)
        if bits == 32:
            assert torch.equal(forms[0][0][:360].view(4, 5, 6, 3).permute(0, 3, 1, 2), m)


def test_zeros_stay_behind_the_last_element():
    """Also in masters of a block that is lost."""
    p = parameter((130,), torch.bfloat16, 50)
    opt = torch_ops.AdamW([([p], 0.01)], moment_bits=8, master_weights=True)
    p.grad[129] = float("nan")
    for _ in range(2):
        opt.step()
    assert torch.isnan(p[128:]).all() and torch.isfinite(p[:128]).all()
    assert not opt.master[130:].any() and not opt.exp_avg[130:].any() and not opt.exp_avg_sq[130:].any()


def test_refusals():
    p = parameter((8, 8))
    make = lambda ps=None, **kw: torch_ops.AdamW([([p] if ps is None else ps, 0.01, 0.0)], **kw)  # noqa: E731
    for bad in (dict(moment_bits=16), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=0.0), dict(ps=[]), dict(ps=[p, p]),
                dict(ps=[torch.zeros(3)]), dict(ps=[torch.zeros(3, dtype=torch.float64, device="cuda")]),
                dict(ps=[torch.zeros(3, dtype=torch.int32, device="cuda")]), dict(ps=[torch.zeros(8, 8, device="cuda")[:, ::2]]),
                dict(ps=[torch.zeros(1, device="cuda").expand(5)])):
        with pytest.raises(RuntimeError):
            make(**bad)
    opt = make()
    for scale in (torch.ones(1), torch.ones(1, dtype=torch.float64, device="cuda"), torch.ones(3, device="cuda"), torch.ones(0, device="cuda"),
                  torch.ones(4, device="cuda")[::2]):
        with pytest.raises(RuntimeError):
            opt.step(grad_scale=scale)
    assert opt.steps() == [0] and not opt.exp_avg.any()
    for call in (lambda: opt.set_lr(1, 0.1), lambda: opt.set_step(-1), lambda: opt.load_moments([], [], 1),
                 lambda: opt.load_moments([torch.zeros(3, device="cuda")], [torch.zeros(3, device="cuda")], 1),
                 lambda: opt.load_moments([torch.zeros(64, device="cuda")], [torch.zeros(64)], 1),
                 lambda: torch_ops.grad_norm([]), lambda: torch_ops.grad_norm([torch.zeros(3)]),
                 lambda: torch_ops.grad_norm([torch.zeros(3, dtype=torch.float64, device="cuda")]),
                 lambda: torch_ops.grad_norm([torch.zeros(3, device="cuda"), torch.zeros(3)]),
                 lambda: torch_ops.grad_norm([torch.zeros(3, device="cuda")], max_norm=float("nan")),
                 lambda: torch_ops.pack_moments([], []),
                 lambda: torch_ops.pack_moments([torch.zeros(3, device="cuda")], []),
                 lambda: torch_ops.pack_moments([torch.zeros(3, device="cuda")], [torch.zeros(4, device="cuda")]),
                 lambda: torch_ops.pack_moments([torch.zeros(3, device="cuda", dtype=torch.bfloat16)] * 1, [torch.zeros(3, device="cuda")]),
                 lambda: torch_ops.unpack_moments(torch.zeros(100, dtype=torch.uint8, device="cuda"), torch.zeros(100, dtype=torch.uint8, device="cuda"),
                                                  torch.zeros(1, 2, dtype=torch.uint8, device="cuda")),
                 lambda: torch_ops.unpack_moments(torch.zeros(128, dtype=torch.uint8, device="cuda"), torch.zeros(128, dtype=torch.uint8, device="cuda"),
                                                  torch.zeros(2, 2, dtype=torch.uint8, device="cuda")),
                 lambda: torch_ops.unpack_moments(*[torch.zeros(128, device="cuda")] * 3)):
        with pytest.raises(RuntimeError):
            call()
    q = parameter((8,))
    turned = torch_ops.AdamW([([q], 0.01)])
    q.data = q.data.bfloat16()
    q.grad = None
    q.grad = torch.zeros_like(q)
    with pytest.raises(RuntimeError, match="type"):
        turned.step()
    fixed = make(capturable=True)
    fixed.step()
    p.data = torch.zeros(3, 3, device="cuda")
    p.grad = None
    p.grad = torch.zeros(3, 3, device="cuda")
    with pytest.raises(RuntimeError):
        fixed.step()


def test_parameters_made_in_inference_mode():
    with torch.inference_mode():
        p = torch.zeros(100, device="cuda")
        p.grad = torch.ones(100, device="cuda")
    opt = torch_ops.AdamW([([p], 0.5)])
    opt.step(zero_grad=True)
    assert opt.steps() == [1] and torch.allclose(p, torch.full_like(p, -0.5)) and not p.grad.any()


def test_no_gradient_anywhere_changes_nothing():
    p = parameter((40,), gradient=False)
    was = p.detach().clone()
    opt = torch_ops.AdamW([([p], 0.01, 0.5)])
    opt.step(zero_grad=True)
    opt.zero_grad()
    assert opt.steps() == [0] and torch.equal(p, was)
    with pytest.raises(RuntimeError):
        opt.grad_norm()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count(bits):
    """Norm and step in a graph: replayed several times with eager work between, every replay is the eager step. One that overflowed
    is left out and not counted."""
    shapes = [(700, 3), (5,), (4096,), (1,)]
    ps = [parameter(s, torch.bfloat16, 20 + k) for k, s in enumerate(shapes)]
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    a, b = (torch_ops.AdamW([(x[:2], 0.01, 0.1), (x[2:], 0.02, 0.0)], moment_bits=bits, stochastic_rounding=True, seed=5, capturable=True) for x in (ps, qs))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm-up outside the graph, with the states put back
        a.step(grad_scale=a.grad_norm(1.0))
        torch.cuda.synchronize()
    b.step(grad_scale=b.grad_norm(1.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = a.grad_norm(0.05)
        a.step(grad_scale=norm)
    for replay in range(6):
        if replay == 2:
            for o in (a, b):
                o.lr_factor.fill_(0.25)
        scale = float("inf") if replay == 4 else 0.5 + replay
        for p, q in zip(ps, qs):
            p.grad.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(replay)) * scale if scale < 1e9 else p.grad * scale)
            q.grad.copy_(p.grad)
        graph.replay()
        want = b.grad_norm(0.05)
        b.step(grad_scale=want)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) or (replay == 4 and not torch.isfinite(norm).any())
        for x, y in zip(ps + states(a), qs + states(b)):
            assert torch.equal(x, y), replay
        _ = torch.ones(1000, device="cuda").sum().item()
    assert a.steps() == [6] * 4 == b.steps() and a.device_step.item() == 6


def test_a_captured_step_needs_its_count_on_the_device():
    p = parameter((40,))
    opt = torch_ops.AdamW([([p], 0.01, 0.0)])
    opt.step()
    was, graph = p.detach().clone(), torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert opt.steps() == [1] and torch.equal(p, was)
    opt.step()
    torch.cuda.synchronize()
    assert opt.steps() == [2] and not torch.equal(p, was)


def test_a_captured_step_does_not_replace_gradients():
    """One that its elements share cannot be cleared in place."""
    p = parameter((40,), gradient=False)
    opt = torch_ops.AdamW([([p], 0.01, 0.0)], capturable=True)
    p.grad = torch.ones(1, device="cuda").expand(40)
    was, graph = p.detach().clone(), torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cleared"):
        with torch.cuda.graph(graph):
            opt.step(zero_grad=True)
    torch.cuda.synchronize()
    assert opt.steps() == [0] and torch.equal(p, was)
    opt.step(zero_grad=True)
    assert opt.steps() == [1] and not p.grad.any() and p.grad.is_contiguous() and not torch.equal(p, was)


def test_two_graphs_of_norms_side_by_side():
    """Each call has scratch memory of its own: two captured norms that run at once on two streams give what they give alone."""
    gs = [[torch.randn(300_001, generator=torch.Generator().manual_seed(k)).cuda(), torch.ones(77, device="cuda") * k] for k in (1, 2)]
    want = [torch_ops.grad_norm(g, 1.0).clone() for g in gs]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for g in gs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append([torch_ops.grad_norm(g, 1.0) for _ in range(8)])
    for _ in range(5):
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(x, w) for x in o)
            for x in o:
                x.zero_()


def test_steps_on_another_stream():
    p, q = (parameter((200_000,), seed=30) for _ in range(2))
    a, b = (torch_ops.AdamW([([x], 0.01, 0.0)], moment_bits=8) for x in (p, q))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        with torch.cuda.stream(side):
            a.step(grad_scale=a.grad_norm(1.0))
        b.step(grad_scale=b.grad_norm(1.0))
    torch.cuda.synchronize()
    assert torch.equal(p, q) and torch.equal(a.exp_avg, b.exp_avg)


def test_host_threads_side_by_side():
    """Each with parameters and a stream of its own: they end where they end one after the other."""
    def train(seed, ends):
        with torch.cuda.stream(torch.cuda.Stream()):
            ps = [parameter((n,), seed=seed + n, gradient=False) for n in (1000, 5, 300000)]
            opt = torch_ops.AdamW([(ps, 0.01, 0.1)], moment_bits=8, seed=seed)
            for k in range(60):
                for p in ps:
                    p.grad = p.detach() * 0.1 + k * 1e-3
                norm = opt.grad_norm(1.0)
                opt.step(True, norm)
            ends[seed] = [t.clone() for t in (*ps, *states(opt), norm)]
            torch.cuda.current_stream().synchronize()

    alone, together = {}, {}
    for seed in range(4):
        train(seed, alone)
    threads = [threading.Thread(target=train, args=(seed, together)) for seed in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in range(4):
        assert all(torch.equal(a, b) for a, b in zip(alone[seed], together[seed], strict=True)), seed


@pytest.mark.parametrize("bits", [32, 8])
def test_training_step_behind_the_rasterizer(bits):
    """Render, a small network in bf16 on the finest image, loss, backward, norm of all gradients, one step on descriptors, confidence,
    background and network together: each step is the definition's, with the gradients that autograd left."""
    scene = synthetic.tiny_scene(num_points=4000, K=8, seed=33)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    rng = np.random.default_rng(2)
    raw = [cu(rng.standard_normal(scene.texture.shape).astype(np.float32)), cu(np.array([0.2, -0.5, 0.7, -0.3], np.float32)),
           cu((0.2 * rng.standard_normal((1, scene.num_points))).astype(np.float32))]
    raw = [t.requires_grad_(True) for t in raw]
    net = [parameter((6, 4), torch.bfloat16, 40), parameter((6,), torch.bfloat16, 41), parameter((3, 6), torch.bfloat16, 42)]
    for p in net:
        p.grad = None
    opt = torch_ops.AdamW([([raw[0]], 0.01, 0.0), ([raw[1]], 0.0004, 0.0), ([raw[2]], 0.001, 0.0), (net, 1e-3, 0.05)], moment_bits=bits, master_weights=True, seed=8)
    rates = [(0.01, 0.0), (0.0004, 0.0), (0.001, 0.0)] + [(1e-3, 0.05)] * 3
    tangents = torch.zeros((scene.poses_se3.shape[0], 6), dtype=torch.float64, device="cuda")
    lay, max_norm = opt.layout(), 0.5
    for step in range(1, 4):
        outs = torch_ops.blend_point_cloud(raw[0], raw[1], cu(scene.position), tangents, cu(scene.intrinsics), raw[2], cu(scene.poses_se3), None,
                                           _views(scene), scene.num_layers, train=False, use_environment_map=0, need_point_gradient=0,
                                           drop_out_points_by_radius=0, debug_max_list_length=scene.max_list_length, fused_confidence_scale=10.0,
                                           fused_texture_abs=1)
        x = outs[0][0].flatten(1).t().to(torch.bfloat16)
        colours = torch.relu(x @ net[0].t() + net[1]) @ net[2].t()
        loss = (colours.float() - 0.3).square().mean() * 100 + sum(o.square().mean() for o in outs[1:])
        loss.backward()
        params = raw + net
        held = [opt.master[f:f + n] if p.dtype != torch.float32 else p.detach().reshape(-1) for (f, n), p in zip(lay, params)]
        before = [numbers(h).copy() for h in held]
        m0, v0 = (numbers(t).copy() for t in opt.moments())
        grads = [numbers(p.grad).reshape(-1) for p in params]
        assert all(np.isfinite(g).all() and g.any() for g in grads)
        norm = opt.grad_norm(max_norm)
        opt.step(zero_grad=True, grad_scale=norm)
        total = np.sqrt(sum((g ** 2).sum() for g in grads))
        got = numbers(norm)
        assert abs(got[0] - total) <= 2 * om.U * total and abs(got[1] - min(1.0, max_norm / total)) <= 2 * om.U
        for k, p in enumerate(params):
            f, n = lay[k]
            want, m, v, tol, tol_m, tol_v = om.step64(before[k], grads[k], m0[f:f + n], v0[f:f + n], step, *rates[k], scale=got[1])
            assert (np.abs(numbers(held[k]) - want) <= tol).all(), (step, k)
            if p.dtype != torch.float32:
                assert torch.equal(p.detach().reshape(-1), held[k].to(p.dtype))
            assert not p.grad.any()
    assert opt.steps() == [3] * 6


def test_kept_descriptors_notice_a_step():
    """Descriptor records that are kept across calls depend on the version counters, which a step moves."""
    scene = synthetic.tiny_scene(num_points=2000, K=8, seed=35)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    texture, confidence = cu(scene.texture), cu(scene.confidence.reshape(1, -1))
    tangents = torch.zeros((scene.poses_se3.shape[0], 6), dtype=torch.float64, device="cuda")

    def render(t, c):
        with torch.no_grad():
            return torch_ops.blend_point_cloud(t, cu(scene.background), cu(scene.position), tangents, cu(scene.intrinsics), c, cu(scene.poses_se3), None,
                                               _views(scene), scene.num_layers, use_environment_map=0, drop_out_points_by_radius=0,
                                               debug_max_list_length=scene.max_list_length)

    for _ in range(4):
        render(texture, confidence)
    texture.requires_grad_(True)
    texture.grad = torch.ones_like(texture)
    version = texture._version
    opt = torch_ops.AdamW([([texture], 0.1, 0.0)])
    opt.step()
    assert texture._version > version
    got = render(texture, confidence)
    want = render(texture.detach().clone(), confidence.clone())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
