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


# ---- parameters whose order in memory changes --------------------------------------------------------------------------

def channels_last(t):
    return t.contiguous(memory_format=torch.channels_last)


def turned(t):
    return t.transpose(0, 3).contiguous().transpose(0, 3)


def turn(p, order):
    """What net.to(memory_format=...) does: the same tensor object, with its elements and its gradient's in another order."""
    p.data = order(p.data)
    g, p.grad = p.grad, None
    p.grad = order(g)


def by_index(flat, p):
    """Elements in the order of p's memory, in the order of p's indices."""
    return flat.as_strided(p.shape, p.stride()).contiguous().reshape(-1)


@pytest.mark.parametrize("dtype,masters", [(torch.float32, False), (torch.bfloat16, True), (torch.bfloat16, False)], ids=["f32", "bf16 masters", "bf16"])
def test_state_follows_another_order_in_memory(dtype, masters):
    """A twin that keeps its order takes the same steps, before and after, there and back and over an order of its own; also where another
    parameter changes its size at the same time."""
    shapes = [(9,), (6, 5, 3, 4), (2, 3, 1, 5)]
    ps, qs = ([parameter(s, dtype, 90 + k) for k, s in enumerate(shapes)] for _ in range(2))
    a, b = (torch_ops.AdamW([(x, 0.01, 0.1)], master_weights=masters) for x in (ps, qs))
    for k, order in enumerate((torch.clone, channels_last, turned, channels_last, torch.Tensor.contiguous)):
        for p in ps[1:]:
            turn(p, order)
        if k == 2:
            for x in (ps, qs):
                grow(x[0], (1000,), 4)
        arrays = [t.data_ptr() for t in states(a)]
        for _ in range(2):
            a.step(zero_grad=False)
            b.step(zero_grad=False)
        assert k == 2 or arrays == [t.data_ptr() for t in states(a)]
        assert a.layout() == b.layout() and a.steps() == b.steps()
        for p, q, (f, n) in zip(ps, qs, a.layout()):
            assert torch.equal(p, q)
            for x, y in zip(states(a), states(b)):
                assert torch.equal(by_index(x[f:f + n], p), by_index(y[f:f + n], q)) and x[f:f + n].any()
            p.grad.mul_(-0.7)
            q.grad.mul_(-0.7)


@pytest.mark.parametrize("masters", [False, True])
def test_codes_follow_another_order_in_memory(masters):
    """Their blocks get other elements: moments are within half a code of what they were, and the step is the definition's from there."""
    dtype = torch.bfloat16 if masters else torch.float32
    p = parameter((16, 5, 3, 4), dtype, 95)
    opt = torch_ops.AdamW([([p], 0.01, 0.1)], moment_bits=8, master_weights=masters, seed=2)
    for _ in range(2):
        opt.step()
    was = [by_index(t, p) for t in opt.moments()]
    turn(p, channels_last)
    m, v = opt.moments()
    unit = np.exp2(numbers(opt.block_scale) - 127.0)
    for k, (x, y) in enumerate(zip((m, v), was)):
        want = numbers(torch.empty_like(p, dtype=torch.float32).copy_(y.view(p.shape)).permute(0, 2, 3, 1).reshape(-1))
        u = np.repeat(unit[:, k], 128)[:960]
        assert (np.abs(numbers(x)[:960] - want) <= (np.abs(want) + u) / 16 * 1.0001 + (u / 8 if k else 0)).all() and not x[960:].any()
    memory = lambda t: t.detach().permute(0, 2, 3, 1).reshape(-1)  # noqa: E731
    held_p = (opt.master[:960] if masters else memory(p)).clone()
    want, *_, tol, _, _ = om.step64(numbers(held_p), numbers(memory(p.grad)), numbers(m)[:960], numbers(v)[:960], 3, 0.01, 0.1)
    opt.step()
    held_p = opt.master[:960] if masters else memory(p)
    assert (np.abs(numbers(held_p) - want) <= tol).all()
    assert not masters or torch.equal(memory(p), held_p.to(dtype))


@pytest.mark.parametrize("bits", [32, 8])
def test_orders_that_are_one_move_nothing(bits):
    """Strides of dimensions of one element, and shapes of contiguous parameters."""
    p = parameter((40, 7, 1, 1), seed=96)
    opt = torch_ops.AdamW([([p], 0.01)], moment_bits=bits)
    opt.step()
    was = [t.clone() for t in states(opt)]
    for data in (channels_last(p.data), p.data.as_strided(p.shape, (7, 1, 5, 9)), p.data.reshape(7, 40), p.data.reshape(-1), p.data.reshape(4, 7, 2, 5)):
        p.data = data
        opt.moments()
        assert all(torch.equal(x, y) for x, y in zip(was, states(opt)))
    p.grad = None
    p.grad = torch.ones_like(p)
    turn(p, channels_last)
    opt.step()
    assert opt.steps() == [2]


@pytest.mark.parametrize("bits", [32, 8])
def test_another_shape_in_another_order_is_refused(bits):
    p = parameter((5, 3), seed=97)
    opt = torch_ops.AdamW([([p], 0.01)], moment_bits=bits)
    opt.step()
    before, data, grad = held(opt), p.data, p.grad
    p.grad = None
    p.data = data.t()
    p.grad = grad.t()
    was = p.detach().clone()
    for call in (opt.step, opt.moments, lambda: opt.load_moments([grad], [grad], 1)):
        with pytest.raises(RuntimeError, match="shape and the order"):
            call()
    assert torch.equal(p, was) and same(before, held(opt))
    p.grad = None
    p.data = data
    p.grad = grad
    opt.step()
    assert opt.steps() == [2]


def test_masters_and_moments_are_taken_over_in_the_present_order():
    p = parameter((6, 5, 3, 4), torch.bfloat16, 98)
    opt = torch_ops.AdamW([([p], 0.01)], master_weights=True)
    opt.step()
    turn(p, channels_last)
    opt.reload_master()
    memory = p.detach().permute(0, 2, 3, 1).reshape(-1)
    assert torch.equal(opt.master[:360], memory.float())
    m, v = torch.rand(6, 5, 3, 4, device="cuda"), torch.rand(6, 5, 3, 4, device="cuda")
    turn(p, torch.Tensor.contiguous)
    opt.load_moments([m], [v], 4)
    assert torch.equal(opt.exp_avg[:360], m.reshape(-1)) and torch.equal(opt.exp_avg_sq[:360], v.reshape(-1))
    assert torch.equal(opt.master[:360], p.detach().float().reshape(-1))


def test_a_captured_step_needs_the_order_that_it_found():
    """With the count on the device the state follows in place, but not inside a graph, which would turn it again with every replay."""
    p, q = (parameter((6, 5, 3, 4), seed=99) for _ in range(2))
    a, b = (torch_ops.AdamW([([x], 0.01)], capturable=True) for x in (p, q))
    a.step()
    b.step()
    turn(p, channels_last)
    before, was = held(a), p.detach().clone()
    with pytest.raises(RuntimeError, match="order in memory"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            a.step()
    torch.cuda.synchronize()
    assert same(before, held(a)) and torch.equal(p, was)
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(4):
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q)
        _ = torch.ones(1000, device="cuda").sum().item()
    assert a.steps() == b.steps() == [6]


# ---- counts ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("by_moments", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_run_is_taken_up_with_every_parameters_count(bits, by_moments):
    """After points were added one parameter is younger than the others, and one had no gradient at first: a run that is taken up from what
    was saved goes on as the one that was never stopped."""
    bits_of_copy = 32 if by_moments else bits  # float32 moments of an 8-bit run continue in 32 bits
    ps = [parameter((4, 300), seed=110), parameter((77,), seed=111), parameter((6, 5), seed=112, gradient=False)]
    opt = torch_ops.AdamW([(ps[:1], 0.01), (ps[1:], 0.02, 0.1)], moment_bits=bits, seed=6)
    for _ in range(5):
        opt.step()
    grow(ps[0], (4, 450), 5)
    ps[2].grad = torch.ones_like(ps[2])
    opt.step()
    opt.step()
    saved = opt.steps()
    assert saved == [2, 7, 2]
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    copy = torch_ops.AdamW([(qs[:1], 0.01), (qs[1:], 0.02, 0.1)], moment_bits=bits_of_copy, seed=6)
    if by_moments:
        ms = [t.clone() for t in opt.moments()]
        copy.load_moments(*([t[f:f + n] for f, n in opt.layout()] for t in ms), saved)
    else:
        for x, y in zip(states(copy), states(opt), strict=True):
            x.copy_(y)
        copy.set_step(saved)
    assert copy.steps() == saved
    before = [numbers(p).reshape(-1) for p in ps]
    m, v = (numbers(t) for t in opt.moments())
    lay = opt.layout()
    opt.step()
    copy.step()
    assert opt.steps() == copy.steps() == [3, 8, 3]
    for k, (p, q, (f, n)) in enumerate(zip(ps, qs, lay)):
        rates = (0.01, 0.0) if k == 0 else (0.02, 0.1)
        want, *_, tol, _, _ = om.step64(before[k], numbers(p.grad).reshape(-1), m[f:f + n], v[f:f + n], saved[k] + 1, *rates)
        for x in (p, q):
            assert (np.abs(numbers(x).reshape(-1) - want) <= tol).all()
        assert bits != bits_of_copy or torch.equal(p, q)
    assert bits != bits_of_copy or all(torch.equal(x, y) for x, y in zip(states(opt), states(copy)))


def test_counts_are_checked():
    ps = [parameter((30,), seed=113), parameter((5,), seed=114)]
    ms = [torch.rand(30, device="cuda"), torch.rand(5, device="cuda")]
    opt, fixed = (torch_ops.AdamW([(ps, 0.01)], capturable=c) for c in (False, True))
    for o, bad in ((opt, [3]), (opt, []), (opt, [1, 2, 3]), (opt, [1, -1]), (fixed, [1, 2]), (fixed, [3]), (fixed, [-1, -1])):
        for call in (lambda: o.set_step(bad), lambda: o.load_moments(ms, ms, bad)):
            with pytest.raises(RuntimeError, match="count"):
                call()
        assert o.steps() == [0, 0] and not o.exp_avg.any() and not o.exp_avg_sq.any()
    fixed.set_step([4, 4])
    assert fixed.steps() == [4, 4] and fixed.device_step.item() == 4
    fixed.load_moments(ms, ms, [6, 6])
    opt.load_moments(ms, ms, [6, 0])
    assert fixed.steps() == [6, 6] and opt.steps() == [6, 0] and torch.equal(opt.exp_avg, fixed.exp_avg) and opt.exp_avg.any()
    opt.set_step(2)
    assert opt.steps() == [2, 2]


def test_more_counts_than_groups_are_refused():
    """Parameters of one group with counts of their own."""
    ps = [torch.zeros(1, device="cuda", requires_grad=True) for _ in range(1025)]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = torch_ops.AdamW([(ps, 0.5)])
    opt.set_step(list(range(1025)))
    with pytest.raises(RuntimeError, match="1025 groups"):
        opt.step()
    assert opt.steps() == list(range(1025)) and not any(p.any() for p in ps) and not opt.exp_avg.any()
    opt.set_step([0, 0] + list(range(2, 1025)))
    opt.step()
    assert opt.steps() == [1, 1] + list(range(3, 1026)) and ps[0].item() == ps[1].item() == pytest.approx(-0.5)


# ---- parts of the state ------------------------------------------------------------------------------------------------

def test_one_parameters_moments_are_read():
    """Its codes and scales, which lie anywhere in the flat arrays."""
    ms, vs = ([torch.rand(n, device="cuda") for n in (100, 300, 0, 1000, 1)] for _ in range(2))
    codes = torch_ops.pack_moments(ms, vs)
    whole, first = torch_ops.unpack_moments(*codes), 0
    for x in ms:
        end = first + -(-x.numel() // 128) * 128
        part = torch_ops.unpack_moments(codes[0][first:end], codes[1][first:end], codes[2][first // 128:end // 128])
        for a, b in zip(part, whole):
            assert torch.equal(a, b[first:end])
        first = end
    moved = []  # at addresses of any byte
    for t in codes:
        moved.append(torch.zeros(t.numel() + 7, dtype=torch.uint8, device="cuda")[7:].view(t.shape).copy_(t))
    assert all(torch.equal(a, b) for a, b in zip(torch_ops.unpack_moments(*moved), whole))


# ---- streams -----------------------------------------------------------------------------------------------------------

def test_norms_on_a_foreign_stream_keep_nothing():
    """The handle of a stream that somebody else made may come back as another stream's: nothing is kept by it."""
    gs = [torch.randn(300_001, device="cuda"), torch.ones(77, device="cuda")]
    want = torch_ops.grad_norm(gs, 1.0)
    for pooled in [torch.cuda.Stream() for _ in range(3)]:  # kept alive; foreign to torch in the second form
        stream = torch.cuda.ExternalStream(pooled.cuda_stream)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        for _ in range(3):
            with torch.cuda.stream(stream):
                got = torch_ops.grad_norm(gs, 1.0)
            stream.synchronize()
            assert torch.equal(got, want)
        del got
        assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["freed with the object", "left for larger ones"])
def test_state_that_another_stream_uses_is_not_given_out(bits, how):
    """The optimiser was made on one stream and steps on another, which has not come to the step yet when the state is freed: its memory
    is not handed out on the first stream meanwhile."""
    p = parameter((3_000_001,), torch.bfloat16, 120)
    opt = torch_ops.AdamW([([p], 0.01)], moment_bits=bits, master_weights=True, capturable=how == "freed with the object")
    sizes = [(t.shape, t.dtype, t.data_ptr()) for t in states(opt)]
    larger = torch.ones(5_000_000, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        if how == "freed with the object":
            opt.step()
            del opt
        else:
            p.data = larger
            p.grad = None
            p.grad = larger
            opt.step()
    busy = not side.query()
    made = [torch.empty(shape, dtype=dtype, device="cuda") for shape, dtype, _ in sizes]
    busy = busy and not side.query()
    torch.cuda.synchronize()
    assert busy and not {t.data_ptr() for t in made} & {address for *_, address in sizes}


def test_an_optimiser_goes_from_stream_to_stream():
    """With a wait in between, it steps as on one, captured or not."""
    p, q = (parameter((100_000,), seed=121) for _ in range(2))
    a, b = (torch_ops.AdamW([([x], 0.01)], moment_bits=8, capturable=True) for x in (p, q))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for k in range(9):
        now, last = streams[k % 3], streams[(k - 1) % 3] if k else torch.cuda.current_stream()
        now.wait_stream(last)
        with torch.cuda.stream(now):
            a.step()
    torch.cuda.current_stream().wait_stream(streams[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    for _ in range(12):
        b.step()
    assert a.steps() == b.steps() == [12]
    assert torch.equal(p, q) and all(torch.equal(x, y) for x, y in zip(states(a), states(b)))


def test_moments_come_in_pairs():
    p = parameter((30,), seed=130)
    opt = torch_ops.AdamW([([p], 0.01)])
    ms = [torch.rand(30, device="cuda") for _ in range(2)]
    for first, second in ((ms[:1], ms), (ms, ms[:1]), (ms[:1], [])):
        with pytest.raises(RuntimeError, match="moments"):
            opt.load_moments(first, second, 1)
        assert opt.steps() == [0] and not opt.exp_avg.any()


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_of_a_parameter_with_gaps_are_refused(bits):
    """It has no order in memory that they could be taken over in."""
    p = parameter((6, 5, 3, 4), seed=131)
    opt = torch_ops.AdamW([([p], 0.01)], moment_bits=bits)
    was, before = p.data, held(opt)
    p.data = torch.zeros(6, 5, 3, 8, device="cuda")[..., ::2]
    for x in (torch.rand(6, 5, 3, 4, device="cuda"), torch.rand(360, device="cuda")):
        with pytest.raises(RuntimeError, match="dense"):
            opt.load_moments([x], [x], 1)
        assert same(before, held(opt))
    p.data = was
    opt.load_moments([torch.rand(6, 5, 3, 4, device="cuda")], [torch.rand(360, device="cuda").view(6, 5, 3, 4)], 1)
    assert opt.steps() == [1]


def test_state_is_not_laid_out_in_a_captured_call():
    """It would lie in the graph's memory, and be filled by replays only."""
    p = parameter((30,), seed=132)
    opt = torch_ops.AdamW([([p], 0.01)])
    opt.step()
    grow(p, (50,), 6)
    before, ms = held(opt), [torch.rand(50, device="cuda")]
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.load_moments(ms, ms, 3)
    torch.cuda.synchronize()
    assert same(before, held(opt))
    opt.load_moments(ms, ms, 3)
    assert opt.steps() == [3] and opt.layout() == [(0, 50)] and torch.equal(opt.exp_avg[:50], ms[0])


def test_a_parameter_without_a_gradient_may_change_shape_and_order():
    """It stops no step of the others, and is refused once it is to be stepped."""
    p, frozen = parameter((5, 3), seed=133), parameter((7, 4), seed=134, gradient=False)
    opt = torch_ops.AdamW([([p, frozen], 0.01)])
    opt.step()
    frozen.data = frozen.data.t()
    opt.step()
    opt.moments()
    assert opt.steps() == [2, 0]
    frozen.grad = torch.ones_like(frozen)
    with pytest.raises(RuntimeError, match="shape and the order"):
        opt.step()
    assert opt.steps() == [2, 0]
    frozen.grad = None
    frozen.data = frozen.data.t()
    frozen.grad = torch.ones_like(frozen)
    opt.step()
    assert opt.steps() == [3, 1]
