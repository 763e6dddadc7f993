"""The AdamW step over lists of tensors, gradient norms and moments in 8 bits, through the C ABI, against plain implementations in 64
bits. Codes of 8-bit moments are held bit by bit: their arithmetic is products and sums in a documented order and integers."""
import numpy as np
import pytest
import torch

from tests import optim_model as om
from vet_amd import abi

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [0, 1, 2, 7, 8, 9, 127, 128, 129, 255, 1000, 2047, 2048, 2049, 4096, 5001, 40_007]


class Guarded:
    """A tensor inside a larger one: `at` elements behind an aligned address, with neighbours that have to stay as they were."""

    def __init__(self, values, dtype, at=0, room=None):
        room = values.size if room is None else room
        self.at, self.n = 16 + at, room
        self.whole = torch.full((room + at + 64,), 3, dtype=dtype, device="cuda")
        self.t = self.whole[self.at:self.at + room]
        self.t[:values.size].copy_(torch.from_numpy(np.ascontiguousarray(values)))

    def check(self):
        assert (self.whole[:self.at] == 3).all() and (self.whole[self.at + self.n:] == 3).all()


def gradients(rng, n, dtype):
    """Over many decades, with zeros and, in float32, values whose square underflows."""
    g = rng.standard_normal(n) * np.exp(rng.normal(-4, 2, n))
    g[rng.random(n) < 0.1] = 0.0
    if dtype == torch.float32:
        g[rng.random(n) < 0.02] *= 1e-22
        g[rng.random(n) < 0.02] *= 1e9
    return torch.from_numpy(g).to(dtype)


def numbers(t):
    return t.detach().cpu().double().numpy()


def make(rng, n, k, param, grad, bits, copy=None, group=0, number=0):
    """A tensor of the list with its state, odd ones of them unaligned, and what the model starts from."""
    off = [0, 1, 3, 0][k % 4]
    p = torch.from_numpy(rng.standard_normal(n) * 0.1).to(param)
    g = gradients(rng, n, grad)
    spread = np.exp(rng.normal(-4, 2, n))
    m, v = (0.2 * spread * rng.standard_normal(n)).astype(np.float32), (spread ** 2 * rng.random(n)).astype(np.float32)
    m[v < 1e-30] = 0
    if k % 3 == 0:
        m[:], v[:] = 0, 0  # a first step
    d = {"param": Guarded(p.double().numpy(), param, off), "grad": Guarded(g.double().numpy(), grad, off)}
    if bits == 32:
        d["exp_avg"], d["exp_avg_sq"] = Guarded(m, torch.float32, off), Guarded(v, torch.float32, off)
    else:
        rm, rv, _ = om.random_bits(5, 1, 0, n)
        mc, vc, scale = om.encode(m, v, rm, rv)
        d["exp_avg"], d["exp_avg_sq"] = Guarded(mc, torch.uint8, 8), Guarded(vc, torch.uint8, 8)
        d["block_scale"] = Guarded(scale.reshape(-1), torch.uint8, 2)
        m, v = (x[:n].astype(np.float32) for x in om.decode(mc, vc, scale))
    if copy is not None:
        d["copy"] = Guarded(np.zeros(n), copy, off)
    start = dict(p=numbers(d["param"].t), g=numbers(d["grad"].t), m=m, v=v)
    return d, start, dict(group=group, first_number=number)


def as_list(made):
    return [{**{k: x.t for k, x in d.items()}, **rest} for d, _, rest in made]


def compare(made, groups, seed=0, bits=32, stochastic=False, scale=1.0, beta1=0.9, beta2=0.999, eps=1e-8):
    for d, s, rest in made:
        lr, decay, step = groups[rest["group"]]
        n = s["p"].size
        for x in d.values():
            x.check()
        if n == 0:
            continue
        p, m, v, tol_p, tol_m, tol_v = om.step64(s["p"], s["g"], s["m"], s["v"], step, lr, decay, beta1, beta2, eps, scale)
        got, half = numbers(d["param"].t), HALF_STEP[d["param"].t.dtype]
        if stochastic and d["param"].t.dtype == torch.bfloat16:
            half *= 2  # up or down, not to the nearest
        tol = tol_p * (1 + 2 * half) + half * np.abs(p) + (2.0 ** -25 if d["param"].t.dtype == torch.float16 else 0)
        assert (np.abs(got - p) <= tol).all(), (n, np.max(np.abs(got - p) / tol))
        if "copy" in d:
            want = d["param"].t.to(d["copy"].t.dtype)
            assert torch.equal(d["copy"].t, want)
        if bits == 32:
            assert (np.abs(numbers(d["exp_avg"].t) - m) <= tol_m).all() and (np.abs(numbers(d["exp_avg_sq"].t) - v) <= tol_v).all()
        else:
            fm, fv = om.moments_in_float(s["m"], s["v"], s["g"], beta1, beta2, scale)
            assert (np.abs(fm - m) <= tol_m).all() and (np.abs(fv - v) <= tol_v).all()
            rm, rv, _ = om.random_bits(seed, step, rest["first_number"], n)
            mc, vc, sc = om.encode(fm, fv, rm, rv)
            np.testing.assert_array_equal(d["exp_avg"].t.cpu().numpy(), mc)
            np.testing.assert_array_equal(d["exp_avg_sq"].t.cpu().numpy(), vc)
            np.testing.assert_array_equal(d["block_scale"].t.cpu().numpy().reshape(-1, 2), sc)


TYPES = [(torch.float32, torch.float32, None), (torch.float32, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16, torch.float16),
         (torch.bfloat16, torch.bfloat16, None), (torch.bfloat16, torch.float32, None), (torch.float16, torch.float16, None),
         (torch.float32, torch.float32, torch.bfloat16), (torch.float16, torch.bfloat16, None), (torch.bfloat16, torch.float16, None),
         (torch.float16, torch.float32, None)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad,copy", TYPES, ids=lambda t: str(t).replace("torch.", ""))
def test_step_against_64_bits(bits, param, grad, copy, rasterizer):
    rng = np.random.default_rng(3)
    groups = [(0.01, 0.1, 7), (0.002, 0.0, 400)]
    made, number = [], 0
    for k, n in enumerate(SIZES):
        made.append(make(rng, n, k, param, grad, bits, copy, group=k % 2, number=number))
        number += -(-n // 128) * 128
    scale = torch.tensor([0.25], device="cuda")
    rasterizer.adamw_step(as_list(made), groups, moment_bits=bits, seed=11, grad_scale=scale)
    compare(made, groups, 11, bits, scale=0.25)
    for d, s, _ in made:
        assert np.array_equal(numbers(d["grad"].t), s["g"])  # gradients are read only
    rasterizer.adamw_step(as_list(made), [(0.0, 0.0, 2)] * 2, moment_bits=bits, zero_grad=True)
    for d, s, _ in made:
        assert not d["grad"].t.any()
        d["grad"].check()


@pytest.mark.parametrize("bits", [32, 8])
def test_bf16_parameters_are_rounded_by_random_bits(bits, rasterizer):
    """Exactly between two neighbours in a known share of cases: the parameter is the one the random bits say."""
    rng = np.random.default_rng(5)
    made = [make(rng, n, k, torch.bfloat16, torch.bfloat16, bits, number=128 * 40 * k) for k, n in enumerate([5001, 128, 3])]
    for d, _, _ in made:
        d["param"].t[::7] = float("inf")
        d["param"].t[1::7] = float("nan")
    made = [(d, dict(s, p=numbers(d["param"].t)), r) for d, s, r in made]
    rasterizer.adamw_step(as_list(made), [(1e-3, 0.0, 9)], moment_bits=bits, seed=3, stochastic_rounding=True)
    for d, s, rest in made:
        got = numbers(d["param"].t)
        finite = np.isfinite(s["p"])
        assert np.array_equal(got[~finite], s["p"][~finite], equal_nan=True)
        want, *_, = om.step64(s["p"], s["g"], s["m"], s["v"], 9, 1e-3)
        rp = om.random_bits(3, 9, rest["first_number"], got.size)[2]
        with np.errstate(invalid="ignore"):
            up = om.floats_of((om.bits_of(want) + rp) & ~0xFFFF)
        # float32 arithmetic may put an element on the other side of its border where the random bits come within its error of it
        off = finite & (up != got)
        assert off.mean() <= 1e-3 and (np.abs(got - want)[finite] <= 2.0 ** -7 * np.abs(want[finite]) + 1e-6).all()


def test_random_rounding_keeps_means(rasterizer):
    """The mean over many seeds of what codes and bf16 parameters stand for is the value itself, to six standard errors of a
    rounding by at most a step. Elements have to differ in their random bits, as seeds and steps have."""
    rng = np.random.default_rng(7)
    n, seeds = 1024, 400
    p0 = torch.from_numpy(rng.standard_normal(n)).to(torch.bfloat16).cuda()
    g = torch.from_numpy(rng.standard_normal(n) * np.exp(rng.normal(0, 1, n))).float().cuda()
    total = {k: np.zeros(n) for k in "pmv"}
    seen = set()
    for seed in range(seeds):
        d = dict(param=p0.clone(), grad=g, exp_avg=torch.zeros(n, dtype=torch.uint8, device="cuda"),
                 exp_avg_sq=torch.zeros(n, dtype=torch.uint8, device="cuda"), block_scale=torch.zeros(n // 128 * 2, dtype=torch.uint8, device="cuda"))
        rasterizer.adamw_step([d], [(1e-3, 0.0, 1)], moment_bits=8, stochastic_rounding=True, seed=seed)
        m, v = om.decode(d["exp_avg"].cpu().numpy(), d["exp_avg_sq"].cpu().numpy(), d["block_scale"].cpu().numpy().reshape(-1, 2))
        seen.add(d["exp_avg"].cpu().numpy().tobytes())
        for k, x in (("p", numbers(d["param"])), ("m", m), ("v", v)):
            total[k] += x
    assert len(seen) == seeds
    want = om.step64(numbers(p0), numbers(g), np.zeros(n), np.zeros(n), 1, 1e-3)
    scale = d["block_scale"].cpu().numpy().reshape(-1, 2).astype(np.float64)
    for k, x, unit in (("p", want[0], None), ("m", want[1], np.exp2(scale[:, 0] - 127)), ("v", want[2], np.exp2(scale[:, 1] - 127))):
        # steps: 2^-7 of the parameter's binade; an eighth of (value + unit)
        step = 2.0 ** -7 * np.abs(x) * 2 if unit is None else (np.abs(x) + np.repeat(unit, 128)) / 8 * 1.001
        if k == "v":
            smallest = np.repeat(unit, 128) / 8
            keep = x >= smallest  # smaller ones are rounded up, on purpose
        else:
            keep = np.ones(n, bool)
        error = np.abs(total[k] / seeds - x)
        assert (error <= 6 * step / 2 / np.sqrt(seeds) + 1e-6 * np.abs(x) + 1e-12)[keep].all(), k


def test_second_moments_above_zero_stay_above_zero(rasterizer):
    n = 256
    g = torch.full((n,), 1e-12, device="cuda")
    g[0] = 1.0
    g[5], g[200:] = 0.0, 0.0
    for seed in range(20):
        d = dict(param=torch.zeros(n, device="cuda"), grad=g, exp_avg=torch.zeros(n, dtype=torch.uint8, device="cuda"),
                 exp_avg_sq=torch.zeros(n, dtype=torch.uint8, device="cuda"), block_scale=torch.zeros(4, dtype=torch.uint8, device="cuda"))
        rasterizer.adamw_step([d], [(1e-3, 0.0, 1)], moment_bits=8, seed=seed)
        assert torch.equal(d["exp_avg_sq"] > 0, g != 0)


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite(bits, rasterizer):
    """In 32 bits an element keeps its own NaN or infinity; in 8 bits its block of 128 reads as NaN, the others go on."""
    rng = np.random.default_rng(8)
    made = [make(rng, 128 * 5 + 9, 0, torch.float32, torch.float32, bits)]
    d, s, _ = made[0]
    bad = {3: np.nan, 130: np.inf, 300: -np.inf, 128 * 5 + 8: np.nan}
    for k, x in bad.items():
        d["grad"].t[k] = x
    rasterizer.adamw_step(as_list(made), [(0.01, 0.0, 4)], moment_bits=bits)
    m, v = (numbers(d[k].t) for k in ("exp_avg", "exp_avg_sq"))
    if bits == 8:
        m, v = om.decode(*(d[k].t.cpu().numpy() for k in ("exp_avg", "exp_avg_sq")), d["block_scale"].t.cpu().numpy().reshape(-1, 2))
        lost = np.isin(np.arange(m.size) // 128, [k // 128 for k in bad])
    else:
        lost = np.isin(np.arange(m.size), list(bad))
    assert np.array_equal(~np.isfinite(m), lost) and np.array_equal(~np.isfinite(v), lost)
    p = numbers(d["param"].t)
    assert np.isfinite(p[~np.isin(np.arange(p.size), list(bad))]).all()
    # a second step reads what the first left
    d["grad"].t.fill_(0.5)
    rasterizer.adamw_step(as_list(made), [(0.01, 0.0, 5)], moment_bits=bits)
    p = numbers(d["param"].t)
    assert np.array_equal(np.isnan(p) | np.isinf(p), lost[:p.size] if bits == 8 else lost)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_step_whose_factor_is_not_finite_is_left_out(bits, value, rasterizer):
    rng = np.random.default_rng(9)
    made = [make(rng, n, k, torch.float32, torch.bfloat16, bits, torch.bfloat16) for k, n in enumerate([5001, 3, 700])]
    before = [{k: x.whole.clone() for k, x in d.items()} for d, _, _ in made]
    rasterizer.adamw_step(as_list(made), [(0.01, 0.1, 4)], moment_bits=bits, grad_scale=torch.tensor([value], device="cuda"))
    for (d, _, _), b in zip(made, before):
        assert all(torch.equal(x.whole, b[k]) for k, x in d.items())
    rasterizer.adamw_step(as_list(made), [(0.01, 0.1, 4)], moment_bits=bits, grad_scale=torch.tensor([value], device="cuda"), zero_grad=True)
    for (d, _, _), b in zip(made, before):
        assert all(torch.equal(x.whole, b[k]) for k, x in d.items() if k != "grad") and not d["grad"].t.any()
        d["grad"].check()


@pytest.mark.parametrize("bits", [32, 8])
def test_long_lists_many_groups_and_mixed_types(bits, rasterizer):
    """More tensors and groups than a launch takes, every combination of types, empty tensors among them."""
    rng = np.random.default_rng(10)
    groups = [(1e-3 * (k + 1), 0.01 * k, k + 1) for k in range(23)]
    made, number = [], 0
    for k in range(331):
        n = int(rng.integers(0, 300)) if k % 5 else int(rng.integers(0, 9000))
        param, grad, copy = TYPES[int(rng.integers(len(TYPES)))]
        made.append(make(rng, n, k, param, grad, bits, copy, group=int(rng.integers(23)) if k % 2 else k % 3, number=number))
        number += -(-n // 128) * 128
    rasterizer.adamw_step(as_list(made), groups, moment_bits=bits, seed=1 << 63, beta1=0.8, beta2=0.99, eps=1e-6)
    compare(made, groups, 1 << 63, bits, beta1=0.8, beta2=0.99, eps=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_betas_of_zero(bits, rasterizer):
    rng = np.random.default_rng(12)
    made = [make(rng, n, k, torch.float32, torch.float32, bits) for k, n in enumerate([1000, 77])]
    rasterizer.adamw_step(as_list(made), [(0.01, 0.0, 1)], moment_bits=bits, beta1=0.0, beta2=0.0, seed=2)
    compare(made, [(0.01, 0.0, 1)], 2, bits, beta1=0.0, beta2=0.0)


def test_random_numbers_wrap(rasterizer):
    """A tensor far up in the stream of random bits, across the place where its 2^33 numbers begin again."""
    rng = np.random.default_rng(13)
    made = [make(rng, 1000, 0, torch.float32, torch.float32, 8, number=(1 << 33) - 512), make(rng, 300, 0, torch.float32, torch.float32, 8, number=1 << 40)]
    rasterizer.adamw_step(as_list(made), [(0.01, 0.0, 6)], moment_bits=8, seed=4)
    compare(made, [(0.01, 0.0, 6)], 4, 8)


def test_a_tensor_of_several_entries(rasterizer):
    """More elements than places of 32 bits in a launch's entry are given: every part as a tensor of its own has it."""
    n = (1 << 30) + (1 << 22) + 77
    gen = torch.Generator("cuda").manual_seed(1)
    g = torch.empty(n, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    whole = -(-n // 128) * 128
    m, v = torch.zeros(whole, dtype=torch.uint8, device="cuda"), torch.zeros(whole, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(whole // 128 * 2, dtype=torch.uint8, device="cuda")
    rasterizer.adamw_step([dict(param=p, grad=g, exp_avg=m, exp_avg_sq=v, block_scale=scale)], [(1e-3, 0.0, 1)], moment_bits=8, stochastic_rounding=True, seed=9)
    for first, end in ((0, 5000), ((1 << 30) - 1280, (1 << 30) + 2560), (n - 77 - 128 * 9, n)):
        k = -(-(end - first) // 128) * 128
        d = dict(param=torch.zeros(end - first, dtype=torch.bfloat16, device="cuda"), grad=g[first:end].clone(), first_number=first,
                 exp_avg=torch.zeros(k, dtype=torch.uint8, device="cuda"), exp_avg_sq=torch.zeros(k, dtype=torch.uint8, device="cuda"),
                 block_scale=torch.zeros(k // 64, dtype=torch.uint8, device="cuda"))
        rasterizer.adamw_step([d], [(1e-3, 0.0, 1)], moment_bits=8, stochastic_rounding=True, seed=9)
        f = first // 128 * 128
        assert torch.equal(d["param"][f - first:], p[f:end]) and d["param"].any()
        if first % 128 == 0:
            b = k if end == n else (end - first) // 128 * 128
            assert torch.equal(d["exp_avg"][:b], m[first:first + b]) and torch.equal(d["exp_avg_sq"][:b], v[first:first + b])
            assert torch.equal(d["block_scale"][:b // 64], scale[first // 64:first // 64 + b // 64])
    # and its norm: a sum of squares of float32 ones at known places, among zeros
    del p, m, v, scale
    g.zero_()
    at = torch.tensor([0, 1, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, n - 1], device="cuda")
    g[at] = 3.0
    assert rasterizer.gradient_norm([g]).cpu()[0].item() == np.float32(3.0 * np.sqrt(6.0))


# ---- steps whose count lies on the device ------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("num_groups", [1, 9, 300])
def test_the_count_on_the_device_is_the_same_step(bits, num_groups, rasterizer):
    rng = np.random.default_rng(14)
    made = [make(rng, n, k, torch.float32, torch.float32, bits, group=k * 7 % num_groups, number=1280 * k) for k, n in enumerate([1000, 1, 0, 500, 129] * 4)]
    plain = [{k: x.t.clone() if isinstance(x, Guarded) else x for k, x in {**d, **r}.items()} for d, _, r in made]
    state = torch.zeros(rasterizer.lib.vetrast_adamw_device_state_bytes(num_groups), dtype=torch.uint8, device="cuda")
    state[:8].view(torch.int64).fill_(41)
    state[8:12].view(torch.float32).fill_(0.5)
    lrs = [0.01 * (k % 5 + 1) for k in range(num_groups)]
    for step in (42, 43):
        scale = torch.tensor([0.5], device="cuda")
        rasterizer.adamw_step(as_list(made), [(lr, 0.1, 0) for lr in lrs], moment_bits=bits, seed=6, device_state=state, grad_scale=scale)
        rasterizer.adamw_step(plain, [(0.5 * lr, 0.1, step) for lr in lrs], moment_bits=bits, seed=6, grad_scale=scale)
        assert state[:8].view(torch.int64).item() == step
        for a, b in zip(as_list(made), plain):
            for k in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(a[k], b[k])
            # pow on the device and on the host may differ in their last bits: the two constants by a rounding each
            x, y = numbers(a["param"]), numbers(b["param"])
            assert (np.abs(x - y) <= 4 * om.U * (np.abs(y) + 0.05)).all()
            a["param"].copy_(b["param"])
    # a step that is left out is not counted
    rasterizer.adamw_step(as_list(made), [(lr, 0.1, 0) for lr in lrs], moment_bits=bits, device_state=state, grad_scale=torch.tensor([np.inf], device="cuda"))
    assert state[:8].view(torch.int64).item() == 43
    rasterizer.adamw_step([], [], moment_bits=bits, device_state=state)
    assert state[:8].view(torch.int64).item() == 44


# ---- norms -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", [[0], [1], [7, 0, 9], SIZES, [3] * 401, [1_000_003], [2_500_000, 5, 300_001]],
                         ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_against_64_bits(dtype, sizes, rasterizer):
    rng = np.random.default_rng(15)
    made = [Guarded(gradients(rng, n, dtype).double().numpy(), dtype, k % 3) for k, n in enumerate(sizes)]
    want = np.sqrt(sum((numbers(g.t) ** 2).sum() for g in made))
    for max_norm, scale in ((0.0, 1.0), (0.5 * want, 0.125), (1e9, -2.0), (np.inf, 1.0)):
        got = numbers(rasterizer.gradient_norm([g.t for g in made], max_norm, scale))
        norm = abs(scale) * want
        factor = scale * min(1.0, max_norm / norm) if max_norm > 0 and norm > 0 else scale
        # sums in 64 bits are off by 2^-53 a term; what is left is the rounding to float32
        assert abs(got[0] - norm) <= 1.001 * om.U * norm + 1e-45 and abs(got[1] - factor) <= 1.001 * om.U * abs(factor)
    a, b = (rasterizer.gradient_norm([g.t for g in made], 1.0, 0.3) for _ in range(2))
    assert torch.equal(a, b)


def test_norm_of_far_values_and_of_none(rasterizer):
    big = torch.full((1000,), 3e38, device="cuda")
    tiny = torch.full((1000,), 1e-30, device="cuda")
    got = numbers(rasterizer.gradient_norm([big], 1.0, 1e-10))  # squares beyond float32
    assert abs(got[0] / (np.float32(3e38).astype(np.float64) * np.sqrt(1000) * 1e-10) - 1) <= 2 * om.U
    got = numbers(rasterizer.gradient_norm([tiny], 1e-35))
    assert abs(got[0] / (np.float32(1e-30).astype(np.float64) * np.sqrt(1000)) - 1) <= 2 * om.U
    got = numbers(rasterizer.gradient_norm([], 1.0, 0.5))
    assert got.tolist() == [0.0, 0.5]
    for bad in (np.nan, np.inf, -np.inf):
        big[77] = bad
        got = numbers(rasterizer.gradient_norm([tiny, big], 1.0))
        assert not np.isfinite(got[0]) and np.isnan(got[1])
    got = numbers(rasterizer.gradient_norm([torch.full((4,), 3e38, device="cuda")], 1.0))
    assert np.isinf(got[0]) and np.isnan(got[1])  # beyond float32: counts as overflowed


# ---- moments to 8 bits and back ----------------------------------------------------------------------------------------

def test_pack_and_unpack(rasterizer):
    rng = np.random.default_rng(16)
    items, start = [], []
    for k, n in enumerate(SIZES * 6):
        m = (rng.standard_normal(n) * np.exp(rng.normal(-3, 3, n))).astype(np.float32)
        v = (rng.random(n) * np.exp(rng.normal(-9, 6, n))).astype(np.float32)
        if k % 5 == 1:
            m[:], v[:] = 0, 0
        if k % 5 == 2:
            m *= np.float32(1e-38)  # below the smallest normal number
            v *= np.float32(1e-38)
        if k % 5 == 3 and n:
            m[n // 2], v[n // 2] = 3.4e38, 3.4e38
        if k % 5 == 4 and n:
            m[0], v[n - 1] = np.nan, np.inf
        room = -(-n // 128) * 128
        items.append((Guarded(m, torch.float32, k % 3), Guarded(v, torch.float32, k % 3), Guarded(np.zeros(0), torch.uint8, 8, room),
                      Guarded(np.zeros(0), torch.uint8, 0, room), Guarded(np.zeros(0), torch.uint8, 2, room // 64)))
        start.append((m, v))
    rasterizer.convert_moments([tuple(x.t for x in i) for i in items], pack=True)
    for i, (m, v) in zip(items, start):
        half = np.full(m.size, 1 << 19)
        mc, vc, scale = om.encode(m, v, half, half)
        got = [x.t.cpu().numpy() for x in i[2:]]
        np.testing.assert_array_equal(got[0], mc)
        np.testing.assert_array_equal(got[1], vc)
        np.testing.assert_array_equal(got[2].reshape(-1, 2), scale)
        for x in i:
            x.check()
        i[0].t.fill_(7.0)
        i[1].t.fill_(7.0)
    rasterizer.convert_moments([tuple(x.t for x in i) for i in items], pack=False)
    for i, (m, v) in zip(items, start):
        mc, vc, scale = (x.t.cpu().numpy() for x in i[2:])
        scale = scale.reshape(-1, 2)
        for k, (x, was, got) in enumerate(zip(om.decode(mc, vc, scale), (m, v), (i[0], i[1]))):
            got.check()
            y = numbers(got.t)
            with np.errstate(over="ignore"):
                x32 = x[:m.size].astype(np.float32)
            # a code's value takes 12 bits, but for the first of an offset that float32 rounds once more
            np.testing.assert_allclose(y, x32, rtol=2 * om.U, atol=0, equal_nan=True)
            fine = np.isfinite(x[:m.size]) & (np.abs(was) < 3e38)
            unit = np.repeat(np.exp2(scale[:, k] - 127.0), 128)[:m.size]
            # nearest: half of an eighth of (value + unit), and above zero at least a code
            with np.errstate(invalid="ignore"):
                assert (np.abs(y - was)[fine] <= ((np.abs(was) + unit) / 16 * 1.0001 + (unit / 8 if k else 0))[fine]).all()
