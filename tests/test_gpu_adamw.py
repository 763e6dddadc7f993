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


class Batch:
    """Tensors of a list with their state, odd ones of them unaligned, their places in the flat arrays apart from each other; and what
    the model starts from. items: (n, param type, gradient type, group). A third of the tensors is at its first step."""

    def __init__(self, rng, items, bits=32, with_master=False, first=256):
        self.bits, self.items, at = bits, [], first
        for k, (n, param, grad, group) in enumerate(items):
            off = [0, 1, 3, 0][k % 4]
            p = torch.from_numpy(rng.standard_normal(n) * 0.1).to(param).double().numpy()
            g = gradients(rng, n, grad).double().numpy()
            spread = np.exp(rng.normal(-4, 2, n))
            m, v = (0.2 * spread * rng.standard_normal(n)).astype(np.float32), (spread ** 2 * rng.random(n)).astype(np.float32)
            m[v < 1e-30] = 0
            if k % 3 == 0:
                m[:], v[:] = 0, 0
            master = with_master and param != torch.float32
            if master:
                p = (rng.standard_normal(n) * 0.1).astype(np.float32).astype(np.float64)
            blocks = -(-n // 128)
            item = dict(n=n, first=at, blocks=blocks, group=group, param=Guarded(p, param, off), grad=Guarded(g, grad, off), g=g, m=m, v=v, master=master)
            item["p"] = p if master else numbers(item["param"].t)
            self.items.append(item)
            at += (blocks + k % 2) * 128
        self.size = at + 256
        f32 = dict(dtype=torch.float32, device="cuda")
        self.master = torch.full((self.size,), 3.0, **f32) if with_master else None
        if bits == 32:
            self.m, self.v, self.scale = torch.full((self.size,), 3.0, **f32), torch.full((self.size,), 3.0, **f32), None
        else:
            self.m, self.v = (torch.full((self.size,), 3, dtype=torch.uint8, device="cuda") for _ in range(2))
            self.scale = torch.full((self.size // 128, 2), 3, dtype=torch.uint8, device="cuda")
        for k, i in enumerate(self.items):
            where = slice(i["first"], i["first"] + i["blocks"] * 128)
            if bits == 32:
                self.m[where], self.v[where] = (torch.from_numpy(om.padded(i[x])).cuda() for x in "mv")
            else:
                rm, rv, _ = om.random_bits(5, 1, 0, i["n"])
                mc, vc, scale = om.encode(i["m"], i["v"], rm, rv)
                self.m[where], self.v[where] = torch.from_numpy(mc).cuda(), torch.from_numpy(vc).cuda()
                self.scale[i["first"] // 128:i["first"] // 128 + i["blocks"]] = torch.from_numpy(scale).cuda()
                i["m"], i["v"] = (x[:i["n"]].astype(np.float32) for x in om.decode(mc, vc, scale))
            if with_master:
                self.master[where] = torch.from_numpy(om.padded(i["p"]).astype(np.float32)).cuda() if i["master"] else 0.0
        self.used = torch.zeros(self.size, dtype=torch.bool, device="cuda")
        for i in self.items:
            self.used[i["first"]:i["first"] + i["blocks"] * 128] = True

    def step(self, rasterizer, groups, **kw):
        tensors = [(i["param"].t, i["grad"].t, i["first"], i["group"]) for i in self.items]
        rasterizer.adamw_step(tensors, groups, self.m, self.v, self.scale, self.master, moment_bits=self.bits, **kw)

    def flat(self):
        return [x for x in (self.m, self.v, self.scale, self.master) if x is not None]

    def of(self, i, flat):
        k = 128 if flat is not self.scale else 1
        return flat[i["first"] // 128 * k:(i["first"] // 128 + i["blocks"]) * k]

    def check(self):
        """Nothing beside the tensors and their places was written, and places behind a tensor's last element hold zeros."""
        for i in self.items:
            i["param"].check()
            i["grad"].check()
            for x in (self.m, self.v):
                assert not self.of(i, x)[i["n"]:].any()
        for x in (self.m, self.v, self.master):
            assert x is None or (x[~self.used] == 3).all()
        assert self.scale is None or (self.scale[~self.used[::128]] == 3).all()

    def compare(self, groups, seed=0, stochastic=False, scale=1.0, beta1=0.9, beta2=0.999, eps=1e-8):
        self.check()
        for i in self.items:
            lr, decay, step = groups[i["group"]]
            n = i["n"]
            if n == 0:
                continue
            p, m, v, tol_p, tol_m, tol_v = om.step64(i["p"], i["g"], i["m"], i["v"], step, lr, decay, beta1, beta2, eps, scale)
            got, kind = numbers(i["param"].t), i["param"].t.dtype
            if i["master"]:
                held = self.of(i, self.master)[:n]
                assert (np.abs(numbers(held) - p) <= tol_p).all()
                assert torch.equal(i["param"].t, held.to(kind))
            else:
                half = HALF_STEP[kind]
                if stochastic and kind == torch.bfloat16:
                    half *= 2  # up or down, not to the nearest
                tol = tol_p * (1 + 2 * half) + half * np.abs(p) + (2.0 ** -25 if kind == torch.float16 else 0)
                assert (np.abs(got - p) <= tol).all(), (n, np.max(np.abs(got - p) / tol))
            if self.bits == 32:
                assert (np.abs(numbers(self.of(i, self.m))[:n] - m) <= tol_m).all() and (np.abs(numbers(self.of(i, self.v))[:n] - v) <= tol_v).all()
            else:
                fm, fv = om.moments_in_float(i["m"], i["v"], i["g"], beta1, beta2, scale)
                assert (np.abs(fm - m) <= tol_m).all() and (np.abs(fv - v) <= tol_v).all()
                rm, rv, _ = om.random_bits(seed, step, i["first"], n)
                for want, x in zip(om.encode(fm, fv, rm, rv), (self.m, self.v, self.scale)):
                    np.testing.assert_array_equal(self.of(i, x).cpu().numpy(), want)


F, B, H = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F, F), (B, B), (H, H), (F, B), (F, H), (B, F), (H, F), (B, H), (H, B)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("param,grad", TYPES, ids=lambda t: str(t).replace("torch.", ""))
def test_step_against_64_bits(bits, master, param, grad, rasterizer):
    groups = [(0.01, 0.1, 7), (0.002, 0.0, 400)]
    batch = Batch(np.random.default_rng(3), [(n, param, grad, k % 2) for k, n in enumerate(SIZES)], bits, master)
    batch.step(rasterizer, groups, seed=11, grad_scale=torch.tensor([0.25], device="cuda"))
    batch.compare(groups, 11, scale=0.25)
    assert all(np.array_equal(numbers(i["grad"].t), i["g"]) for i in batch.items)  # read only
    batch.step(rasterizer, [(0.0, 0.0, 2)] * 2, zero_grad=True)
    assert not any(i["grad"].t.any() for i in batch.items)
    batch.check()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("param,grad", [(F, F), (B, B), (F, B), (H, H), (B, F)], ids=lambda t: str(t).replace("torch.", ""))
def test_step_of_many_elements(bits, master, param, grad, rasterizer):
    """Calls that are large enough for workgroups of four waves."""
    sizes = [1_400_003, 0, 2048 * 40, 2048 * 3 + 5, 7, 130_000]
    groups = [(0.01, 0.1, 3), (0.002, 0.0, 40)]
    batch = Batch(np.random.default_rng(17), [(n, param, grad, k % 2) for k, n in enumerate(sizes)], bits, master)
    batch.step(rasterizer, groups, seed=12, stochastic_rounding=True, grad_scale=torch.tensor([3.0], device="cuda"))
    batch.compare(groups, 12, stochastic=True, scale=3.0)


def test_tiny_eps_and_many_elements(rasterizer):
    batch = Batch(np.random.default_rng(18), [(1_600_001, F, F, 0), (300, B, B, 0)], 8)
    batch.step(rasterizer, [(0.01, 0.0, 2)], eps=1e-15, seed=1)
    batch.compare([(0.01, 0.0, 2)], 1, eps=1e-15)


@pytest.mark.parametrize("eps", [1e-6, 1e-15, 1e-30])
def test_tiny_eps_and_tiny_gradients(eps, rasterizer):
    """Second moments below the smallest normal number count where eps is small enough to let them."""
    batch = Batch(np.random.default_rng(4), [(1000, F, F, 0)], 8)
    g = np.float32(1e-18) * np.random.default_rng(5).standard_normal(1000).astype(np.float32)
    batch.items[0]["grad"].t.copy_(torch.from_numpy(g))
    batch.items[0]["g"] = g.astype(np.float64)
    batch.step(rasterizer, [(0.01, 0.0, 1)], eps=eps)
    # the second moment is rounded below 2^-126 by 2^-150 a product, which the model does not carry into the root: up to 2^-75 there,
    # so it is held to where that does not show
    i = batch.items[0]
    p, _, v, tol, *_ = om.step64(i["p"], i["g"], i["m"], i["v"], 1, 0.01, eps=eps)
    fm, fv = om.moments_in_float(i["m"], i["v"], i["g"], 0.9, 0.999)
    q = 0.01 * (fm.astype(np.float64) / (1 - 0.9)) / (np.sqrt(fv.astype(np.float64) / (1 - 0.999)) + eps)
    assert (np.abs(numbers(i["param"].t) - (i["p"] - q)) <= 5 * om.U * np.abs(i["p"]) + 22 * om.U * np.abs(q) + 1e-44).all()
    assert eps > 1e-10 or np.median(np.abs(q)) > 1e-6


@pytest.mark.parametrize("bits", [32, 8])
def test_bf16_parameters_are_rounded_by_random_bits(bits, rasterizer):
    """The parameter is the neighbour that the random bits say; infinities and NaN stay."""
    batch = Batch(np.random.default_rng(5), [(n, B, B, 0) for n in (5001, 128, 3)], bits)
    for i in batch.items:
        i["param"].t[::7] = float("inf")
        i["param"].t[1::7] = float("nan")
        i["p"] = numbers(i["param"].t)
    batch.step(rasterizer, [(1e-3, 0.0, 9)], seed=3, stochastic_rounding=True)
    for i in batch.items:
        got = numbers(i["param"].t)
        finite = np.isfinite(i["p"])
        assert np.array_equal(got[~finite], i["p"][~finite], equal_nan=True)
        with np.errstate(invalid="ignore"):
            want, *_ = om.step64(i["p"], i["g"], i["m"], i["v"], 9, 1e-3)
            rp = om.random_bits(3, 9, i["first"], got.size)[2]
            up = om.floats_of((om.bits_of(want) + rp) & ~0xFFFF)
        # float32 arithmetic may put an element on the other side of its border where the random bits come within its error of it
        off = finite & (up != got)
        assert off.mean() <= 1e-3 and (np.abs(got - want)[finite] <= 2.0 ** -7 * np.abs(want[finite]) + 1e-6).all()


def fresh(n, flat=torch.uint8):
    """Flat arrays of a new state of n elements, a multiple of 128."""
    return torch.zeros(n, dtype=flat, device="cuda"), torch.zeros(n, dtype=flat, device="cuda"), torch.zeros(n // 128, 2, dtype=torch.uint8, device="cuda")


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
        p, (mc, vc, scale) = p0.clone(), fresh(n)
        rasterizer.adamw_step([(p, g, 0, 0)], [(1e-3, 0.0, 1)], mc, vc, scale, moment_bits=8, stochastic_rounding=True, seed=seed)
        m, v = om.decode(*(t.cpu().numpy() for t in (mc, vc, scale)))
        seen.add(mc.cpu().numpy().tobytes())
        for k, x in (("p", numbers(p)), ("m", m), ("v", v)):
            total[k] += x
    assert len(seen) == seeds
    want = om.step64(numbers(p0), numbers(g), np.zeros(n), np.zeros(n), 1, 1e-3)
    unit = np.exp2(numbers(scale) - 127)
    for k, x, u in (("p", want[0], None), ("m", want[1], unit[:, 0]), ("v", want[2], unit[:, 1])):
        # steps: 2^-7 of the parameter's binade; an eighth of (value + unit)
        step = 2.0 ** -7 * np.abs(x) * 2 if u is None else (np.abs(x) + np.repeat(u, 128)) / 8 * 1.001
        keep = x >= np.repeat(u, 128) / 8 if k == "v" else np.ones(n, bool)  # smaller ones are rounded up, on purpose
        error = np.abs(total[k] / seeds - x)
        assert (error <= 6 * step / 2 / np.sqrt(seeds) + 1e-6 * np.abs(x) + 1e-12)[keep].all(), k


def test_second_moments_above_zero_stay_above_zero(rasterizer):
    n = 256
    g = torch.full((n,), 1e-12, device="cuda")
    g[0] = 1.0
    g[5], g[200:] = 0.0, 0.0
    for seed in range(20):
        mc, vc, scale = fresh(n)
        rasterizer.adamw_step([(torch.zeros(n, device="cuda"), g, 0, 0)], [(1e-3, 0.0, 1)], mc, vc, scale, moment_bits=8, seed=seed)
        assert torch.equal(vc > 0, g != 0)


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite(bits, rasterizer):
    """In 32 bits an element keeps its own NaN or infinity; in 8 bits its block of 128 reads as NaN, the others go on."""
    batch = Batch(np.random.default_rng(8), [(128 * 5 + 9, F, F, 0)], bits)
    i = batch.items[0]
    bad = {3: np.nan, 130: np.inf, 300: -np.inf, 128 * 5 + 8: np.nan}
    for k, x in bad.items():
        i["grad"].t[k] = x
    batch.step(rasterizer, [(0.01, 0.0, 4)])
    place = np.arange(i["n"])

    def moments():
        if bits == 32:
            return [numbers(batch.of(i, x))[:i["n"]] for x in (batch.m, batch.v)]
        return [x[:i["n"]] for x in om.decode(*(batch.of(i, x).cpu().numpy() for x in (batch.m, batch.v, batch.scale)))]

    lost = np.isin(place // 128, [k // 128 for k in bad]) if bits == 8 else np.isin(place, list(bad))
    for x in moments():
        assert np.array_equal(~np.isfinite(x), lost)
    p = numbers(i["param"].t)
    assert np.isfinite(p[~np.isin(place, list(bad))]).all()
    # a second step reads what the first left
    i["grad"].t.fill_(0.5)
    batch.step(rasterizer, [(0.01, 0.0, 5)])
    assert np.array_equal(~np.isfinite(numbers(i["param"].t)), lost)
    for x in moments():
        assert np.array_equal(~np.isfinite(x), lost)
    batch.check()


def test_a_lost_first_moment_stays_lost(rasterizer):
    """Also where the second moment of the same block is fine, and in a block that ends early."""
    n = 128 * 2 + 5
    m, v = torch.full((n,), 0.5, device="cuda"), torch.full((n,), 0.25, device="cuda")
    m[130], m[n - 1] = float("inf"), float("nan")
    mc, vc, scale = fresh(384)
    rasterizer.convert_moments([(m, v, 0)], mc, vc, scale, pack=True)
    p, g = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    for step in (1, 2, 3):
        rasterizer.adamw_step([(p, g, 0, 0)], [(0.01, 0.0, step)], mc, vc, scale, moment_bits=8)
        assert scale[1:, 0].tolist() == [255, 255] and scale[0, 0] < 255 and (scale[:, 1] < 255).all()
        assert torch.isfinite(p[:128]).all() and torch.isnan(p[128:]).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_step_whose_factor_is_not_finite_is_left_out(bits, value, rasterizer):
    batch = Batch(np.random.default_rng(9), [(n, t, t, 0) for n, t in ((5001, F), (3, B), (700, B), (2048, H))], bits, True)
    everything = lambda: [x.clone() for x in batch.flat()] + [i["param"].whole.clone() for i in batch.items]  # noqa: E731
    before, grads = everything(), [i["grad"].whole.clone() for i in batch.items]
    scale = torch.tensor([value], device="cuda")
    batch.step(rasterizer, [(0.01, 0.1, 4)], grad_scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(before, everything()))
    assert all(torch.equal(i["grad"].whole, g) for i, g in zip(batch.items, grads))
    batch.step(rasterizer, [(0.01, 0.1, 4)], grad_scale=scale, zero_grad=True)
    assert all(torch.equal(a, b) for a, b in zip(before, everything())) and not any(i["grad"].t.any() for i in batch.items)
    batch.check()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [8, 9, 64, 65, 160, 161, 531])
def test_long_lists_many_groups_and_mixed_types(bits, count, rasterizer):
    """Up to and beyond what a launch takes, in tensors and in groups, every combination of types, empty tensors among them."""
    rng = np.random.default_rng(10)
    groups = [(1e-3 * (k + 1), 0.01 * k, k + 1) for k in range(23)]
    items = []
    for k in range(count):
        n = int(rng.integers(0, 300)) if k % 5 else int(rng.integers(0, 9000))
        items.append((n, *TYPES[int(rng.integers(len(TYPES)))], int(rng.integers(23)) if k % 2 and count > 100 else k % 3))
    batch = Batch(rng, items, bits, count % 2 == 1)
    batch.step(rasterizer, groups, seed=1 << 63, beta1=0.8, beta2=0.99, eps=1e-6)
    batch.compare(groups, 1 << 63, beta1=0.8, beta2=0.99, eps=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_betas_of_zero(bits, rasterizer):
    batch = Batch(np.random.default_rng(12), [(n, F, F, 0) for n in (1000, 77)], bits)
    batch.step(rasterizer, [(0.01, 0.0, 1)], beta1=0.0, beta2=0.0, seed=2)
    batch.compare([(0.01, 0.0, 1)], 2, beta1=0.0, beta2=0.0)


def test_far_places(rasterizer):
    """A tensor whose place in the flat arrays passes 2^33, where the numbers of the random bits begin again, and 2^32."""
    rng = np.random.default_rng(13)
    for first in ((1 << 33) - 512, (1 << 32) - 128):
        n = 1000
        size = first + 1024
        mc, vc = (torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2))
        scale = torch.empty(size // 128, 2, dtype=torch.uint8, device="cuda")
        for x, at in ((mc, first), (vc, first), (scale, first // 128)):
            x[at - 1:] = 0
        g, p = torch.from_numpy(rng.standard_normal(n)).float().cuda(), torch.zeros(n, device="cuda")
        rasterizer.adamw_step([(p, g, first, 0)], [(0.01, 0.0, 1)], mc, vc, scale, moment_bits=8, seed=4)
        zero = np.zeros(n, np.float32)
        fm, fv = om.moments_in_float(zero, zero, g.cpu().numpy(), 0.9, 0.999)
        rm, rv, _ = om.random_bits(4, 1, first, n)
        for want, x, at in zip(om.encode(fm, fv, rm, rv), (mc, vc, scale), (first, first, first // 128)):
            np.testing.assert_array_equal(x[at:at + len(want)].cpu().numpy(), want)
            assert not x[at - 1].any()
        del mc, vc, scale


def test_a_tensor_of_several_entries(rasterizer):
    """More elements than an entry of a launch has: every part as a tensor of its own has it."""
    n = (1 << 30) + (1 << 22) + 77
    gen = torch.Generator("cuda").manual_seed(1)
    g = torch.empty(n, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    flat = fresh(-(-n // 128) * 128)
    rasterizer.adamw_step([(p, g, 0, 0)], [(1e-3, 0.0, 1)], *flat, moment_bits=8, stochastic_rounding=True, seed=9)
    for first, end in ((0, 5120), ((1 << 28) - 1280, (1 << 28) + 2560), ((1 << 30) - 1280, (1 << 30) + 2560), ((n // 128 - 9) * 128, n)):
        part, own = torch.zeros(end - first, dtype=torch.bfloat16, device="cuda"), fresh(-(-end // 128) * 128)
        rasterizer.adamw_step([(part, g[first:end].clone(), first, 0)], [(1e-3, 0.0, 1)], *own, moment_bits=8, stochastic_rounding=True, seed=9)
        assert torch.equal(part, p[first:end]) and part.any()
        for x, y, k in zip(own, flat, (1, 1, 128)):
            assert torch.equal(x[first // k:], y[first // k:first // k + len(x[first // k:])])
        del own
    # and its norm: a sum of squares of ones at known places, among zeros
    del p, flat
    g.zero_()
    at = torch.tensor([0, 1, (1 << 29) - 1, 1 << 29, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, n - 1], device="cuda")
    g[at] = 3.0
    assert rasterizer.gradient_norm([g]).cpu()[0].item() == np.float32(3.0 * np.sqrt(8.0))


# ---- steps whose count lies on the device ------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("num_groups", [1, 9, 300])
def test_the_count_on_the_device_is_the_same_step(bits, num_groups, rasterizer):
    items = [(n, F, F, k * 7 % num_groups) for k, n in enumerate([1000, 1, 0, 500, 129] * 4)]
    a, b = (Batch(np.random.default_rng(14), items, bits) for _ in range(2))
    state = torch.zeros(rasterizer.lib.vetrast_adamw_device_state_bytes(num_groups), dtype=torch.uint8, device="cuda")
    state[:8].view(torch.int64).fill_(41)
    state[8:12].view(torch.float32).fill_(0.5)
    lrs = [0.01 * (k % 5 + 1) for k in range(num_groups)]
    for step in (42, 43):
        scale = torch.tensor([0.5], device="cuda")
        a.step(rasterizer, [(lr, 0.1, 0) for lr in lrs], seed=6, device_state=state, grad_scale=scale)
        b.step(rasterizer, [(0.5 * lr, 0.1, step) for lr in lrs], seed=6, grad_scale=scale)
        assert state[:8].view(torch.int64).item() == step
        assert all(torch.equal(x, y) for x, y in zip(a.flat(), b.flat()))
        for i, j in zip(a.items, b.items):
            # pow on the device and on the host may differ in their last bits: the two constants by a rounding each
            x, y = numbers(i["param"].t), numbers(j["param"].t)
            assert (np.abs(x - y) <= 4 * om.U * (np.abs(y) + 0.05)).all()
            i["param"].t.copy_(j["param"].t)
    # a step that is left out is not counted
    a.step(rasterizer, [(lr, 0.1, 0) for lr in lrs], device_state=state, grad_scale=torch.tensor([np.inf], device="cuda"))
    assert state[:8].view(torch.int64).item() == 43
    rasterizer.adamw_step([], [], None, None, moment_bits=bits, device_state=state)
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
    items, start, at = [], [], 128
    for k, n in enumerate(SIZES * 8):
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
        items.append((Guarded(m, torch.float32, k % 3), Guarded(v, torch.float32, k % 3), at))
        start.append((m, v))
        at += (-(-n // 128) + k % 2) * 128
    flat = [x + 3 for x in fresh(at + 128)]
    arguments = [(m.t, v.t, first) for m, v, first in items]
    rasterizer.convert_moments(arguments, *flat, pack=True)
    used = np.zeros(at + 128, bool)
    for (gm, gv, first), (m, v) in zip(items, start):
        half, room = np.full(m.size, 1 << 19), -(-m.size // 128) * 128
        used[first:first + room] = True
        for want, x, k in zip(om.encode(m, v, half, half), flat, (1, 1, 128)):
            np.testing.assert_array_equal(x[first // k:(first + room) // k].cpu().numpy(), want)
        for x, was in ((gm, m), (gv, v)):
            x.check()
            np.testing.assert_array_equal(x.t.cpu().numpy(), was)
            x.t.fill_(7.0)
    for x, k in zip(flat, (1, 1, 128)):
        assert (x.cpu().numpy()[~used[::k]] == 3).all()
    rasterizer.convert_moments(arguments, *flat, pack=False)
    for (gm, gv, first), (m, v) in zip(items, start):
        room = -(-m.size // 128) * 128
        mc, vc, scale = (x[first // k:(first + room) // k].cpu().numpy() for x, k in zip(flat, (1, 1, 128)))
        for k, (x, was, got) in enumerate(zip(om.decode(mc, vc, scale), (m, v), (gm, gv))):
            got.check()
            y, x = numbers(got.t), x[:m.size]
            # a difference of two floats that float32 rounds once, where their exponents lie far apart
            np.testing.assert_allclose(y, x, rtol=om.U, atol=0, equal_nan=True)
            unit = np.repeat(np.exp2(scale[:, k] - 127.0), 128)[:m.size]
            fine = np.isfinite(x)
            # nearest: half of an eighth of (value + unit), and above zero at least a code
            with np.errstate(invalid="ignore"):
                assert (np.abs(y - was)[fine] <= ((np.abs(was) + unit) / 16 * 1.0001 + (unit / 8 if k else 0))[fine]).all()
