"""Eviction on the GPU: which entries a budget keeps against a sort in 64 bits, and rows of tensors bit by bit."""
import numpy as np
import pytest
import torch

from tests import entries_model as em
from vet_amd import torch_ops

pytestmark = pytest.mark.gpu


def scores(rows, n, kind, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed + n)
    s = torch.randn(rows, n, generator=gen, device="cuda")
    if kind == "weights":  # a third was seen by nobody
        s = torch.exp(2 * s) * (torch.rand(rows, n, generator=gen, device="cuda") < 0.67)
    if kind == "ties":  # few values, both zeros among them
        s = torch.round(s).clamp(-1, 1) * 0.5 * torch.where(s > 0.1, 1.0, -1.0)
    if kind == "equal":
        s = torch.full_like(s, -3.5)
    if kind == "special":
        values = torch.tensor([float("nan"), -float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-45, -1e-45, torch.finfo(torch.float32).min,
                               torch.finfo(torch.float32).max, 1.0, 1.0 + 2.0 ** -23], device="cuda")
        s = values[(torch.rand(rows, n, generator=gen, device="cuda") * len(values)).long().clamp(max=len(values) - 1)]
    return s


def check(score, budget, recent=0, length=None, got=None):
    index, count = torch_ops.select_kept(score, budget, recent, length) if got is None else got
    want, kept = em.select_kept(score.view(-1, score.shape[-1]).cpu().numpy(), budget, recent, None if length is None else length.cpu().numpy())
    assert index.dtype == torch.int32 and index.shape == score.shape[:-1] + (budget,)
    assert np.array_equal(index.view(-1, budget).cpu().numpy(), want)
    assert np.array_equal(count.cpu().numpy(), kept)


@pytest.mark.parametrize("kind", ["plain", "weights", "ties", "equal", "special"])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1023, 1024, 1025, 4097, 12_289, 20_000, 32_768, 32_769, 40_001, 300_007])
def test_scores_and_sizes(n, kind):
    s = scores(2, n, kind)
    for budget in sorted({1, n // 3, n // 2, n - 1, n, n + 3} - {0}):
        for recent in sorted({0, 1, budget // 2, budget}):
            check(s, budget, recent)


@pytest.mark.parametrize("n", [1, 70, 5000, 33_000])
def test_lengths(n):
    """Rows of any length; what lies behind it is not looked at."""
    length = torch.tensor([0, 1, n // 2, n, n + 5, -3, max(n - 1, 0)], dtype=torch.int32, device="cuda")
    s = scores(len(length), n, "weights")
    for row, m in enumerate(length.tolist()):
        s[row, max(m, 0):] = float("inf")
    for budget, recent in ((1, 0), (1, 1), (max(n // 3, 1), max(n // 3, 1) // 4), (n, 0), (n + 2, 2)):
        check(s, budget, recent, length)


def test_the_lowest_digits_decide():
    """Scores that differ in their last bits alone, in one row of a workgroup and in one of several."""
    for n in (30_000, 200_000):
        gen = torch.Generator(device="cuda").manual_seed(n)
        bits = torch.randint(0, 1500, (1, n), generator=gen, device="cuda", dtype=torch.int32)
        check((bits + 0x3F800000).view(torch.float32), n // 2, 17)
        check((bits + 0x3F800000).view(torch.float32).neg(), n // 2, 17)


def test_a_cloud():
    check(scores(1, 5_500_000, "weights")[0], 4_125_000, 550_000)
    check(scores(1, 2_000_003, "plain")[0], 5, 2)


def test_long_rows_that_end_anywhere():
    """Workgroups with several shares, some of them empty; rows beside one another whose budget ends among zeros and elsewhere."""
    n = 2_000_003
    length = torch.tensor([n, 1_234_567, 6144 * 4 + 1, 17, 1_600_000], dtype=torch.int32, device="cuda")
    s = torch.cat([scores(3, n, "weights"), scores(1, n, "plain"), scores(1, n, "ties")])
    s[1, :700_000] = 0
    for budget, recent in ((20_000, 0), (1_000_000, 333), (1_500_000, 100_000)):
        check(s, budget, recent, length)
        check(s.flip(0), budget, recent, length)


def test_many_rows():
    check(scores(70_001, 3, "ties"), 2, 1)
    s = scores(300, 1000, "plain")
    check(s[:, 100:900], 77, 9)  # rows further apart than their scores
    check(s.t()[:300], 100, 9)
    check(s[:1].expand(5, 1000), 10)
    check(s[:, :1], 1)
    check(s[:, :1].expand(300, 7), 3)
    check(s[:0], 4)
    index, count = torch_ops.select_kept(s[:, :0], 3)
    assert (index == -1).all() and (count == 0).all()
    index, count = torch_ops.select_kept(s, 0)
    assert index.shape == (300, 0) and (count == 0).all()


def test_rows_behind_one_another_beyond_32_bits():
    """More rows than a launch takes, of several workgroups each."""
    n = 32_770
    s = torch.zeros(n, n, device="cuda")
    s[:, 7] = 1
    s[n - 1, n - 2] = 5
    s[n - 2, 0] = -1
    index, count = torch_ops.select_kept(s, 3, recent=1)
    want = torch.tensor([0, 7, n - 1], dtype=torch.int32, device="cuda")
    assert (count == 3).all() and (index[:n - 2] == want).all()
    assert index[n - 1].tolist() == [7, n - 2, n - 1] and index[n - 2].tolist() == [1, 7, n - 1]


def test_more_rows_than_threads_have_numbers():
    """Rows of one workgroup each, more than a launch takes."""
    rows = 2 ** 21 + 7
    s = torch.zeros(rows, 3, device="cuda")
    s[:, 1] = 1
    s[rows - 2, 0] = 2
    index, count = torch_ops.select_kept(s, 2, recent=1)
    assert (count == 2).all() and (index[:, 1] == 2).all()
    assert (index[:rows - 2, 0] == 1).all() and index[rows - 2, 0] == 0 and index[rows - 1, 0] == 1


def test_the_longest_row_and_a_budget_beyond_it():
    n = 2 ** 30
    s = torch.zeros(n, device="cuda")
    s[5], s[n - 2], s[n // 2] = 1, 1, -1
    index, count = torch_ops.select_kept(s, 4, recent=1)
    assert index.tolist() == [0, 5, n - 2, n - 1] and count.item() == 4
    index, count = torch_ops.select_kept(s[:70_000], 2 ** 28 + 3)
    assert count.item() == 70_000 and torch.equal(index[:70_000], torch.arange(70_000, dtype=torch.int32, device="cuda")) and (index[70_000:] == -1).all()
    index, count = torch_ops.select_kept(s[:7], 2 ** 26 + 3)
    assert count.item() == 7 and index[:7].tolist() == list(range(7)) and (index[7:] == -1).all()


def test_the_rasterizer_class(rasterizer):
    for n in (100, 50_000):
        s = scores(3, n, "weights")
        length = torch.tensor([n, n // 2, 0], dtype=torch.int32, device="cuda")
        check(s, n // 4, 5, length, rasterizer.select_kept(s, n // 4, 5, length))
        need = rasterizer.lib.vetrast_select_kept_workspace_bytes(3, n)
        dirty = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
        for _ in range(2):  # whatever the workspace holds
            check(s, n // 4, 5, length, rasterizer.select_kept(s, n // 4, 5, length, workspace=dirty))


def test_select_refusals():
    s = torch.zeros(2, 10, device="cuda")
    for bad in (torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="length"):
            torch_ops.select_kept(s, 2, length=bad)
    for bad in (s.double(), s.half(), s.view(1, 2, 10)):
        with pytest.raises(RuntimeError, match="score"):
            torch_ops.select_kept(bad, 2)


# ---- rows of tensors -------------------------------------------------------------------------------------------------------

def same(got, t, index, dim):
    a = (t.view(torch.int16) if t.dtype == torch.bfloat16 else t).detach().cpu().numpy()
    want = em.keep_rows(a, index.cpu().numpy(), dim % t.dim())
    assert got.dtype == t.dtype and got.is_contiguous() and not got.requires_grad and list(got.shape) == list(want.shape)
    got = (got.view(torch.int16) if t.dtype == torch.bfloat16 else got).cpu().numpy()
    assert got.tobytes() == np.ascontiguousarray(want).tobytes()


def some_indices(n, kept, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    i = torch.randint(-2, n + 2, (kept,), generator=gen, device="cuda", dtype=torch.int32)  # any order, some twice, some none
    i[0] = max(n - 1, 0)
    return i


@pytest.mark.parametrize("n, kept", [(1, 1), (5, 3), (100, 7), (257, 1030), (5003, 4100)])
def test_keep_rows_of_any_kind(n, kept):
    tensors, dims = [], []
    for dtype in (torch.uint8, torch.int16, torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64, torch.float64, torch.complex128, torch.bool):
        for shape, dim in (((n,), 0), ((n, 3), 0), ((4, n), 1), ((n, 4), -2), ((2, 3, n, 5), 2), ((1, n), 1), ((n, 1), 0)):
            tensors.append((torch.randn(shape, device="cuda") * 50).to(dtype))
            dims.append(dim)
    index = some_indices(n, kept)
    for got, t, d in zip(torch_ops.keep_rows(tensors, index, dims), tensors, dims):  # 70 tensors: several launches
        same(got, t, index, d)


def test_keep_rows_of_heads():
    rows, n, kept = 6, 501, 130
    index = torch.stack([some_indices(n, kept, k) for k in range(rows)])
    index[2] = -1
    tensors = [torch.randn(rows, n, 128, device="cuda").bfloat16(), torch.randn(rows, n, device="cuda"), torch.randn(rows, 3, n, 33, device="cuda").half(),
               torch.randn(rows, 2, 2, n, device="cuda")]
    dims = [1, 1, 2, 3]
    for got, t, d in zip(torch_ops.keep_rows(tensors, index, dims), tensors, dims):
        same(got, t, index, d)


def test_keep_rows_of_views():
    """Caches with room behind the last entry, every second entry, dimensions turned, one row for all, an odd address; indices of a view."""
    index = some_indices(40, 25)
    heads = torch.stack([some_indices(40, 25, k) for k in range(4)])
    x = torch.randn(4, 64, 24, device="cuda")
    wide = torch.zeros(4, 60, dtype=torch.int32, device="cuda")
    wide[:, 10:35] = heads
    for t, d in ((x[:, :40], 1), (x[:, 1:41, 3:19], 1), (x[:, 3:64:2].narrow(1, 0, 30), 1), (x.transpose(0, 1)[:40], 0), (x.permute(0, 2, 1)[:, :, :40], 2),
                 (x[:, :1].expand(4, 40, 24), 1), (x[:1].expand(4, 64, 24), 1), (x.bfloat16()[:, :40, 1:], 1), (x[0, :, 0], 0)):
        (got,) = torch_ops.keep_rows([t], index, [d])
        same(got, t, index, d)
        if d > 0:
            (got,) = torch_ops.keep_rows([t], wide[:, 10:35], [d])
            same(got, t, heads, d)


def test_nothing_and_empty():
    index = some_indices(9, 5)
    assert torch_ops.keep_rows([], index, []) == []
    got = torch_ops.keep_rows([torch.randn(0, 3, device="cuda"), torch.randn(9, 0, device="cuda"), torch.randn(0, 9, device="cuda")], index, [0, 0, 1])
    assert [list(g.shape) for g in got] == [[5, 3], [5, 0], [0, 5]] and (got[0] == 0).all()
    (got,) = torch_ops.keep_rows([torch.randn(9, device="cuda")], index[:0], [0])
    assert got.shape == (0,)


def test_offsets_beyond_32_bits():
    n = 1_200_000_007
    x = torch.zeros(1, n, dtype=torch.float32, device="cuda")
    there = torch.tensor([0, 1 << 30, n - 1, n - 2], device="cuda")
    x[0, there] = torch.arange(1.0, 5.0, device="cuda")
    at = torch.cat([there, there.new_tensor([-1, n])]).int()
    (got,) = torch_ops.keep_rows([x], at, [1])
    assert got.tolist() == [[1.0, 2.0, 3.0, 4.0, 0.0, 0.0]]


def test_results_of_many_bytes():
    """More units than a launch counts in one entry: an outer of 2^30 bytes and more, byte by byte."""
    kept = (1 << 30) + 5000
    x = torch.arange(251, dtype=torch.uint8, device="cuda")
    index = (torch.arange(kept, device="cuda", dtype=torch.int32) % 251)
    (got,) = torch_ops.keep_rows([x], index, [0])
    assert (got == index).all()


def test_keep_refusals():
    x, index = torch.randn(4, 9, device="cuda"), some_indices(9, 5)
    for tensors, i, dims, match in (([x], index, [], "dimensions"), ([x], index, [2], "no entries"), ([x], index, [-3], "no entries"), ([x], index.long(), [1], "int32"),
                                    ([x], index.view(1, 1, 5), [1], "int32"), ([x], index.view(1, 5), [1], "rows"), ([x], index.expand(4, 5), [0], "no entries"),
                                    ([x.cpu()], index, [1], "on cuda"), ([torch.randn(3, dtype=torch.complex64, device="cuda").conj()], index, [0], "conjugate")):
        with pytest.raises(RuntimeError, match=match):
            torch_ops.keep_rows(tensors, i, dims)
    same(torch_ops.keep_rows([x], index.expand(4, 5), [1])[0], x, index.expand(4, 5), 1)


def test_captured_and_on_another_stream():
    s, x = scores(1, 100_000, "weights"), torch.randn(4, 100_000, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch_ops.keep_rows([x, s], torch_ops.select_kept(s[0], 60_000, 100)[0], [1, 1])
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = torch_ops.select_kept(s[0], 60_000, 100)
        rows = torch_ops.keep_rows([x, s], got[0], [1, 1])
    for k in range(4):
        s.copy_(scores(1, 100_000, ["weights", "ties", "plain", "equal"][k], seed=k))
        graph.replay()
        torch.cuda.synchronize()
        check(s[0], 60_000, 100, got=got)
        assert torch.equal(rows[0], x[:, got[0].long()]) and torch.equal(rows[1], s[:, got[0].long()])
        torch.randn(100_000, device="cuda").sort()
