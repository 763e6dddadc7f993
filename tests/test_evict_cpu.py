"""Eviction's entry points without a GPU: layout of the structs, what is refused, sizes of workspaces."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import entries_model as em
from tests.test_dropout_cpu import AT, compare_layout
from vet_amd import abi, torch_ops


CONTEXT = C.create_string_buffer(1 << 16)  # refusals come before anything reads it


def lib_and_context():
    return abi.load_library(), C.addressof(CONTEXT)


def test_every_struct_field_sits_where_the_c_compiler_puts_it(tmp_path):
    compare_layout(tmp_path, [("vetrast_select_args", abi.SelectArgs), ("vetrast_keep_tensor", abi.KeepTensor), ("vetrast_keep_args", abi.KeepArgs)])


def select_args(**changes):
    a = abi.SelectArgs()
    a.score = a.index = a.count = a.workspace = AT
    a.row_stride = a.n = 100
    a.rows, a.budget, a.recent = 3, 10, 4
    for k, v in changes.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("changes", [dict(rows=-1), dict(n=-1), dict(budget=-1), dict(recent=-1), dict(recent=11), dict(row_stride=99), dict(score=None),
                                     dict(index=None), dict(count=None), dict(score=AT + 2), dict(length=AT + 1), dict(index=AT + 2), dict(count=AT + 3),
                                     dict(workspace=AT + 8), dict(n=100_000, row_stride=100_000, workspace=None)])
def test_select_refusals(changes):
    lib, ctx = lib_and_context()
    assert lib.vetrast_select_kept(ctx, C.byref(select_args(**changes)), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_select_kept(None, C.byref(select_args()), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_select_kept(ctx, None, None) == abi.ERR_INVALID_ARG


def test_select_workspaces():
    lib, ctx = lib_and_context()
    need = lib.vetrast_select_kept_workspace_bytes
    assert need(1, 32768) == 0 and need(0, 1 << 20) == 0 and need(5, -1) == 0
    assert need(1, 32769) >= 3 * 2048 * 4 and need(7, 1 << 20) == 7 * need(1, 1 << 20) and need(1, (1 << 31) - 1) < 1 << 20
    assert need((1 << 31) - 1, (1 << 31) - 1) == ((1 << 31) - 1) * need(1, (1 << 31) - 1)
    a = select_args(n=100_000, row_stride=100_000, workspace_bytes=need(3, 100_000) - 1)
    assert lib.vetrast_select_kept(ctx, C.byref(a), None) == abi.ERR_WORKSPACE_SMALL
    assert lib.vetrast_select_kept(ctx, C.byref(select_args(rows=0, score=None, index=None, count=None)), None) == abi.OK


def keep_args(t_changes=(), **changes):
    t, a = abi.KeepTensor(), abi.KeepArgs()
    t.src, t.dst, t.outers, t.n, t.row_bytes, t.src_outer_bytes, t.src_row_bytes = AT, 2 * AT, 4, 100, 16, 1600, 16
    a.num_tensors, a.index_rows, a.kept, a.index_row_stride, a.index = 1, 2, 10, 10, AT
    for k, v in changes.items():
        setattr(a, k, v)
    for k, v in dict(t_changes).items():
        setattr(t, k, v)
    a.tensors = C.pointer(t) if changes.get("tensors", 1) else None
    return a


@pytest.mark.parametrize("changes", [dict(num_tensors=-1), dict(tensors=0), dict(index_rows=0), dict(kept=-1), dict(index_row_stride=9), dict(index=None),
                                     dict(index=AT + 2)])
def test_keep_refusals(changes):
    lib, ctx = lib_and_context()
    tensors = changes.pop("tensors", 1)
    a = keep_args(**changes)
    if not tensors:
        a.tensors = None
    assert lib.vetrast_keep_rows(ctx, C.byref(a), None) == abi.ERR_INVALID_ARG


@pytest.mark.parametrize("changes", [dict(outers=-2), dict(outers=3), dict(outers=1 << 31), dict(n=-1), dict(n=1 << 31), dict(row_bytes=0), dict(row_bytes=(1 << 30) + 1),
                                     dict(src_outer_bytes=-1), dict(src_row_bytes=-16), dict(src=None), dict(dst=None), dict(dst=AT), dict(dst=AT + 6399),
                                     dict(dst=AT - 639), dict(src_outer_bytes=1 << 60), dict(src_row_bytes=1 << 62), dict(outers=1 << 30, row_bytes=1 << 20)])
def test_keep_refusals_of_a_tensor(changes):
    lib, ctx = lib_and_context()
    assert lib.vetrast_keep_rows(ctx, C.byref(keep_args(changes)), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_keep_rows(None, C.byref(keep_args()), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_keep_rows(ctx, None, None) == abi.ERR_INVALID_ARG


def test_nothing_to_keep_is_done():
    lib, ctx = lib_and_context()
    assert lib.vetrast_keep_rows(ctx, C.byref(keep_args(num_tensors=0)), None) == abi.OK
    assert lib.vetrast_keep_rows(ctx, C.byref(keep_args(kept=0, index=None)), None) == abi.OK
    assert lib.vetrast_keep_rows(ctx, C.byref(keep_args(dict(outers=0, src=None, dst=None))), None) == abi.OK


def test_tensors_on_the_host_are_refused():
    with pytest.raises(RuntimeError, match="on the GPU"):
        torch_ops.select_kept(torch.zeros(5), 3)
    with pytest.raises(RuntimeError, match="on the GPU"):
        torch_ops.keep_rows([torch.zeros(5)], torch.zeros(3, dtype=torch.int32), [0])
    for bad in (dict(budget=-1), dict(budget=1 << 31), dict(budget=3, recent=4), dict(budget=3, recent=-1)):
        with pytest.raises(RuntimeError, match="budget|recent"):
            torch_ops.select_kept(torch.zeros(5), **bad)


def test_the_model():
    nan = float("nan")
    index, count = em.select_kept(np.array([[1, nan, 0, -0.0, 5, 0, 2]]), 4, recent=1)
    assert index.tolist() == [[0, 2, 4, 6]] and count.tolist() == [4]
    index, count = em.select_kept(np.array([[1.0, 2, 3]] * 4), 2, length=[0, 1, 2, 9])
    assert index.tolist() == [[-1, -1], [0, -1], [0, 1], [1, 2]] and count.tolist() == [0, 1, 2, 2]
    assert em.keep_rows(np.arange(6).reshape(2, 3), np.array([2, -1, 0, 3]), 1).tolist() == [[2, 0, 0, 0], [5, 0, 3, 0]]


@pytest.mark.parametrize("changes", [dict(budget=2 ** 30 + 1), dict(budget=2 ** 31 - 1), dict(n=2 ** 30 + 1, row_stride=2 ** 31, workspace_bytes=2 ** 62),
                                     dict(n=2 ** 31 - 1, row_stride=2 ** 31, workspace_bytes=2 ** 62)])
def test_select_refuses_rows_whose_places_pass_32_bits(changes):
    lib, ctx = lib_and_context()
    assert lib.vetrast_select_kept(ctx, C.byref(select_args(**changes)), None) == abi.ERR_INVALID_ARG


def test_the_calls_on_tensors_refuse_a_budget_that_passes_32_bits():
    with pytest.raises(RuntimeError, match="budget"):
        torch_ops.select_kept(torch.zeros(5), 2 ** 30 + 1)
