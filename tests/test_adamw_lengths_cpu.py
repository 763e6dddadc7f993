"""Lengths that no memory has are refused by every call over a list, and give no workspace."""
import ctypes as C

import pytest

from tests.test_adamw_cpu import AT, norm_args, step_args
from vet_amd import abi

LENGTHS = [(1 << 38) + 1, 1 << 40, (1 << 63) - (1 << 27), (1 << 63) - 1]


@pytest.mark.parametrize("n", LENGTHS)
def test_lengths_beyond_memory_are_refused(n):
    lib, ctx = abi.load_library(), C.addressof(C.create_string_buffer(1 << 16))
    g = abi.Gradient()
    g.n = n
    assert lib.vetrast_gradient_norm_workspace_bytes(C.byref(g), 1) == 0  # what the calls below count their launches by
    assert lib.vetrast_gradient_norm(ctx, C.byref(norm_args(t_n=n)), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_adamw_step(ctx, C.byref(step_args(t_n=n)), None) == abi.ERR_INVALID_ARG
    t, a = abi.MomentTensor(), abi.MomentsArgs()
    t.exp_avg = t.exp_avg_sq = a.exp_avg = a.exp_avg_sq = a.block_scale = AT
    t.n, a.num_tensors, a.tensors = n, 1, C.pointer(t)
    for call in (lib.vetrast_pack_moments, lib.vetrast_unpack_moments):
        assert call(ctx, C.byref(a), None) == abi.ERR_INVALID_ARG


def test_the_longest_have_a_workspace():
    g = abi.Gradient()
    g.n = 1 << 38  # 2048 entries of 2^27, 240 a launch
    one = abi.Gradient()
    one.n = 1
    lib = abi.load_library()
    assert lib.vetrast_gradient_norm_workspace_bytes(C.byref(g), 1) == lib.vetrast_gradient_norm_workspace_bytes(C.byref(one), 1) + 8 * 768 * 8
