"""The optimiser's entry points without a GPU: layout of their structs, what they refuse, sizes of workspaces, and the format of 8-bit
moments against its own definition."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from tests import optim_model as om
from vet_amd import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 4096  # an address that is never read: these calls are refused before


@pytest.fixture(scope="module")
def lib():
    return abi.load_library()


@pytest.fixture(scope="module")
def ctx():
    return C.addressof(C.create_string_buffer(1 << 16))  # refusals come before anything reads it


def test_every_struct_field_sits_where_the_c_compiler_puts_it(tmp_path):
    pairs = [("vetrast_adamw_tensor", abi.AdamWTensor), ("vetrast_adamw_group", abi.AdamWGroup), ("vetrast_adamw_args", abi.AdamWArgs),
             ("vetrast_adamw_device_state", abi.AdamWDeviceState), ("vetrast_gradient", abi.Gradient),
             ("vetrast_gradient_norm_args", abi.GradientNormArgs), ("vetrast_moment_tensor", abi.MomentTensor),
             ("vetrast_moments_args", abi.MomentsArgs)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "vetrast.h"', 'int main(void) {']
    for name, mirror in pairs:
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {field} %zu\\n", offsetof({name}, {field}));' for field, _ in mirror._fields_]
    lines += ['printf("constants block %d\\n", VETRAST_MOMENT_BLOCK); printf("constants groups %d\\n", VETRAST_ADAMW_MAX_GROUPS);',
              'printf("constants types %d\\n", VETRAST_F32 + 10 * VETRAST_BF16 + 100 * VETRAST_F16);', 'return 0; }']
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for name, mirror in pairs:
        assert got[(name, "size")] == C.sizeof(mirror), name
        for field, _ in mirror._fields_:
            assert got[(name, field)] == getattr(mirror, field).offset, (name, field)
    assert got[("constants", "block")] == abi.MOMENT_BLOCK == om.BLOCK and got[("constants", "groups")] == abi.ADAMW_MAX_GROUPS
    assert got[("constants", "types")] == abi.F32 + 10 * abi.BF16 + 100 * abi.F16


def step_args(bits=8, **changes):
    t, g, a = abi.AdamWTensor(), abi.AdamWGroup(), abi.AdamWArgs()
    t.param = t.grad = a.exp_avg = a.exp_avg_sq = a.block_scale = AT
    t.n = 10
    g.lr, g.step = 1e-3, 1
    a.num_tensors = a.num_groups = 1
    a.beta1, a.beta2, a.eps, a.moment_bits = 0.9, 0.999, 1e-8, bits
    for k, v in changes.items():
        where, name = k.split("_", 1)
        setattr({"t": t, "g": g, "a": a}[where], name, v)
    a.tensors, a.groups = C.pointer(t), C.pointer(g)
    a._keep = (t, g)
    return a


@pytest.mark.parametrize("change", [
    dict(a_num_tensors=-1), dict(a_num_groups=-1), dict(a_num_groups=abi.ADAMW_MAX_GROUPS + 1), dict(a_num_groups=0),
    dict(a_moment_bits=16), dict(a_moment_bits=0), dict(a_beta1=1.0), dict(a_beta1=-0.1), dict(a_beta1=float("nan")), dict(a_beta2=1.0),
    dict(a_beta2=float("nan")), dict(a_eps=0.0), dict(a_eps=-1e-8), dict(a_eps=float("nan")), dict(a_eps=float("inf")), dict(a_eps=1e-60),
    dict(a_eps=1e-39), dict(a_grad_scale=AT + 2), dict(a_device_state=AT + 8), dict(g_step=0), dict(g_step=-3), dict(g_lr=float("nan")),
    dict(g_lr=float("inf")), dict(g_weight_decay=float("nan")), dict(t_n=-1), dict(t_group=1), dict(t_group=-1), dict(t_param_type=3),
    dict(t_param_type=-1), dict(t_grad_type=3), dict(t_first=-128), dict(t_first=64), dict(t_first=1 << 38), dict(t_n=(1 << 38) + 1),
    dict(t_param=None), dict(t_grad=None), dict(a_exp_avg=None), dict(a_exp_avg_sq=None), dict(a_block_scale=None), dict(t_param=AT + 2),
    dict(t_grad=AT + 2), dict(t_param=AT + 1, t_param_type=1), dict(t_grad=AT + 1, t_grad_type=2), dict(a_exp_avg=AT + 8),
    dict(a_exp_avg_sq=AT + 4), dict(a_block_scale=AT + 2), dict(a_master=AT + 4)], ids=str)
def test_step_refuses(change, lib, ctx):
    assert lib.vetrast_adamw_step(ctx, C.byref(step_args(**change)), None) == abi.ERR_INVALID_ARG


def test_step_refuses_in_32_bits_too(lib, ctx):
    for change in (dict(a_exp_avg=AT + 8), dict(a_exp_avg_sq=AT + 1), dict(a_exp_avg=None), dict(t_param=None)):
        assert lib.vetrast_adamw_step(ctx, C.byref(step_args(bits=32, **change)), None) == abi.ERR_INVALID_ARG
    a = step_args()
    a.tensors = None
    assert lib.vetrast_adamw_step(ctx, C.byref(a), None) == abi.ERR_INVALID_ARG
    a = step_args()
    a.groups = None
    assert lib.vetrast_adamw_step(ctx, C.byref(a), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_adamw_step(None, C.byref(step_args()), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_adamw_step(ctx, None, None) == abi.ERR_INVALID_ARG


def test_device_state_bytes(lib):
    assert lib.vetrast_adamw_device_state_bytes(0) == 16 == C.sizeof(abi.AdamWDeviceState)
    assert lib.vetrast_adamw_device_state_bytes(3) == 16 + 3 * 16
    assert lib.vetrast_adamw_device_state_bytes(-1) == lib.vetrast_adamw_device_state_bytes(abi.ADAMW_MAX_GROUPS + 1) == 0


def norm_args(**changes):
    g, a = abi.Gradient(), abi.GradientNormArgs()
    g.grad, g.n = AT, 10
    a.num_gradients, a.scale, a.out, a.workspace, a.workspace_bytes = 1, 1.0, AT, AT, 1 << 30
    for k, v in changes.items():
        where, name = k.split("_", 1)
        setattr({"t": g, "a": a}[where], name, v)
    a.gradients = C.pointer(g)
    a._keep = g
    return a


@pytest.mark.parametrize("change", [
    dict(a_num_gradients=-1), dict(a_out=None), dict(a_out=AT + 2), dict(a_workspace=None), dict(a_workspace=AT + 8),
    dict(a_scale=float("nan")), dict(a_scale=float("inf")), dict(a_max_norm=float("nan")), dict(t_n=-1), dict(t_type=3), dict(t_type=-1),
    dict(t_grad=None), dict(t_grad=AT + 2), dict(t_grad=AT + 1, t_type=1)], ids=str)
def test_norm_refuses(change, lib, ctx):
    assert lib.vetrast_gradient_norm(ctx, C.byref(norm_args(**change)), None) == abi.ERR_INVALID_ARG


def test_norm_workspace(lib, ctx):
    one = abi.Gradient()
    one.n = 10
    need = lib.vetrast_gradient_norm_workspace_bytes(C.byref(one), 1)
    assert need > 0 and lib.vetrast_gradient_norm_workspace_bytes(None, 0) > 0
    assert lib.vetrast_gradient_norm_workspace_bytes(None, 1) == lib.vetrast_gradient_norm_workspace_bytes(C.byref(one), -1) == 0
    one.n = -1
    assert lib.vetrast_gradient_norm_workspace_bytes(C.byref(one), 1) == 0
    many = (abi.Gradient * 1000)()
    for g in many:
        g.n = 1 << 33
    assert lib.vetrast_gradient_norm_workspace_bytes(many, 1000) > 60 * (need - 4096)  # 16 entries each, 240 a launch
    a = norm_args(a_workspace_bytes=need - 1)
    assert lib.vetrast_gradient_norm(ctx, C.byref(a), None) == abi.ERR_WORKSPACE_SMALL
    a.gradients = None
    assert lib.vetrast_gradient_norm(ctx, C.byref(a), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_gradient_norm(None, C.byref(norm_args()), None) == lib.vetrast_gradient_norm(ctx, None, None) == abi.ERR_INVALID_ARG


@pytest.mark.parametrize("change", [
    dict(t_n=-1), dict(t_exp_avg=None), dict(t_exp_avg_sq=None), dict(t_exp_avg=AT + 2), dict(t_exp_avg_sq=AT + 1), dict(t_first=-128),
    dict(t_first=100), dict(t_first=1 << 38), dict(a_exp_avg=None), dict(a_exp_avg_sq=None), dict(a_block_scale=None), dict(a_exp_avg=AT + 8),
    dict(a_exp_avg_sq=AT + 4), dict(a_block_scale=AT + 2), dict(a_num_tensors=-1), dict(a_tensors=None)], ids=str)
def test_conversions_refuse(change, lib, ctx):
    t, a = abi.MomentTensor(), abi.MomentsArgs()
    t.exp_avg = t.exp_avg_sq = a.exp_avg = a.exp_avg_sq = a.block_scale = AT
    t.n, a.num_tensors, a.tensors = 10, 1, C.pointer(t)
    for k, v in change.items():
        where, name = k.split("_", 1)
        setattr({"t": t, "a": a}[where], name, v)
    for call in (lib.vetrast_pack_moments, lib.vetrast_unpack_moments):
        assert call(ctx, C.byref(a), None) == abi.ERR_INVALID_ARG
        assert call(None, C.byref(a), None) == call(ctx, None, None) == abi.ERR_INVALID_ARG


@pytest.mark.parametrize("size", [1e-44, 1e-38, 1e-20, 1.0, 1.9374999, 1.9375, 1.9999999, 1e30, 3.4e38])
def test_codes_fit_and_hold_their_precision(size):
    """The format itself, on the CPU: codes stay within 7 and 8 bits for every largest value and every rounding, and stand for what
    they were made from to a step of an eighth of (value + offset)."""
    rng = np.random.default_rng(4)
    m = (size * np.exp(-rng.exponential(4, 128 * 40)) * rng.choice([-1, 1], 128 * 40)).astype(np.float32)
    m.reshape(-1, 128)[:, 7] = np.float32(size)
    v = np.abs(m) * rng.random(m.size).astype(np.float32)
    v.reshape(-1, 128)[:, 9] = np.float32(size)
    for r in (0, 1 << 19, (1 << 20) - 1):
        bits = np.full(m.size, r)
        mc, vc, scale = om.encode(m, v, bits, bits)
        dm, dv = om.decode(mc, vc, scale)
        if size > 3.19e38:  # a code next to it would be infinite: reads as overflowed
            assert np.isnan(dm).all() and np.isnan(dv).all() and (scale == 255).all()
            continue
        for x, y, k in ((m, dm, 0), (v, dv, 1)):
            unit = np.repeat(np.exp2(scale[:, k] - 127.0), 128)
            assert (np.abs(x.astype(np.float64) - y) <= (np.abs(x.astype(np.float64)) + unit) / 8 * 1.000001).all()
            assert k == 1 or (np.sign(x) * y >= 0).all()


def test_random_rounding_is_what_second_moments_need():
    """A second moment of constant expectation, held in 8 bits: rounded by random bits it stays with the one in 64 bits on average,
    rounded to nearest it does not (why the format comes with random bits)."""
    rng = np.random.default_rng(6)
    steps, n = 600, 128 * 16
    sigma = np.exp(rng.normal(0, 1, n))
    exact = np.zeros(n)
    held = {True: np.zeros(n, np.float32), False: np.zeros(n, np.float32)}
    for step in range(1, steps + 1):
        g = (rng.standard_normal(n) * sigma).astype(np.float32)
        exact = 0.99 * exact + 0.01 * g.astype(np.float64) ** 2
        for by_bits, v in held.items():
            _, v = om.moments_in_float(v, v, g, 0.9, 0.99)
            rm, rv, _ = om.random_bits(3, step, 0, n)
            rv = rv if by_bits else np.full(n, 1 << 19)
            mc, vc, scale = om.encode(np.zeros(n, np.float32), v, rv, rv)
            held[by_bits] = om.decode(mc, vc, scale)[1].astype(np.float32)
    ratio = {k: np.mean(v / exact) for k, v in held.items()}
    # a random walk of steps of 1/16..1/8 that is pulled back at a rate of 1/100: 10 % an element, 0.3 % the mean of 2048
    assert abs(ratio[True] - 1) < 0.02 and abs(ratio[False] - 1) > 0.05
