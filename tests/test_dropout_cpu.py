"""Dropout's entry points without a GPU: layout of the struct, what is refused, and the generator against published values."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from tests import entries_model as em
from vet_amd import abi, torch_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONTEXT = C.create_string_buffer(1 << 16)  # refusals come before anything reads it
AT = 1 << 20  # an address that is never read: these calls are refused before


def compare_layout(tmp_path, pairs):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "vetrast.h"', 'int main(void) {']
    for name, mirror in pairs:
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {field} %zu\\n", offsetof({name}, {field}));' for field, _ in mirror._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for name, mirror in pairs:
        assert got[(name, "size")] == C.sizeof(mirror), name
        for field, _ in mirror._fields_:
            assert got[(name, field)] == getattr(mirror, field).offset, (name, field)


def test_every_struct_field_sits_where_the_c_compiler_puts_it(tmp_path):
    compare_layout(tmp_path, [("vetrast_dropout_args", abi.DropoutArgs)])


def test_the_generator_gives_the_published_values():
    # known answers of Philox4x32 with ten and with seven rounds
    zeros, ones = [np.zeros(1, np.uint64)] * 4, [np.full(1, em.M32, np.uint64)] * 4
    words = [int(w[0]) for w in em.philox4x32(zeros, (0, 0), 10)]
    assert words == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    words = [int(w[0]) for w in em.philox4x32(ones, (em.M32, em.M32), 10)]
    assert words == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    words = [int(w[0]) for w in em.philox4x32(zeros, (0, 0), 7)]
    assert words == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]


def args(**changes):
    a = abi.DropoutArgs()
    a.x, a.y, a.n, a.type, a.p = AT, AT + 64, 16, abi.F32, 0.1
    for k, v in changes.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("changes", [dict(n=-1), dict(n=(1 << 38) + 1), dict(type=3), dict(type=-1), dict(p=-1e-9), dict(p=1.0 + 1e-9), dict(p=float("nan")),
                                     dict(x=None), dict(y=None), dict(x=AT + 2), dict(y=AT + 66), dict(residual=AT + 1), dict(device_step=AT + 4),
                                     dict(y=AT + 60), dict(y=AT - 4), dict(residual=AT + 68)])
def test_refusals(changes):
    lib, ctx = abi.load_library(), C.addressof(CONTEXT)
    assert lib.vetrast_dropout(ctx, C.byref(args(**changes)), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_dropout(None, C.byref(args()), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_dropout(ctx, None, None) == abi.ERR_INVALID_ARG


def test_nothing_to_do_is_done():
    lib, ctx = abi.load_library(), C.addressof(CONTEXT)
    assert lib.vetrast_dropout(ctx, C.byref(args(n=0, x=None, y=None)), None) == abi.OK


@pytest.mark.parametrize("p", [-0.1, 1.5, float("nan")])
def test_probabilities_are_looked_at_first(p):
    with pytest.raises(RuntimeError, match="p lies in"):
        torch_ops.dropout(torch.zeros(3), p, seed=1)


def test_tensors_on_the_host_are_refused():
    with pytest.raises(RuntimeError, match="on the GPU"):
        torch_ops.dropout(torch.zeros(3), 0.1, seed=1)
    with pytest.raises(TypeError):
        torch_ops.dropout(torch.zeros(3), 0.1, seed=-1)
