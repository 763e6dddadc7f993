"""vetrast_point_weights and the points' drop-out without a GPU: layout of the structs and what is refused."""
import ctypes as C

import pytest

from tests.test_dropout_cpu import AT, CONTEXT, compare_layout
from vet_amd import abi, synthetic
from vet_amd.rasterizer import fill_forward_args, make_params, make_views


def test_every_struct_field_sits_where_the_c_compiler_puts_it(tmp_path):
    compare_layout(tmp_path, [("vetrast_point_weights_args", abi.PointWeightsArgs), ("vetrast_forward_args", abi.ForwardArgs)])


def forward_args(**changes):
    scene = synthetic.tiny_scene()
    a = abi.ForwardArgs()
    params = make_params(scene)
    views = make_views(scene)
    fill_forward_args(a, scene, params, views, lambda name: None if name in ("index", "dropout") else AT)
    a.save_for_backward, a.workspace, a.workspace_bytes = 1, AT, 1 << 60
    for l in range(scene.num_layers):
        a.out[l] = AT
    for k, v in changes.items():
        if hasattr(a.params, k):
            setattr(a.params, k, v)
        else:
            setattr(a, k, v)
    return a, views


@pytest.mark.parametrize("changes", [dict(save_for_backward=0), dict(position=None), dict(workspace=None), dict(workspace=AT + 16), dict(num_views=0)])
def test_weights_of_a_call_that_is_none(changes):
    lib, ctx = abi.load_library(), C.addressof(CONTEXT)
    w = abi.PointWeightsArgs()
    a, views = forward_args(**changes)
    C.memmove(C.byref(w.fwd), C.byref(a), C.sizeof(a))
    w.weight, w.decay = AT, 1.0
    assert lib.vetrast_point_weights(ctx, C.byref(w), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_point_weights(None, C.byref(w), None) == abi.ERR_INVALID_ARG
    assert lib.vetrast_point_weights(ctx, None, None) == abi.ERR_INVALID_ARG


@pytest.mark.parametrize("weight, decay", [(None, 1.0), (AT + 2, 1.0), (AT, -0.5), (AT, float("nan")), (AT, float("inf"))])
def test_weights_and_decays_that_are_refused(weight, decay):
    lib, ctx = abi.load_library(), C.addressof(CONTEXT)
    w = abi.PointWeightsArgs()
    a, views = forward_args()
    C.memmove(C.byref(w.fwd), C.byref(a), C.sizeof(a))
    w.weight, w.decay = weight, decay
    assert lib.vetrast_point_weights(ctx, C.byref(w), None) == abi.ERR_INVALID_ARG
    a, views = forward_args(workspace_bytes=1000)
    C.memmove(C.byref(w.fwd), C.byref(a), C.sizeof(a))
    assert lib.vetrast_point_weights(ctx, C.byref(w), None) == abi.ERR_WORKSPACE_SMALL
    a, views = forward_args(render_mode=4)
    C.memmove(C.byref(w.fwd), C.byref(a), C.sizeof(a))
    assert lib.vetrast_point_weights(ctx, C.byref(w), None) == abi.ERR_UNSUPPORTED


@pytest.mark.parametrize("changes", [dict(point_dropout=-0.1), dict(point_dropout=1.1), dict(point_dropout=float("nan")), dict(point_dropout=0.1, dropout=AT),
                                     dict(point_dropout=0.1, dropout_device_step=AT + 4)])
def test_drop_outs_that_are_refused(changes):
    lib, ctx = abi.load_library(), C.addressof(CONTEXT)
    a, views = forward_args(**changes)
    assert lib.vetrast_forward(ctx, C.byref(a), None) == abi.ERR_INVALID_ARG
    g = abi.BackwardArgs()
    C.memmove(C.byref(g.fwd), C.byref(a), C.sizeof(a))
    g.grad_texture = g.grad_confidence = g.grad_background = AT
    for l in range(3):
        g.grad_out[l] = AT
    assert lib.vetrast_backward(ctx, C.byref(g), None) == abi.ERR_INVALID_ARG
