"""The pointwise layers without a GPU: refusals of the Python calls and of the
C entry points (which validate before they touch the device), and the formulas
of the gradients against differences in 64 bits."""

from __future__ import annotations

import pytest
import torch

from fast_compressai import _native, layers
from tests import layers_reference as R

BF16, F16, F32 = 0, 1, 2


@pytest.mark.parametrize("call", [
    lambda t: layers.linear_forward(t, t),
    lambda t: layers.layer_norm_forward(t),
    lambda t: layers.activation_forward(t, "gelu"),
    lambda t: layers.save_checkpoint(t),
    lambda t: layers.linear(t, t),
    lambda t: layers.layer_norm(t),
    lambda t: layers.activation(t, "relu"),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(ValueError, match="CUDA"):
        call(torch.zeros(4, 4, dtype=torch.bfloat16))


def test_unknown_names_are_refused():
    t = torch.zeros(4, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="activation"):
        layers.linear_forward(t, t, activation="swish")
    with pytest.raises(ValueError, match="keep"):
        layers.linear_forward(t, t, keep="int4")
    with pytest.raises(ValueError, match="keep"):
        layers.linear(t, t, keep=None)
    with pytest.raises(ValueError, match="format"):
        layers.save_checkpoint(t, "full")
    with pytest.raises(ValueError, match="activation"):
        layers.activation_forward(t, "tanh")
    with pytest.raises(ValueError, match="kept"):
        layers.linear_backward(t, None, t)


def test_other_objects_are_refused():
    t = torch.zeros(4, 4, dtype=torch.bfloat16)
    for call in (lambda: layers.linear([1.0], t), lambda: layers.layer_norm(None), lambda: layers.activation(2.0, "relu")):
        with pytest.raises(ValueError, match="tensor"):
            call()


def _code(name, *args):
    return getattr(_native.lib(), name)(*args)


P = 1 << 20  # stands for a device address; no refused call reads it


def _forward(x=P, ldx=64, w=P, ldw=64, bias=None, res=None, ldr=0, y=P, ldy=32, pre=None, ldpre=0, codes=None,
             scales=None, rows=8, cin=64, cout=32, dtype=BF16, act=0, keep=0, ws=None, wsb=0):
    return _code("fcai_linear_forward", x, ldx, w, ldw, bias, res, ldr, y, ldy, pre, ldpre, codes, scales, rows, cin, cout,
                 dtype, act, keep, ws, wsb, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=F32), dict(dtype=3), dict(rows=-1), dict(rows=2 ** 31), dict(cin=0), dict(cout=0), dict(ldx=63), dict(ldw=10),
    dict(ldy=31), dict(act=4), dict(act=-1), dict(x=None), dict(w=None), dict(y=None), dict(x=P + 1), dict(res=P, ldr=8),
    dict(pre=P, ldpre=31, keep=1), dict(keep=1), dict(keep=2, codes=P), dict(keep=3, scales=P), dict(keep=4),
    dict(keep=2, codes=P, scales=P + 2), dict(rows=80, keep=2, codes=P + 4, scales=P),
    dict(rows=80, keep=2, codes=P, scales=P, y=P + 2),
])
def test_linear_refusals(bad):
    assert _forward(**bad) == _native.FCAI_ERR_INVALID
    assert _native.lib().fcai_last_error()


def test_linear_asks_for_its_workspace():
    # a row stride of 65 elements is not 16-byte aligned: x is repacked
    need = _code("fcai_linear_workspace", 0, 80, 64, 32, 1, 0)
    assert need >= 80 * 64 * 2
    assert _forward(rows=80, ldx=65, ws=None, wsb=0) == _native.FCAI_ERR_WORKSPACE
    assert _forward(rows=80, ldx=65, ws=P, wsb=need - 1) == _native.FCAI_ERR_WORKSPACE
    assert _forward(rows=80, ldx=65, ws=P + 8, wsb=need + 8) == _native.FCAI_ERR_WORKSPACE
    assert _code("fcai_linear_workspace", 3, 8, 64, 32, 0, 0) == -1
    assert _code("fcai_linear_workspace", 0, -1, 64, 32, 0, 0) == -1
    assert _code("fcai_linear_workspace", 2, 0, 64, 32, 0, 0) == 0


def test_no_rows_need_no_device():
    assert _forward(rows=0) == 0
    assert _code("fcai_activation_forward", None, 8, None, 8, None, None, 0, 8, BF16, 2, 2, None) == 0
    assert _code("fcai_layer_norm_forward", None, 8, None, None, BF16, None, 8, None, None, None, None, 0, 8, 1e-5, BF16, 0,
                 None) == 0
    assert _code("fcai_checkpoint_load", None, None, None, 8, 0, 8, F32, 2, None) == 0
    assert _code("fcai_linear_backward_input", None, 8, None, 8, None, 8, 0, 8, 8, BF16, None, 0, None) == 0


@pytest.mark.parametrize("name,args", [
    ("fcai_linear_backward_input", (P, 31, P, 64, P, 64, 8, 64, 32, BF16, None, 0, None)),      # dp's stride
    ("fcai_linear_backward_weight", (P, 32, P, 63, P, 64, 8, 64, 32, BF16, None, 0, None)),     # x's stride
    ("fcai_linear_backward_weight", (P, 32, P, 64, None, 64, 8, 64, 32, BF16, None, 0, None)),  # no dw
    ("fcai_activation_forward", (P, 8, P, 8, None, None, 4, 8, BF16, 2, 2, None)),              # int8 without codes
    ("fcai_activation_forward", (P, 8, None, 8, None, None, 4, 8, BF16, 2, 0, None)),           # nothing to write
    ("fcai_activation_forward", (P, 8, P, 8, P, P, 4, 8, BF16, 2, 5, None)),
    ("fcai_activation_forward", (P, 7, P, 8, None, None, 4, 8, BF16, 2, 0, None)),
    ("fcai_activation_forward", (P + 2, 8, P, 8, None, None, 4, 8, F32, 2, 0, None)),
    ("fcai_activation_forward", (P, 8, P, 8, None, None, 4, 0, BF16, 2, 0, None)),
    ("fcai_activation_backward", (P, 8, None, 8, None, None, P, 8, None, 4, 8, BF16, 2, 1, None, 0, None)),  # no x
    ("fcai_activation_backward", (P, 8, P, 8, None, None, None, 8, None, 4, 8, BF16, 2, 1, None, 0, None)),  # no output
    ("fcai_activation_backward", (P, 8, P, 8, None, None, P, 8, None, 4, 8, BF16, 2, 0, None, 0, None)),     # keep none
    ("fcai_checkpoint_load", (P, P, P, 8, 4, 8, BF16, 1, None)),
    ("fcai_checkpoint_load", (P, P + 1, P, 8, 4, 8, BF16, 2, None)),
    ("fcai_layer_norm_forward", (P, 8, P, P, F16, P, 8, None, None, None, None, 4, 8, 1e-5, BF16, 0, None)),
    ("fcai_layer_norm_forward", (P, 8, P, P, BF16, P, 8, P, None, None, None, 4, 8, 1e-5, BF16, 0, None)),
    ("fcai_layer_norm_forward", (P, 8, P, P, BF16, P, 8, None, None, None, None, 4, 8, -1.0, BF16, 0, None)),
    ("fcai_layer_norm_forward", (P, 8, P, P, BF16, P, 8, None, None, None, None, 4, 8, float("nan"), BF16, 0, None)),
    ("fcai_layer_norm_forward", (P, 8, P, P, BF16, P, 8, None, None, None, None, 4, 8, 1e-5, BF16, 2, None)),
    ("fcai_layer_norm_backward", (P, 8, P, 8, None, None, None, None, None, BF16, P, 8, None, None, 4, 8, BF16, 1, P, 1 << 20, None)),
    ("fcai_layer_norm_backward", (P, 8, P, 8, None, None, P, P, None, BF16, None, 8, None, None, 4, 8, BF16, 1, P, 1 << 20, None)),
])
def test_c_refusals(name, args):
    assert _code(name, *args) == _native.FCAI_ERR_INVALID, _native.lib().fcai_last_error()


def test_row_kernels_ask_for_their_workspace():
    need = _code("fcai_layer_norm_workspace", 100, 40)
    args = (P, 40, P, 40, None, None, P, P, None, BF16, P, 40, P, P, 100, 40, BF16, 1)
    assert _code("fcai_layer_norm_backward", *args, None, 0, None) == _native.FCAI_ERR_WORKSPACE
    assert _code("fcai_layer_norm_backward", *args, P, need - 1, None) == _native.FCAI_ERR_WORKSPACE
    need = _code("fcai_activation_workspace", 100, 40)
    args = (P, 40, None, 0, None, None, None, 40, P, 100, 40, BF16, 0, 1)
    assert _code("fcai_activation_backward", *args, P, need - 1, None) == _native.FCAI_ERR_WORKSPACE
    assert _code("fcai_layer_norm_workspace", -1, 40) == -1 and _code("fcai_activation_workspace", 4, 0) == -1


@pytest.mark.parametrize("kind", layers.ACTIVATIONS)
def test_activation_derivative_against_differences(kind):
    p = torch.linspace(-9, 9, 181, dtype=torch.float64) + 0.013
    h = 1e-5
    diff = (R.act64(p + h, kind) - R.act64(p - h, kind)) / (2 * h)
    # third derivatives are below 2: h^2 / 3, and cancellation at 2^-52 * 9 / h
    assert torch.allclose(diff, R.act_grad64(p, kind), atol=1e-9, rtol=0)


def test_linear_formula_against_differences():
    torch.manual_seed(0)
    x, w, b, dy = torch.randn(5, 7).double(), torch.randn(6, 7).double(), torch.randn(6).double(), torch.randn(5, 6).double()
    p, _ = R.linear64(x, w, b)
    (dx, _), (dw, _), (db, _) = R.linear_grads(dy, x, w, p, "gelu", torch.bfloat16)
    h = 1e-6

    def value(x, w, b):
        return (R.linear64(x, w, b, None, "gelu")[1] * dy).sum()

    for t, g, put in ((x, dx, lambda v: value(v, w, b)), (w, dw, lambda v: value(x, v, b)), (b, db, lambda v: value(x, w, v))):
        v = torch.randn_like(t)
        diff = (put(t + h * v) - put(t - h * v)) / (2 * h)
        assert abs(float(diff - (g * v).sum())) < 1e-7


def test_norm_formula_against_differences():
    torch.manual_seed(1)
    x, w, b, dy = torch.randn(4, 9).double(), torch.randn(9).double(), torch.randn(9).double(), torch.randn(4, 9).double()
    (dx, _), (dw, _), (db, _) = R.norm_grads(dy, x, x, w, 1e-3, torch.float32, torch.float32)
    h = 1e-6

    def value(x, w, b):
        return (R.norm64(x, w, b, 1e-3, torch.float32)[0] * dy).sum()

    for t, g, put in ((x, dx, lambda v: value(v, w, b)), (w, dw, lambda v: value(x, v, b)), (b, db, lambda v: value(x, w, v))):
        v = torch.randn_like(t)
        diff = (put(t + h * v) - put(t - h * v)) / (2 * h)
        assert abs(float(diff - (g * v).sum())) < 1e-7


@pytest.mark.parametrize("bad", [
    dict(bias=P + 1), dict(res=P + 1, ldr=32), dict(res=P, ldr=2 ** 37), dict(keep=1, pre=P + 1, ldpre=32),
    dict(keep=1, pre=P, ldpre=2 ** 37),
])
def test_linear_refuses_pointers_of_its_options(bad):
    assert _forward(**bad) == _native.FCAI_ERR_INVALID
