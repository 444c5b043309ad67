"""The pointwise layers without a GPU: what happens to their calls under a
trace and in forward mode."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from fast_compressai import _native, layers


class _PlainHost:
    """Stands for the compiled calls: like them it writes its results past torch's dispatcher."""

    def linear_forward(self, x, w, b, r, act, keep):
        assert torch._C._get_tracing_state() is None
        y = torch.from_numpy(x.detach().numpy() @ w.detach().numpy().T)
        return y if keep == 0 else (y, None)

    def layer_norm_forward(self, x, w, b, eps, keep):
        assert torch._C._get_tracing_state() is None
        v = x.detach().numpy()
        y = torch.from_numpy((v - v.mean(-1, keepdims=True)) / (v.var(-1, keepdims=True) + eps) ** 0.5)
        return y if keep == 0 else (y, torch.zeros(2, x.shape[0]))

    def activation_forward(self, x, act, keep):
        assert torch._C._get_tracing_state() is None
        y = torch.from_numpy(x.detach().numpy().clip(min=0))
        return y if keep < 2 else (y, torch.zeros(x.shape, dtype=torch.uint8), torch.zeros(x.shape[0], 1))


CALLS = {
    "linear": lambda x, w: layers.linear(x, w),
    "layer_norm": lambda x, w: layers.layer_norm(x),
    "activation": lambda x, w: layers.activation(x, "relu"),
}


@pytest.mark.parametrize("name", CALLS)
def test_a_trace_holds_the_call_not_its_result(monkeypatch, name):
    monkeypatch.setattr(layers, "_host", _PlainHost())
    call = CALLS[name]
    x, w = torch.randn(3, 8), torch.randn(8, 8)
    traced = torch.jit.trace(lambda q: call(q, w) + q, (x,), check_trace=False)
    z = torch.randn(3, 8)
    assert torch.equal(traced(z), call(z, w) + z)


EXPLICIT = {
    "linear_forward": lambda x: layers.linear_forward(x, x),
    "linear_forward with keep": lambda x: layers.linear_forward(x, x, keep="int8")[0],
    "layer_norm_forward": lambda x: layers.layer_norm_forward(x),
    "activation_forward": lambda x: layers.activation_forward(x, "gelu"),
    "save_checkpoint": lambda x: layers.save_checkpoint(x).codes,
}


@pytest.mark.parametrize("name", EXPLICIT)
def test_explicit_calls_refuse_a_trace(name):
    x = torch.randn(4, 4)
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda q: EXPLICIT[name](q) + q, (x,), check_trace=False)
    assert torch._C._get_tracing_state() is None


@pytest.mark.parametrize("name", [*EXPLICIT, *CALLS])
def test_a_graph_of_recorded_operations_is_refused(name):
    x = torch.randn(4, 4)
    call = EXPLICIT.get(name) or (lambda q: CALLS[name](q, q))
    with pytest.raises(ValueError, match="traced"):
        make_fx(lambda q: call(q) + q)(x)


@pytest.mark.parametrize("name", [*EXPLICIT, *CALLS])
def test_forward_mode_is_refused(name):
    x = torch.randn(4, 4)
    call = EXPLICIT.get(name) or (lambda q: CALLS[name](q, q))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="tangent"):
            call(dual)
        with pytest.raises(ValueError, match="CUDA"):  # a dual level alone changes nothing
            call(x)


def test_check_takes_a_cuda_device():
    with pytest.raises(ValueError, match="CUDA"):
        layers.check("cpu")


def test_nothing_is_kept_in_fewer_bits_unless_asked(monkeypatch):
    asked = []

    class Host(_PlainHost):
        def linear_forward(self, x, w, b, r, act, keep):
            asked.append(keep)
            return super().linear_forward(x, w, b, r, act, keep)

        def layer_norm_forward(self, x, w, b, eps, keep):
            asked.append(keep)
            return super().layer_norm_forward(x, w, b, eps, keep)

        def activation_forward(self, x, act, keep):
            asked.append(keep)
            return super().activation_forward(x, act, keep)

    monkeypatch.setattr(layers, "_host", Host())
    x = torch.randn(3, 8, requires_grad=True)
    for call in CALLS.values():
        call(x, torch.randn(8, 8))
    assert asked == [1, 1, 1]


@pytest.mark.parametrize("keep", [2, 3])
@pytest.mark.parametrize("rows,cin,cout", [(147456, 128, 520), (36864, 192, 1032), (1 << 20, 16, 2056), (70001, 64, 333),
                                           (300, 64, 65), (33, 8, 100001), (5000, 24, 100008)])
def test_scratch_of_products_kept_in_8_bits(rows, cin, cout, keep):
    bytes_ = _native.lib().fcai_linear_workspace(0, rows, cin, cout, 0, keep)
    # fp32 values of small or split products, or the codes once more
    assert 0 <= bytes_ <= max(32 << 20, rows * (cout + 15) + 256)
    # unaligned operands add their copies, nothing else
    more = _native.lib().fcai_linear_workspace(0, rows, cin, cout, 3, keep)
    assert more - bytes_ <= 2 * (rows + cout) * (cin + 7) + 512
