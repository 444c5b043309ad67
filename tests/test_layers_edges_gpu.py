"""The pointwise layers on the B200 at the edges of what they take: infinities
and values that leave the type's range, rows beside other rows, constant rows,
waits that ran out, large matrices, and calls at the same time."""

from __future__ import annotations

import pytest
import torch

from fast_compressai import layers
from tests import layers_reference as R
from tests.test_layers_gpu import _randn

pytestmark = pytest.mark.gpu

INF = float("inf")
T16 = [torch.bfloat16, torch.float16]
T3 = T16 + [torch.float32]


@pytest.mark.parametrize("dtype", T3)
@pytest.mark.parametrize("kind", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("n", [8, 7])
def test_activation_gradient_at_infinities(cuda_device, dtype, kind, n):
    # the limits: 0 on the left, 1 on the right
    x = torch.tensor([[-INF, INF, -60000.0, 60000.0, -INF, 1.0, INF, -INF]], device="cuda").to(dtype)[:, :n]
    _, saved = layers.activation_forward(x, kind, keep="full")
    dx = layers.activation_backward(torch.full_like(x, 3.0), saved)
    far = x.abs() > 1
    assert torch.equal(dx[far], (3.0 * (x > 0)).to(dtype)[far])
    assert dx.isfinite().all()


@pytest.mark.parametrize("kind", ["relu", "gelu", "silu"])
def test_linear_gradients_where_the_activation_input_leaves_fp16(cuda_device, kind):
    x = torch.full((40, 64), 100.0, dtype=torch.float16, device="cuda")
    x[::3] *= -1
    w = torch.full((24, 64), 16.0, dtype=torch.float16, device="cuda")  # |p| = 102400
    dy = _randn(40, 24, dtype=torch.float16, seed=4)
    y, saved = layers.linear_forward(x, w, activation=kind, keep="full")
    assert saved.pre.isinf().all()
    p64, _ = R.linear64(x, w)
    for name, got, (g, e) in zip(("dx", "dw"), layers.linear_backward(dy, saved, w),
                                 R.linear_grads(dy, x, w, p64, kind, torch.float16)):
        R.check(got, g, e, name)
