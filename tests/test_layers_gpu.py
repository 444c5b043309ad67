"""The pointwise layers on the B200 against their plain forms in 64 bits
(tests/layers_reference.py, which derives each bound)."""

from __future__ import annotations

import pytest
import torch

from fast_compressai import layers
from fast_compressai.layers import Checkpoint8
from tests import layers_reference as R

pytestmark = pytest.mark.gpu

T16 = [torch.bfloat16, torch.float16]
T3 = T16 + [torch.float32]


def _randn(*shape, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 17 * sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _sliced(t, pad=3):
    """The same values inside a wider matrix, at an odd offset: rows that are not 16-byte aligned."""
    big = torch.full((t.shape[0], t.shape[1] + 2 * pad + 1), float("nan"), dtype=t.dtype, device=t.device)
    view = big[:, pad:pad + t.shape[1]]
    view.copy_(t)
    return view


# ------------------------------------------------------------------------ linear

SHAPES = [(1, 8, 1), (1, 64, 8), (1, 4096, 512), (2, 200, 131), (3, 17, 40), (8, 1000, 72), (16, 512, 264), (17, 96, 33),
          (24, 1024, 4096), (31, 520, 64), (63, 40, 200), (64, 2048, 128), (100, 65, 65), (127, 64, 128), (129, 321, 577),
          (200, 72, 16), (256, 256, 256), (300, 513, 384), (1000, 192, 768), (2049, 128, 520), (4100, 1032, 24),
          (777, 2048, 1000), (9000, 40, 48)]


@pytest.mark.parametrize("rows,cin,cout", SHAPES)
@pytest.mark.parametrize("dtype", T16)
def test_linear_forward(cuda_device, rows, cin, cout, dtype):
    x, w = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1, scale=cin ** -0.5)
    b, r = _randn(cout, dtype=dtype, seed=2), _randn(rows, cout, dtype=dtype, seed=3)
    for i, kind in enumerate(layers.ACTIVATIONS):
        bias, res = (b if i != 1 else None), (r if i % 2 else None)
        y = layers.linear_forward(x, w, bias, activation=kind, residual=res)
        assert y.shape == (rows, cout) and y.dtype == dtype
        want, bound = R.linear_bound(x, w, bias, res, kind, dtype)
        R.check(y, want, bound, f"{kind} {rows}x{cin}x{cout}")


@pytest.mark.parametrize("rows,cin,cout", [(5, 40, 24), (1, 256, 64), (130, 72, 136), (300, 200, 88)])
@pytest.mark.parametrize("which", ["x", "w", "residual", "all"])
def test_linear_strided(cuda_device, rows, cin, cout, which):
    dtype = torch.bfloat16
    x, w = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1, scale=cin ** -0.5)
    b, r = _randn(cout + 1, dtype=dtype, seed=2)[1:], _randn(rows, cout, dtype=dtype, seed=3)
    want, bound = R.linear_bound(x, w, b, r, "gelu", dtype)
    xs = _sliced(x) if which in ("x", "all") else x
    ws = _sliced(w) if which in ("w", "all") else w
    rs = _sliced(r) if which in ("residual", "all") else r
    y, saved = layers.linear_forward(xs, ws, b, activation="gelu", residual=rs, keep="full")
    R.check(y, want, bound, which)
    dy = _randn(rows, cout, dtype=dtype, seed=4)
    grads = layers.linear_backward(_sliced(dy) if which == "all" else dy, saved, ws)
    for got, (g, e) in zip(grads, R.linear_grads(dy, x, w, saved.pre.double(), "gelu", dtype)):
        R.check(got, g, e, which)
    # aligned rows of a wider matrix, and channels that are not contiguous
    wide = torch.zeros(rows, cin + 64, dtype=dtype, device="cuda")
    wide[:, 64:] = x
    assert torch.equal(layers.linear_forward(wide[:, 64:], w, b, activation="gelu", residual=r),
                       layers.linear_forward(x, w, b, activation="gelu", residual=r))
    assert torch.equal(layers.linear_forward(x.t().contiguous().t(), w.t().contiguous().t(), b, activation="gelu", residual=r),
                       layers.linear_forward(x, w, b, activation="gelu", residual=r))


@pytest.mark.parametrize("rows,cin,cout", [(1, 64, 40), (7, 33, 65), (130, 64, 128), (129, 321, 577), (1000, 192, 320),
                                           (20000, 128, 64), (5000, 24, 8), (300, 1032, 2056), (16, 4096, 128),
                                           (70001, 16, 40), (6001, 333, 100), (901, 1001, 577), (20001, 333, 100)])
@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("kind", ["none", "relu", "gelu", "silu"])
def test_linear_backward(cuda_device, rows, cin, cout, dtype, kind):
    x, w = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1, scale=cin ** -0.5)
    b, dy = _randn(cout, dtype=dtype, seed=2), _randn(rows, cout, dtype=dtype, seed=4)
    y, saved = layers.linear_forward(x, w, b, activation=kind, keep="full")
    want, bound = R.linear_bound(x, w, b, None, kind, dtype)
    R.check(y, want, bound, "y")
    p64, _ = R.linear64(x, w, b)
    pre = p64
    if kind != "none":  # the gradient is that of the value kept, which is p rounded once
        e = (cin + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
        R.check(saved.pre, p64, e + R.half_step(dtype) * (p64.abs() + e) + R.tiny(dtype), "pre")
        pre = saved.pre.double()
    for name, got, (g, e) in zip(("dx", "dw", "db"), layers.linear_backward(dy, saved, w),
                                 R.linear_grads(dy, x, w, pre, kind, dtype)):
        R.check(got, g, e, name)


@pytest.mark.parametrize("rows,cin,cout", [(1, 64, 40), (7, 33, 65), (130, 200, 136), (1000, 128, 512), (257, 321, 577)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", T16)
def test_linear_kept_in_8_bits(cuda_device, rows, cin, cout, fmt, dtype):
    x, w = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1, scale=cin ** -0.5)
    b, dy = _randn(cout, dtype=dtype, seed=2), _randn(rows, cout, dtype=dtype, seed=4)
    y, saved = layers.linear_forward(x, w, b, activation="silu", keep=fmt)
    assert torch.equal(y, layers.linear_forward(x, w, b, activation="silu"))
    assert isinstance(saved.kept, Checkpoint8) and isinstance(saved.pre, Checkpoint8)
    assert torch.equal(saved.kept.load(torch.float32), R.keep8(x, fmt)[0])
    # the activation's input: within half a step of p, on top of p's own error (it
    # may be rounded to the type first)
    p64, _ = R.linear64(x, w, b)
    e = (cin + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    e = e + R.half_step(dtype) * (p64.abs() + e) + R.tiny(dtype)
    pre = saved.pre.load(torch.float32).double()
    R.check(pre, p64, e + R.keep8_step(p64.abs() + e, saved.pre.scales, fmt), "pre")
    for name, got, (g, e) in zip(("dx", "dw", "db"), layers.linear_backward(dy, saved, w),
                                 R.linear_grads(dy, saved.kept.load(), w, pre, "silu", dtype)):
        R.check(got, g, e, name)


# residual and everything kept at once: results and what is kept leave through different tiles of the same epilogue;
# 20000 x 512 gives every CTA several tiles, widths that are no multiple of 16 or 8 take the other ways out
@pytest.mark.parametrize("rows,cin,cout", [(20, 64, 72), (40, 64, 24), (300, 200, 136), (333, 72, 96), (700, 264, 577),
                                           (5000, 64, 1040), (20000, 128, 512), (20001, 96, 264), (2001, 72, 333),
                                           (1000, 100, 1030), (20001, 72, 333)])
@pytest.mark.parametrize("keep", layers.KEEPS)
@pytest.mark.parametrize("dtype", T16)
def test_linear_residual_and_keep(cuda_device, rows, cin, cout, keep, dtype):
    x, w = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1, scale=cin ** -0.5)
    b = _randn(cout + 1, dtype=dtype, seed=2)[1:]  # 2-byte aligned
    r = _sliced(_randn(rows, cout, dtype=dtype, seed=3)) if cout % 3 else _randn(rows, cout, dtype=dtype, seed=3)
    y, saved = layers.linear_forward(x, w, b, activation="gelu", residual=r, keep=keep)
    want, bound = R.linear_bound(x, w, b, r, "gelu", dtype)
    R.check(y, want, bound, "y")
    p64, _ = R.linear64(x, w, b)
    e = (cin + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    if keep == "full":
        R.check(saved.pre, p64, e + R.half_step(dtype) * (p64.abs() + e) + R.tiny(dtype), "pre")
        pre = saved.pre.double()
    else:
        pre = saved.pre.load(torch.float32).double()
        # the scale comes from the largest of 128 values that are off by e at most
        amax = torch.nn.functional.pad(p64.abs(), (0, -cout % 128)).reshape(rows, -1, 128).amax(2)
        top = 127 if keep == "int8" else 448
        slack = torch.nn.functional.pad(e, (0, -cout % 128)).reshape(rows, -1, 128).amax(2) / top + amax / top * 2.0 ** -22
        R.check(saved.pre.scales, amax / top, slack, "scales")
        R.check(pre, p64, e + R.keep8_step(p64.abs() + e, saved.pre.scales, keep), "pre")
    dy = _randn(rows, cout, dtype=dtype, seed=4)
    kept = x if keep == "full" else saved.kept.load()
    for name, got, (g, bound) in zip(("dx", "dw", "db"), layers.linear_backward(dy, saved, w),
                                     R.linear_grads(dy, kept, w, pre, "gelu", dtype)):
        R.check(got, g, bound, name)


def test_linear_needs_and_shapes(cuda_device):
    x, w = _randn(2, 5, 64, dtype=torch.bfloat16), _randn(40, 64, dtype=torch.bfloat16, seed=1)
    y, saved = layers.linear_forward(x, w, keep="full")
    assert y.shape == (2, 5, 40)
    dy = torch.ones_like(y)
    dx, dw, db = layers.linear_backward(dy, saved, w)
    assert dx.shape == x.shape and dw.shape == w.shape and db is None  # no bias
    assert torch.equal(layers.linear_backward(dy[:1, :1].expand_as(dy), saved, w)[0], dx)  # a broadcast gradient
    only = layers.linear_backward(dy, saved, w, needs=(False, True, True))
    assert only[0] is None and torch.equal(only[1], dw) and only[2] is None
    one = layers.linear_forward(x[0, 0], w)
    assert one.shape == (40,) and torch.equal(one, layers.linear_forward(x[0, :1], w)[0])


@pytest.mark.parametrize("kind", ["none", "gelu"])
def test_no_rows(cuda_device, kind):
    x, w, b = _randn(0, 64, dtype=torch.bfloat16), _randn(40, 64, dtype=torch.bfloat16), _randn(40, dtype=torch.bfloat16)
    for keep in layers.KEEPS:
        y, saved = layers.linear_forward(x, w, b, activation=kind, keep=keep)
        dx, dw, db = layers.linear_backward(y, saved, w)
        assert y.shape == (0, 40) and dx.shape == (0, 64)
        assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))
        y, saved = layers.layer_norm_forward(x, keep=keep)
        dx, dw, db = layers.layer_norm_backward(y, saved)
        assert dx.shape == (0, 64) and not dw.any() and not db.any()
        y, saved = layers.activation_forward(x, "silu", keep=keep)
        assert layers.activation_backward(y, saved).shape == (0, 64)


def test_linear_nonfinite_values_stay_in_their_row(cuda_device):
    x, w = _randn(300, 200, dtype=torch.bfloat16), _randn(136, 200, dtype=torch.bfloat16, seed=1)
    clean = layers.linear_forward(x, w)
    bad = x.clone()
    bad[5, 7], bad[250, 199], bad[251, 0] = float("nan"), float("inf"), torch.finfo(torch.bfloat16).min
    y = layers.linear_forward(bad, w)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[5, 250, 251]] = False
    assert torch.equal(y[keep], clean[keep])
    assert y[5].isnan().all() and not y[250].isfinite().any()


def test_linear_past_32_bit_offsets(cuda_device):
    rows, cin, cout = (1 << 20) + 3, 16, 2056  # 2.16e9 outputs
    x, w = _randn(rows, cin, dtype=torch.bfloat16), _randn(cout, cin, dtype=torch.bfloat16, seed=1)
    y = layers.linear_forward(x, w)
    tail = slice(rows - 300, rows)
    want, bound = R.linear_bound(x[tail], w, None, None, "none", torch.bfloat16)
    R.check(y[tail], want, bound)
    y, saved = layers.activation_forward(y, "relu", keep="int8")
    assert bool((y[tail] >= 0).all())
    z = layers.layer_norm_forward(y)
    want, bound, *_ = R.norm64(y[tail], None, None, 1e-5, torch.bfloat16)
    R.check(z[tail], want, bound)


# ------------------------------------------------------------- activations, checkpoints

ROWS = [(1, 1), (1, 8), (3, 127), (2, 128), (5, 129), (17, 64), (33, 1021), (4, 4096), (300, 200), (1000, 24), (2, 20000)]


@pytest.mark.parametrize("rows,n", ROWS)
@pytest.mark.parametrize("dtype", T3)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_checkpoint_codes_are_exact(cuda_device, rows, n, dtype, fmt):
    x = _randn(rows, n, dtype=dtype, scale=3.0)
    x[0, 0] = 0
    c = layers.save_checkpoint(x, fmt)
    want, scales = R.keep8(x, fmt)
    assert torch.equal(c.scales, scales)
    assert torch.equal(c.load(torch.float32), want)
    assert torch.equal(c.load(), want.to(dtype))
    R.check(c.load(torch.float32), x.double(), R.keep8_step(x.double(), scales, fmt), "half a step")
    assert c.nbytes == rows * n + 4 * rows * -(-n // 128)
    xs = _sliced(x)
    assert torch.equal(layers.save_checkpoint(xs, fmt).codes, c.codes)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_checkpoint_of_extreme_values(cuda_device, fmt):
    x = _randn(8, 300, dtype=torch.float32)
    x[0, 5], x[1, 140], x[2, 299] = float("nan"), float("inf"), -float("inf")
    x[3] = 0
    x[4] *= 1e-38
    x[5] *= 1e38
    x[6, :128] = torch.finfo(torch.float32).max
    x[7, 128:256] = -0.0
    got = layers.save_checkpoint(x, fmt).load()
    want, _ = R.keep8(x, fmt)
    assert torch.equal(torch.nan_to_num(got, nan=123.0), torch.nan_to_num(want, nan=123.0))
    assert got[0, :128].isnan().all() and not got[0, 128:].isnan().any()
    assert got[1, 128:256].isnan().all() and got[2, 256:].isnan().all() and not got[2, :256].isnan().any()
    assert not got[3].any()


@pytest.mark.parametrize("rows,n", ROWS)
@pytest.mark.parametrize("dtype", T3)
@pytest.mark.parametrize("kind", ["relu", "gelu", "silu"])
def test_activation(cuda_device, rows, n, dtype, kind):
    x, dy = _randn(rows, n, dtype=dtype, scale=3.0), _randn(rows, n, dtype=dtype, seed=5)
    h = R.half_step(dtype)
    for keep in (None,) + layers.KEEPS:
        xs = _sliced(x) if keep == "e4m3" else x
        got = layers.activation_forward(xs, kind, keep=keep)
        y, saved = got if keep else (got, None)
        want = R.act64(x.double(), kind)
        e = R.act_bound(x.double(), kind)
        R.check(y, want, e + h * (want.abs() + e) + R.tiny(dtype), f"y {keep}")
        if saved is None:
            continue
        kept = x.double() if keep == "full" else saved.kept.load(torch.float32).double()
        want = dy.double() * R.act_grad64(kept, kind)
        e = dy.double().abs() * R.act_grad_bound(kept, kind) + R.U32 * want.abs()
        R.check(layers.activation_backward(dy, saved), want, e + h * (want.abs() + e) + R.tiny(dtype), f"dx {keep}")


def test_activation_special_values(cuda_device):
    v = torch.tensor([0.0, -0.0, float("nan"), torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max, -30.0, 30.0,
                      float("inf")], dtype=torch.bfloat16, device="cuda").reshape(1, 8)
    for kind in ("relu", "gelu", "silu"):
        y = layers.activation_forward(v, kind)[0]
        assert y[2].isnan() and y[0] == 0 and y[1] == 0 and y[3] == 0 and y[4] == v[0, 4] and y[6] == 30 and y[7] == v[0, 7]
        assert abs(float(y[5])) < 1e-10


def test_activation_gradient_against_differences(cuda_device):
    x, v, dy = (_randn(64, 96, dtype=torch.float32, seed=s) for s in (1, 2, 3))
    for kind in ("gelu", "silu"):
        _, saved = layers.activation_forward(x, kind, keep="full")
        slope = float((layers.activation_backward(dy, saved).double() * v.double()).sum())
        h = 1e-2
        diff = float(((layers.activation_forward(x + h * v, kind).double() - layers.activation_forward(x - h * v, kind).double())
                      * dy.double()).sum()) / (2 * h)
        # h^2 / 6 times third derivatives below 2, fp32 roundings of x and y over h
        size = float((dy.abs() * v.abs() ** 3).sum()) * h * h / 3 + float((dy.abs() * (1 + x.abs())).sum()) * 2 ** -22 / h
        assert abs(slope - diff) <= size


# ------------------------------------------------------------------------ layer norm

NORMS = [(1, 1), (1, 8), (1, 4096), (3, 127), (2, 128), (5, 129), (17, 64), (33, 1021), (40, 256), (9, 512), (6, 1032), (7, 2048),
         (5, 4096), (3, 8192), (300, 192), (2000, 24), (2, 16384), (3, 20001), (2, 40000), (5000, 320), (70000, 8)]


@pytest.mark.parametrize("rows,n", NORMS)
@pytest.mark.parametrize("dtype", T3)
@pytest.mark.parametrize("keep", [None, "full", "int8", "e4m3"])
def test_layer_norm(cuda_device, rows, n, dtype, keep):
    x = _randn(rows, n, dtype=dtype) + _randn(rows, 1, dtype=dtype, seed=9) * 3
    wdtype = torch.float32 if n % 3 else dtype
    w, b = 1 + _randn(n, dtype=wdtype, seed=1, scale=0.3), _randn(n, dtype=wdtype, seed=2)
    if keep is None:
        w, b = (w, None) if rows % 2 else (None, None)
    dy = _randn(rows, n, dtype=dtype, seed=4)
    got = layers.layer_norm_forward(_sliced(x) if keep == "int8" else x, w, b, eps=1e-4, keep=keep)
    y, saved = got if keep else (got, None)
    want, bound, *_ = R.norm64(x, w, b, 1e-4, dtype)
    R.check(y, want, bound, "y")
    if saved is None:
        return
    kept = x
    if keep != "full":
        kept = saved.kept.load(torch.float32)
        assert torch.equal(kept, R.keep8(x, keep)[0])
    dy = _sliced(dy) if keep == "int8" else dy
    grads = layers.layer_norm_backward(dy, saved, w)
    for name, t, (g, e) in zip(("dx", "dw", "db"), grads, R.norm_grads(dy, kept, x, w, 1e-4, dtype, wdtype)):
        assert t.dtype == (dtype if name == "dx" else wdtype)
        R.check(t, g, e, name)
    only = layers.layer_norm_backward(dy, saved, w, needs=(False, False, True))
    assert only[0] is None and only[1] is None and torch.equal(only[2], grads[2])
    if n > 1:
        assert torch.equal(layers.layer_norm_backward(dy, saved, w, needs=(True, False, False))[0], grads[0])


# enough rows for the kernels that take several rows a CTA at a time: tails, widths that leave threads idle, two
# chunks a thread
@pytest.mark.parametrize("rows,n,dtype", [(9500, 520, torch.bfloat16), (6001, 1032, torch.float16), (6000, 1024, torch.bfloat16),
                                          (2500, 4096, torch.bfloat16), (2405, 2048, torch.float32), (3001, 6160, torch.float16),
                                          (1300, 8192, torch.bfloat16), (1301, 4096, torch.float32)])
@pytest.mark.parametrize("keep", [None, "full", "int8", "e4m3"])
def test_layer_norm_many_rows(cuda_device, rows, n, dtype, keep):
    x = _randn(rows, n, dtype=dtype) + _randn(rows, 1, dtype=dtype, seed=9) * 3
    w, b = 1 + _randn(n, dtype=torch.float32, seed=1, scale=0.3), _randn(n, dtype=torch.float32, seed=2)
    dy = _randn(rows, n, dtype=dtype, seed=4)
    wide = torch.zeros(rows, n + 64, dtype=dtype, device="cuda")  # rows with a stride of their own
    wide[:, 64:] = x
    got = layers.layer_norm_forward(wide[:, 64:], w, b, eps=1e-4, keep=keep)
    y, saved = got if keep else (got, None)
    want, bound, *_ = R.norm64(x, w, b, 1e-4, dtype)
    R.check(y, want, bound, "y")
    if saved is None:
        return
    kept = x
    if keep != "full":
        kept = saved.kept.load(torch.float32)
        assert torch.equal(kept, R.keep8(x, keep)[0])
    grads = layers.layer_norm_backward(dy, saved, w)
    for name, t, (g, e) in zip(("dx", "dw", "db"), grads, R.norm_grads(dy, kept, x, w, 1e-4, dtype, torch.float32)):
        R.check(t, g, e, name)
    assert torch.equal(layers.layer_norm_backward(dy, saved, w, needs=(True, False, False))[0], grads[0])
    assert torch.equal(layers.layer_norm_backward(dy, saved, w, needs=(False, True, False))[1], grads[1])


def test_layer_norm_constant_rows(cuda_device):
    # no variance: the centred values are zero, and y is the bias
    x = torch.full((4, 200), 3.25, dtype=torch.bfloat16, device="cuda")
    b = _randn(200, dtype=torch.float32)
    y, saved = layers.layer_norm_forward(x, None, b, keep="full")
    assert torch.equal(y, b.to(torch.bfloat16).expand(4, 200))
    dx, _, _ = layers.layer_norm_backward(_randn(4, 200, dtype=torch.bfloat16), saved)
    assert dx.isfinite().all()


def test_layer_norm_gradient_against_differences(cuda_device):
    x, v, dy = (_randn(16, 96, dtype=torch.float32, seed=s) for s in (1, 2, 3))
    w = 1 + _randn(96, dtype=torch.float32, seed=5, scale=0.3)
    _, saved = layers.layer_norm_forward(x, w, None, keep="full")
    slope = float((layers.layer_norm_backward(dy, saved, w)[0].double() * v.double()).sum())
    h = 1e-2
    diff = float(((layers.layer_norm_forward(x + h * v, w).double() - layers.layer_norm_forward(x - h * v, w).double())
                  * dy.double()).sum()) / (2 * h)
    # the third derivative along v of a row of unit variance is below 20 |v|^3 a value
    size = 20 * h * h / 6 * float((dy.abs() * v.abs() ** 3).sum()) + float((dy.abs() * (1 + x.abs())).sum()) * 2 ** -21 / h
    assert abs(slope - diff) <= size


# -------------------------------------------------------------------------- together

def _block(x, p, keep):
    """A pre-norm feed-forward block, as a context model has them."""
    h = layers.layer_norm(x, p["g"], p["c"], keep=keep)
    h = layers.linear(h, p["w1"], p["b1"], activation="gelu", keep=keep)
    return layers.linear(h, p["w2"], p["b2"], residual=x, keep=keep)


def _block_parameters(cin=192, inner=520, dtype=torch.bfloat16):
    p = {"g": 1 + _randn(cin, dtype=torch.float32, scale=0.2), "c": _randn(cin, dtype=torch.float32, seed=1, scale=0.2),
         "w1": _randn(inner, cin, dtype=dtype, seed=2, scale=cin ** -0.5), "b1": _randn(inner, dtype=dtype, seed=3, scale=0.2),
         "w2": _randn(cin, inner, dtype=dtype, seed=4, scale=inner ** -0.5), "b2": _randn(cin, dtype=dtype, seed=5, scale=0.2)}
    return {k: v.requires_grad_() for k, v in p.items()}


@pytest.mark.parametrize("keep", layers.KEEPS)
@pytest.mark.parametrize("rows", [1, 48, 1537])
def test_block_trains_and_serves(cuda_device, keep, rows):
    p = _block_parameters()
    x = _randn(rows, 192, dtype=torch.bfloat16).requires_grad_()
    y = _block(x, p, keep)
    dy = _randn(rows, 192, dtype=torch.bfloat16, seed=8)
    grads = torch.autograd.grad(y, [x, *p.values()], dy)
    with torch.no_grad():  # serving is the same numbers, without anything kept, position by position too
        z = _block(x, p, keep)
        assert torch.equal(z, y)
    # the same block in 64 bits
    q = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    xd = x.detach().double().requires_grad_()
    h = torch.nn.functional.layer_norm(xd, (192,), q["g"], q["c"], 1e-5)
    h = torch.nn.functional.gelu(h @ q["w1"].t() + q["b1"])
    yd = h @ q["w2"].t() + q["b2"] + xd
    want = torch.autograd.grad(yd, [xd, *q.values()], dy.double())
    # relative 2-norms: the forward pass rounds 3 times to bf16 (2^-8 at most, about
    # 2^-9.2 in the norm, each); a gradient passes about 6 such roundings, and an
    # 8-bit checkpoint moves the values it stands for by 0.7% (int8: a step of
    # amax / 127 with amax near 3 sigma) or 2.6% (e4m3, 2^-4 / sqrt(6))
    tol = {"full": 0.01, "int8": 0.03, "e4m3": 0.08}[keep]
    assert float((y.double() - yd).norm() / yd.norm()) < 0.01
    for g, e, name in zip(grads, want, ["x", *p]):
        assert g.dtype == (x if name == "x" else p[name]).dtype
        assert float((g.double() - e).norm() / e.norm()) < tol, name


def test_results_repeat_bitwise_and_on_other_streams(cuda_device):
    p = _block_parameters()
    x = _randn(1537, 192, dtype=torch.bfloat16).requires_grad_()
    dy = _randn(1537, 192, dtype=torch.bfloat16, seed=8)

    def once():
        y = _block(x, p, "int8")
        return [y.detach(), *torch.autograd.grad(y, [x, *p.values()], dy)]

    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams:  # in flight at the same time
        with torch.cuda.stream(s):
            results.append(once())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_captured_in_graphs(cuda_device):
    # two graphs of a forward and backward pass, replayed at once on two streams with new inputs
    w, b = _randn(512, 192, dtype=torch.bfloat16, scale=0.07), _randn(512, dtype=torch.bfloat16, seed=1)
    g = 1 + _randn(192, dtype=torch.float32, seed=2, scale=0.2)

    def step(x, dy):
        h, s0 = layers.layer_norm_forward(x, g, None, keep="int8")
        y, s1 = layers.linear_forward(h, w, b, activation="silu", keep="e4m3")
        dh, dw, db = layers.linear_backward(dy, s1, w)
        dx, dg, _ = layers.layer_norm_backward(dh, s0, g)
        return y, dx, dw, db, dg

    ins = [(_randn(700, 192, dtype=torch.bfloat16, seed=s), _randn(700, 512, dtype=torch.bfloat16, seed=s + 50)) for s in (3, 4)]
    step(*ins[0])
    graphs, outs = [], []
    for x, dy in ins:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(x, dy))
        graphs.append(graph)
    for x, dy in ins:
        x.copy_(x.flip(0))
        dy.mul_(0.5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for s, graph in zip(streams, graphs):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for (x, dy), out in zip(ins, outs):
        assert all(torch.equal(a, e) for a, e in zip(out, step(x, dy)))


def test_first_calls_of_a_process_can_be_captured(cuda_device):
    # nothing has to be set up outside a capture
    code = """
import sys
sys.path[:0] = [%r, %r]
import torch
from fast_compressai import layers
x = torch.randn(700, 200, device="cuda", dtype=torch.bfloat16)
w = torch.randn(264, 200, device="cuda", dtype=torch.bfloat16) / 14
dy = torch.randn(700, 264, device="cuda", dtype=torch.bfloat16)
def step():
    h, s0 = layers.layer_norm_forward(x, keep="int8")
    y, s1 = layers.linear_forward(h, w, activation="gelu", keep="e4m3")
    dh, dw, _ = layers.linear_backward(dy, s1, w)
    one = layers.linear_forward(x[:1], w)
    return y, dw, layers.layer_norm_backward(dh, s0)[0], one
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, step()))
print("captured")
"""
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code % (str(root), str(root / "fast-compressai_b200"))], capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


def test_in_place_change_of_a_kept_tensor_is_noticed(cuda_device):
    x, w = _randn(8, 64, dtype=torch.bfloat16), _randn(40, 64, dtype=torch.bfloat16, seed=1).requires_grad_()
    y = layers.linear(x, w, activation="gelu")
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_gpu_refusals(cuda_device):
    x, w = _randn(4, 64, dtype=torch.bfloat16), _randn(40, 64, dtype=torch.bfloat16)
    bad = [
        lambda: layers.linear_forward(x.float(), w.float()),
        lambda: layers.linear_forward(x, w.half()),
        lambda: layers.linear_forward(x, w[:, :63]),
        lambda: layers.linear_forward(x, w.reshape(-1)),
        lambda: layers.linear_forward(x, w.cpu()),
        lambda: layers.linear_forward(x, w, x[0]),
        lambda: layers.linear_forward(x, w, residual=x),
        lambda: layers.linear_forward(x[:, :0], w[:, :0]),
        lambda: layers.layer_norm_forward(x, w[0].half()),
        lambda: layers.layer_norm_forward(x, w[0, :63]),
        lambda: layers.layer_norm_forward(x, w[0], w[0].float()),
        lambda: layers.layer_norm_forward(x, eps=-1.0),
        lambda: layers.layer_norm_forward(x.double()),
        lambda: layers.layer_norm_forward(x[:, :0]),
        lambda: layers.activation_forward(x.to(torch.int32), "relu"),
        lambda: layers.save_checkpoint(x).load(torch.float64),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    y, saved = layers.linear_forward(x, w, keep="full")
    for call in (lambda: layers.linear_backward(y[:2], saved, w), lambda: layers.linear_backward(y.half(), saved, w),
                 lambda: layers.linear_backward(y, saved, w[:20]), lambda: layers.layer_norm_backward(y, saved)):
        with pytest.raises(ValueError):
            call()


def test_relu_gradient_at_special_values(cuda_device):
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[-1.0, 0.0, -0.0, 2.0, nan, -inf, inf, 3.0]], device="cuda")
    g = torch.tensor([[inf, -inf, nan, inf, 5.0, inf, 7.0, nan]], device="cuda")
    want = torch.tensor([[0.0, 0.0, 0.0, inf, 5.0, 0.0, 7.0, nan]], device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _, saved = layers.activation_forward(x.to(dtype), "relu", keep="full")
        dx = layers.activation_backward(g.to(dtype), saved)
        assert torch.equal(dx.float().nan_to_num(nan=99.0), want.nan_to_num(nan=99.0))


def test_what_was_kept_must_fit(cuda_device):
    x, w = _randn(40, 64, dtype=torch.bfloat16), _randn(40, 64, dtype=torch.bfloat16, seed=1)
    y, saved = layers.linear_forward(x, w, activation="gelu", keep="full")
    for part in ("kept", "pre"):
        whole = getattr(saved, part)
        for bad in (whole.half(), whole.cpu(), whole[:, :8], whole[:8]):
            setattr(saved, part, bad)
            with pytest.raises(ValueError):
                layers.linear_backward(y, saved, w, (True, False, False))
        setattr(saved, part, whole)
    layers.linear_backward(y, saved, w)
    with pytest.raises(ValueError, match="dense"):
        layers.linear_forward(torch._neg_view(x), w)


def test_a_wait_that_ran_out_is_reported_by_the_next_call(cuda_device):
    from fast_compressai import _native

    word = _native.lib().fcai_linear_error_word()
    assert word and word[0] == 0  # no product so far ran into it
    for rows in (1, 300):
        x, w = _randn(rows, 64, dtype=torch.bfloat16), _randn(40, 64, dtype=torch.bfloat16, seed=1)
        want, saved = layers.linear_forward(x, w, keep="full")
        word[0] = 1
        with pytest.raises(_native.NativeCallError, match="ran out"):
            layers.linear_forward(x, w)
        assert word[0] == 0 and torch.equal(layers.linear_forward(x, w), want)
        word[0] = 1
        with pytest.raises(_native.NativeCallError, match="ran out"):
            layers.linear_backward(want, saved, w)
        assert word[0] == 0


@pytest.mark.parametrize("rows,cout", [(50003, 136), (20001, 333), (40, 136), (8, 40), (300, 65)])
def test_linear_unaligned_residual_of_any_size(cuda_device, rows, cout):
    dtype = torch.float16
    x, w = _randn(rows, 24, dtype=dtype), _randn(cout, 24, dtype=dtype, seed=1, scale=0.2)
    b, r = _randn(cout + 1, dtype=dtype, seed=2)[1:], _randn(rows, cout, dtype=dtype, seed=3)
    want, bound = R.linear_bound(x, w, b, r, "silu", dtype)
    for keep in (None, "full", "int8"):
        out = layers.linear_forward(x, w, b, activation="silu", residual=_sliced(r), keep=keep)
        R.check(out if keep is None else out[0], want, bound, f"{keep}")


@pytest.mark.parametrize("rows,cin,cout", [(50003, 24, 136), (20001, 24, 333), (300, 72, 65), (20, 64, 40), (3, 33, 17)])
@pytest.mark.parametrize("ld_more,offset", [(0, 0), (8, 0), (8, 8), (5, 0), (7, 3)])
def test_outputs_inside_wider_matrices(cuda_device, rows, cin, cout, ld_more, offset):
    # the C entry writes y's columns and nothing beside them
    from fast_compressai import _native

    lib, dtype = _native.lib(), torch.bfloat16
    x, w = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1, scale=cin ** -0.5)
    b = _randn(cout, dtype=dtype, seed=2)
    ld = cout + ld_more + offset
    big = torch.full((rows + 2, ld), 7.0, dtype=dtype, device="cuda")
    y = big[1:-1, offset:offset + cout]

    def bits(p, stride, bit):
        return 0 if p % 16 == 0 and stride % 8 == 0 else bit

    repack = (bits(x.data_ptr(), cin, 1) | bits(w.data_ptr(), cin, 2) | bits(y.data_ptr(), ld, 4) | bits(b.data_ptr(), cout, 16))
    n = lib.fcai_linear_workspace(0, rows, cin, cout, repack, 0)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    code = lib.fcai_linear_forward(x.data_ptr(), cin, w.data_ptr(), cin, b.data_ptr(), None, 0, y.data_ptr(), ld, None, 0, None,
                                   None, rows, cin, cout, 0, 2, 0, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    assert code == 0, lib.fcai_last_error()
    want, bound = R.linear_bound(x, w, b, None, "gelu", dtype)
    R.check(y, want, bound, "y")
    assert (big[0] == 7).all() and (big[-1] == 7).all()
    assert (big[:, :offset] == 7).all() and (big[:, offset + cout:] == 7).all()


@pytest.mark.parametrize("rows,n", [(33, 40), (5, 1021), (70, 24), (9, 9000), (300, 200)])
@pytest.mark.parametrize("ld_more,offset", [(8, 0), (8, 8), (5, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rowwise_outputs_inside_wider_matrices(cuda_device, rows, n, ld_more, offset, dtype):
    # the same numbers as the calls that allocate, and nothing written beside them
    from fast_compressai import _native

    lib, code = _native.lib(), {torch.bfloat16: 0, torch.float32: 2}[dtype]
    x, dy = _randn(rows, n, dtype=dtype), _randn(rows, n, dtype=dtype, seed=1)
    ld = n + ld_more + offset
    stream = torch.cuda.current_stream().cuda_stream

    def inside(call, want, exact=True):
        big = torch.full((rows + 2, ld), 7.0, dtype=dtype, device="cuda")
        y = big[1:-1, offset:offset + n]
        assert call(y.data_ptr()) == 0, lib.fcai_last_error()
        # another alignment sums a row's channels in another order: fp32 results some 2^-20 apart (values of order 1, hence
        # 1e-5), whose roundings are at most one step, eps of the value, apart
        assert torch.equal(y, want) if exact else torch.allclose(y.float(), want.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-5)
        assert (big[0] == 7).all() and (big[-1] == 7).all()
        assert (big[:, :offset] == 7).all() and (big[:, offset + n:] == 7).all()

    inside(lambda p: lib.fcai_activation_forward(x.data_ptr(), n, p, ld, None, None, rows, n, code, 3, 0, stream),
           layers.activation_forward(x, "silu"))
    _, saved = layers.activation_forward(x, "silu", keep="int8")
    c, s = saved.kept.codes.data_ptr(), saved.kept.scales.data_ptr()
    inside(lambda p: lib.fcai_activation_backward(dy.data_ptr(), n, None, 0, c, s, p, ld, None, rows, n, code, 3, 2, None, 0,
                                                  stream), layers.activation_backward(dy, saved))
    inside(lambda p: lib.fcai_checkpoint_load(c, s, p, ld, rows, n, code, 2, stream), saved.kept.load())
    y, saved = layers.layer_norm_forward(x, keep="full")
    mean, rstd = saved.stats[0].data_ptr(), saved.stats[1].data_ptr()
    inside(lambda p: lib.fcai_layer_norm_forward(x.data_ptr(), n, None, None, code, p, ld, None, None, None, None, rows, n, 1e-5,
                                                 code, 0, stream), y, exact=False)
    need = lib.fcai_layer_norm_workspace(rows, n)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    inside(lambda p: lib.fcai_layer_norm_backward(dy.data_ptr(), n, x.data_ptr(), n, None, None, mean, rstd, None, code, p, ld,
                                                  None, None, rows, n, code, 1, ws.data_ptr(), need, stream),
           layers.layer_norm_backward(dy, saved, needs=(True, False, False))[0], exact=False)
