"""Plain 64-bit forms of the pointwise layers and bounds on the rounding of the
kernels, shared by the CPU and GPU tests.

Unit roundoffs: a value rounded to type t is off by at most eps(t) / 2 of it.
Sums in fp32 are off by at most (number of additions in sequence) * 2^-24 of
the sum of magnitudes; tensor-core sums are counted with 2^-23 an addition,
since they may truncate.
"""

from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half of the spacing of subnormal numbers: the rounding of values next to zero."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def act64(p: torch.Tensor, kind: str) -> torch.Tensor:
    if kind == "relu":
        return torch.relu(p)
    if kind == "gelu":
        return p * 0.5 * torch.special.erfc(-p / math.sqrt(2))
    if kind == "silu":
        return p * torch.sigmoid(p)
    return p


def act_grad64(p: torch.Tensor, kind: str) -> torch.Tensor:
    if kind == "relu":
        return (p > 0).double()
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-p / math.sqrt(2)) + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
    if kind == "silu":
        s = torch.sigmoid(p)
        return s + p * s * (1 - s)
    return torch.ones_like(p)


def act_bound(p: torch.Tensor, kind: str) -> torch.Tensor:
    """|act(p) computed in fp32 - act(p)|.  relu: exact.  gelu: x * Phi with the
    tail's fit (7.6e-7 of it) and a handful of fp32 roundings, and the fp32
    argument p^2 / 2 of the exponential, relative p^2 * 2^-23.  silu: exp2 and
    reciprocal, 2^-22 each, and the argument's rounding, relative |p| * 2^-22.
    Values below 2^-100 may be flushed to zero."""
    if kind in ("none", "relu"):
        return torch.zeros_like(p)
    a = act64(p, kind).abs()
    tail = torch.where(p < 0, p * p, torch.zeros_like(p)) if kind == "gelu" else p.abs()
    return a * (2e-6 + tail * 2.0 ** -22) + p.abs() * 2.0 ** -100


def act_grad_bound(p: torch.Tensor, kind: str) -> torch.Tensor:
    """|act'(p) computed in fp32 - act'(p)|: the two terms of each derivative as in act_bound."""
    if kind in ("none", "relu"):
        return torch.zeros_like(p)
    if kind == "gelu":
        phi = torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
        cdf = 0.5 * torch.special.erfc(-p / math.sqrt(2))
        return (cdf + p.abs() * phi) * (2e-6 + p * p * 2.0 ** -22) + 2.0 ** -24 + p.abs() * 2.0 ** -100
    s = torch.sigmoid(p)
    return (s + 2 * p.abs() * s) * (2e-6 + p.abs() * 2.0 ** -22) + p.abs() * 2.0 ** -100


def keep8(x: torch.Tensor, fmt: str):
    """(values read back in fp32, scales) of an 8-bit checkpoint, by its definition in torch fp32."""
    rows, n = x.shape
    pad = -n % 128
    v = torch.nn.functional.pad(x.float(), (0, pad)).reshape(rows, -1, 128)
    amax = v.abs().amax(dim=2, keepdim=True)
    top = 127.0 if fmt == "int8" else 448.0
    scale = (amax * torch.tensor(1 / top, dtype=torch.float32, device=x.device)).clamp(min=torch.finfo(torch.float32).tiny)
    scale = torch.where(torch.isfinite(amax), scale, torch.full_like(scale, math.nan))
    q = (v * (torch.ones_like(scale) / scale)).clamp(-top, top)
    q = torch.round(q) if fmt == "int8" else q.to(torch.float8_e4m3fn).float()
    return (q * scale).reshape(rows, -1)[:, :n], scale[:, :, 0]


def keep8_step(x: torch.Tensor, scales: torch.Tensor, fmt: str) -> torch.Tensor:
    """Half a step of the checkpoint's grid at x (64 bits), with room for fp32 roundings of the code's argument."""
    s = scales.double().repeat_interleave(128, dim=1)[:, :x.shape[1]]
    if fmt == "int8":
        return s * (0.5 + 127 * 2.0 ** -22)
    return torch.maximum(x.abs() * (2.0 ** -4 + 2.0 ** -22), s * 2.0 ** -10)


def linear64(x, w, b=None, r=None, kind="none"):
    """(p, y) in 64 bits."""
    p = x.double() @ w.double().t()
    if b is not None:
        p = p + b.double()
    y = act64(p, kind)
    return p, y if r is None else y + r.double()


def linear_bound(x, w, b, r, kind, dtype):
    """|y - y64|: the product's sum, the slope of the activation (at most 1.13), its own error, and the rounding."""
    p, y = linear64(x, w, b, r, kind)
    mag = x.double().abs() @ w.double().abs().t() + (0 if b is None else b.double().abs())
    e = (x.shape[-1] + 2) * 2.0 ** -23 * mag
    e = 1.13 * e + act_bound(p, kind) + 2 * U32 * y.abs()
    return y, e + half_step(dtype) * (y.abs() + e) + tiny(dtype)


def linear_grads(dy, x, w, pre, kind, dtype, bias=True):
    """((dx, bound), (dw, bound), (db, bound)) in 64 bits, from the values `pre` and x that were kept."""
    dy, x, w = dy.double(), x.double(), w.double()
    rows, cout = dy.shape
    h = half_step(dtype)
    dp = dy * act_grad64(pre, kind)
    e32 = dy.abs() * act_grad_bound(pre, kind) + U32 * dp.abs()           # dp in fp32
    edp = e32 + (h * (dp.abs() + e32) + tiny(dtype) if kind != "none" else 0)  # and rounded for the products
    adp = dp.abs() + edp

    def bound(v, e):
        return v, e + h * (v.abs() + e) + tiny(dtype)

    dx, dw = dp @ w, dp.t() @ x
    ex = edp @ w.abs() + (cout + 2) * 2.0 ** -23 * (adp @ w.abs())
    ew = edp.t() @ x.abs() + (rows + 2) * 2.0 ** -23 * (adp.t() @ x.abs())
    db = dp.sum(0)
    eb = e32.sum(0) + (rows + 2) * U32 * adp.sum(0)
    return bound(dx, ex), bound(dw, ew), bound(db, eb)


def _depth(n):
    """Additions in sequence of a row's sum: at most n / 32 in a lane and a tree above."""
    return n / 32 + 40


def norm64(x, w, b, eps, dtype):
    """(y, bound, mean, rstd, bound of xhat) in 64 bits; x [rows, n]."""
    x = x.double()
    n = x.shape[1]
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = (c * c).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    d = _depth(n)
    emean = (d + 2) * U32 * x.abs().mean(1, keepdim=True)
    # the variance's error relative to var + eps: the centred values are off by
    # emean + u |c| each, the sum of squares by its own additions
    evar = (2 * emean * c.abs().mean(1, keepdim=True) + emean ** 2 + (d + 8) * 2 * U32 * var) / (var + eps)
    erstd = evar / 2 + 6 * U32
    xhat = c * rstd
    exhat = emean * rstd + xhat.abs() * (erstd + 4 * U32)
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
    y = xhat * w + b
    e = w.abs() * exhat + 2 * U32 * (y.abs() + b.abs())
    return y, e + half_step(dtype) * (y.abs() + e) + tiny(dtype), mean, rstd, xhat, exhat, erstd


def norm_grads(dy, x_kept, x, w, eps, dtype, wdtype):
    """((dx, bound), (dw, bound), (db, bound)): statistics of x, values of x_kept."""
    _, _, mean, rstd, _, _, erstd = norm64(x, None, None, eps, dtype)
    dy, xk = dy.double(), x_kept.double()
    rows, n = dy.shape
    w = torch.ones(n, dtype=torch.float64, device=dy.device) if w is None else w.double()
    d = _depth(n)
    emean = (d + 2) * U32 * x.double().abs().mean(1, keepdim=True)
    xhat = (xk - mean) * rstd
    exhat = emean * rstd + xhat.abs() * (erstd + 4 * U32)
    t = dy * w
    m1, m2 = t.mean(1, keepdim=True), (t * xhat).mean(1, keepdim=True)
    em1 = (d + 3) * U32 * t.abs().mean(1, keepdim=True)
    em2 = (d + 4) * U32 * (t * xhat).abs().mean(1, keepdim=True) + (t.abs() * exhat).mean(1, keepdim=True)
    inner = t - m1 - xhat * m2
    dx = rstd * inner
    e = rstd * (3 * U32 * (t.abs() + m1.abs() + (xhat * m2).abs()) + em1 + xhat.abs() * em2 + exhat * (m2.abs() + em2))
    e = e + dx.abs() * (erstd + 2 * U32)
    h, hw = half_step(dtype), half_step(wdtype)
    dx_b = e + h * (dx.abs() + e) + tiny(dtype)
    seq = rows + 4
    dw = (dy * xhat).sum(0)
    ew = (dy.abs() * exhat).sum(0) + seq * U32 * (dy * xhat).abs().sum(0)
    db = dy.sum(0)
    eb = seq * U32 * dy.abs().sum(0)
    return ((dx, dx_b), (dw, ew + hw * (dw.abs() + ew) + tiny(wdtype)), (db, eb + hw * (db.abs() + eb) + tiny(wdtype)))


def check(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    err = (got.double() - want).abs()
    over = err - bound
    assert bool((over <= 0).all()), (f"{what}: {int((over > 0).sum())} of {err.numel()} values over the bound, "
                                     f"worst {err.flatten()[over.argmax()].item():.4g} against "
                                     f"{bound.expand_as(err).flatten()[over.argmax()].item():.4g}")
