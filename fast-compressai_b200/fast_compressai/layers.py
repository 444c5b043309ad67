"""Pointwise layers for B200: the matrix product with bias, activation and
residual in its epilogue, layer norm, and activations whose input is kept in 8
bits for the backward pass (include/fcai_layers.h).

They work on rows of channels (``[..., channels]``, channels contiguous: the
positions of an NHWC latent or activation, the tokens of a context model) and
come in two forms:

* explicit calls: ``linear_forward`` / ``linear_backward``,
  ``layer_norm_forward`` / ``layer_norm_backward``, ``activation_forward`` /
  ``activation_backward``.  Without ``keep`` a forward call returns its output
  alone (serving); with ``keep`` it also returns what its backward call needs:
  ``"full"`` keeps tensors in their own type, ``"int8"`` and ``"e4m3"`` keep
  them as ``Checkpoint8`` (about half the bytes of a 16-bit tensor, blocks of
  128 channels with one scale each);
* differentiable calls over them: ``linear``, ``layer_norm``, ``activation``.

A backward pass takes the derivatives of what was kept.  A ReLU input above 0
that an 8-bit checkpoint rounds to 0 (in int8, below 1 / 254 of the largest of
its 128 channels) so has the gradient 0; ``"full"`` keeps its sign.

``torch.autocast`` does not reach these calls.  ``linear`` takes tensors of one
16-bit type; the others take fp32 too, layer norm's weight and bias in x's type
or fp32; anything else is refused.

Every call runs on the current stream of its tensors' device and allocates its
outputs and scratch from torch's caching allocator, so calls on different
streams or in different captured graphs share nothing.  Tensors that belong to
another stream need the caller's ``wait_stream`` / ``record_stream``, as with
any torch operation.  Results are bitwise reproducible: no sum depends on the
order in which CTAs finish.  To capture a backward pass into a CUDA graph, use
the explicit calls, or release eager autograd graphs of the same parameters
first (torch's own gradient accumulation ties them to the stream they were
first used on).

The results of the explicit calls carry no gradient.  Under ``torch.jit.trace``
the differentiable calls are recorded as nodes that run them again; the explicit
calls refuse it, and all refuse ``make_fx`` and tensors with a forward-mode
tangent, since nothing would follow what they do.

Arguments that do not fit raise ``ValueError`` before anything is launched.
There is no fallback: the tensors are on a CUDA device and the native library
is built.  The products' kernels give up a wait that takes longer than a second
(a bug, never expected) and leave wrong results; the next product on the device
then raises ``NativeCallError``.  After the last product, or a replayed graph,
``check()`` asks.
"""

from __future__ import annotations

import torch

from . import _native

ACTIVATIONS = ("none", "relu", "gelu", "silu")
KEEPS = ("full", "int8", "e4m3")
BLOCK = 128  # channels that share a scale (FCAI_KEEP_BLOCK)

_ACT = {name: i for i, name in enumerate(ACTIVATIONS)}
_KEEP = {None: 0, "full": 1, "int8": 2, "e4m3": 3}
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_count = _native.count_launches


class _Host:
    """The compiled calls; loaded on first use, so that importing the package
    needs no built library."""

    def __getattr__(self, name):
        fn = getattr(_native.layers_host(), name)
        setattr(self, name, fn)
        return fn


_host = _Host()


class Checkpoint8:
    """A tensor kept in 8 bits: ``codes`` (uint8 ``[rows, channels]``, int8 or
    e4m3 by ``format``) and one fp32 scale per row and block of 128 channels
    (``scales``).  A block that held an infinity or a NaN reads back as NaN."""

    __slots__ = ("codes", "scales", "shape", "dtype", "format")

    def __init__(self, codes, scales, shape, dtype, format):
        self.codes, self.scales, self.shape, self.dtype, self.format = codes, scales, shape, dtype, format

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()

    def load(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values it stands for, in ``dtype`` (its tensor's type if not given)."""
        code = _DTYPE.get(self.dtype if dtype is None else dtype)
        if code is None:
            raise ValueError(f"a checkpoint reads back as bf16, fp16 or fp32, not {dtype}")
        out = _host.load8(self.codes, self.scales, _KEEP[self.format], code, self.shape)
        _count(1)
        return out


class Saved:
    """What a forward call kept for its backward call."""

    __slots__ = ("op", "kept", "pre", "stats", "activation", "shape", "dtype", "bias")

    def __init__(self, op, kept, shape, dtype, pre=None, stats=None, activation="none", bias=None):
        self.op, self.kept, self.shape, self.dtype = op, kept, shape, dtype
        self.pre, self.stats, self.activation, self.bias = pre, stats, activation, bias


def _code(what: str, value, known: dict) -> int:
    try:
        return known[value]
    except (KeyError, TypeError):
        names = ", ".join(repr(k) for k in known if k is not None)
        raise ValueError(f"unknown {what} {value!r} (one of {names})") from None


def _parts(kept):
    """(tensor or codes, scales, keep code) as the compiled calls take them."""
    if isinstance(kept, Checkpoint8):
        return kept.codes, kept.scales, _KEEP[kept.format]
    return kept, None, 1


def _check_saved(saved, op: str, grad) -> None:
    if not isinstance(saved, Saved) or saved.op != op:
        raise ValueError(f"expected what {op}_forward kept")
    if not isinstance(grad, torch.Tensor) or grad.shape != saved.shape:
        raise ValueError(f"grad must be a tensor of shape {tuple(saved.shape)}")
    if grad.dtype is not saved.dtype:
        raise ValueError(f"grad has dtype {grad.dtype}, expected {saved.dtype}")


def check(device: torch.device | str | int | None = None) -> None:
    """Waits for ``device`` (the current one by default) and raises
    ``NativeCallError`` if a product on it, run by a call or by a replayed graph,
    gave up a wait since the last report: its results are wrong."""
    index = torch.cuda.current_device() if device is None else device
    device = torch.device("cuda", index) if isinstance(index, int) else torch.device(index)
    if device.type != "cuda":
        raise ValueError(f"check takes a CUDA device, not {device}")
    with torch.cuda.device(device):
        torch.cuda.synchronize()
        word = _native.lib().fcai_linear_error_word()
        if not word:
            raise _native.NativeCallError(_native.FCAI_ERR_CUDA, f"no error word for {device}")
        if word[0]:
            word[0] = 0
            raise _native.NativeCallError(_native.FCAI_ERR_CUDA, f"a pipeline wait of a product on {device} ran out; its results are wrong")


# ------------------------------------------------------------------ activations

def save_checkpoint(x: torch.Tensor, format: str = "int8") -> Checkpoint8:
    """x (``[..., channels]``, bf16, fp16 or fp32) in 8 bits."""
    keep = _code("checkpoint format", format, {k: _KEEP[k] for k in KEEPS[1:]})
    codes, scales = _host.save8(x, keep)
    _count(1)
    return Checkpoint8(codes, scales, x.shape, x.dtype, format)


def activation_forward(x: torch.Tensor, kind: str, *, keep: str | None = None):
    """y = act(x) (``kind``: "none", "relu", "gelu" (exact) or "silu"), and the
    ``Saved`` input with ``keep`` ("full", "int8", "e4m3")."""
    out = _host.activation_forward(x, _code("activation", kind, _ACT), _code("keep", keep, _KEEP))
    _count(1)
    if keep is None:
        return out
    if keep == "full":
        return out, Saved("activation", x, x.shape, x.dtype, activation=kind)
    y, codes, scales = out
    return y, Saved("activation", Checkpoint8(codes, scales, x.shape, x.dtype, keep), x.shape, x.dtype, activation=kind)


def activation_backward(grad: torch.Tensor, saved: Saved) -> torch.Tensor:
    """dx of ``activation_forward(x, ..., keep=...)``."""
    _check_saved(saved, "activation", grad)
    t, scales, keep = _parts(saved.kept)
    dx = _host.activation_backward(grad, t, scales, keep, _ACT[saved.activation])
    _count(1)
    return dx


# ----------------------------------------------------------------------- linear

def linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                   activation: str = "none", residual: torch.Tensor | None = None, keep: str | None = None):
    """``act(x @ weight.T + bias) + residual``; x ``[..., cin]``, weight
    ``[cout, cin]``, bias ``[cout]``, residual ``[..., cout]``, all bf16 or all
    fp16.  With ``keep`` also what ``linear_backward`` needs: x, and the
    activation's input unless there is no activation."""
    out = _host.linear_forward(x, weight, bias, residual, _code("activation", activation, _ACT), _code("keep", keep, _KEEP))
    if keep is None:
        _count(1)
        return out
    y, pre, kept = out[0], None, x
    if keep == "full":
        pre = out[1]
        _count(1)
    else:
        kept = Checkpoint8(out[1], out[2], x.shape, x.dtype, keep)
        if out[3] is not None:
            pre = Checkpoint8(out[3], out[4], y.shape, x.dtype, keep)
        _count(2)
    return y, Saved("linear", kept, y.shape, x.dtype, pre=pre, activation=activation, bias=bias is not None)


def linear_backward(grad: torch.Tensor, saved: Saved, weight: torch.Tensor,
                    needs: tuple[bool, bool, bool] = (True, True, True)):
    """``(dx, dweight, dbias)`` of ``linear_forward(..., keep=...)`` for the
    output's gradient; the residual's gradient is ``grad`` itself.  ``needs``
    says which are computed (the others, and dbias without a bias, are None).
    The gradient at the activation's input is rounded to the tensors' type
    between the activation's derivative and the two products, which the tensor
    cores read in that type."""
    _check_saved(saved, "linear", grad)
    t, scales, keep = _parts(saved.kept)
    pre, pre_scales, _ = _parts(saved.pre)
    mask = (1 if needs[0] else 0) | (2 if needs[1] else 0) | (4 if needs[2] and saved.bias else 0)
    out = _host.linear_backward(grad, weight, t, scales, pre, pre_scales, keep, _ACT[saved.activation], mask)
    _count(sum(o is not None for o in out) + (saved.activation != "none"))
    return out


# ------------------------------------------------------------------- layer norm

def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                       eps: float = 1e-5, keep: str | None = None):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    (bf16, fp16 or fp32; weight and bias of x's type or fp32).  With ``keep``
    also what ``layer_norm_backward`` needs: x and each row's mean and 1 / std."""
    out = _host.layer_norm_forward(x, weight, bias, eps, _code("keep", keep, _KEEP))
    _count(1)
    if keep is None:
        return out
    affine = weight if weight is not None else bias
    kept = x if keep == "full" else Checkpoint8(out[2], out[3], x.shape, x.dtype, keep)
    return out[0], Saved("layer_norm", kept, x.shape, x.dtype, stats=out[1],
                         bias=x.dtype if affine is None else affine.dtype)


def layer_norm_backward(grad: torch.Tensor, saved: Saved, weight: torch.Tensor | None = None,
                        needs: tuple[bool, bool, bool] = (True, True, True)):
    """``(dx, dweight, dbias)`` of ``layer_norm_forward(..., keep=...)``, the
    latter two in the type the norm's weight and bias had (x's type without
    them).  ``needs`` says which are computed; the others are None."""
    _check_saved(saved, "layer_norm", grad)
    t, scales, keep = _parts(saved.kept)
    mask = (1 if needs[0] else 0) | (2 if needs[1] else 0) | (4 if needs[2] else 0)
    out = _host.layer_norm_backward(grad, t, scales, saved.stats, weight, keep, mask, saved.bias is torch.float32)
    _count(2)
    return out


# ------------------------------------------------------------ differentiable forms

def _pack(ctx, saved: Saved, weight) -> None:
    """Tensors go through save_for_backward, which notices in-place changes."""
    tensors = [weight]
    ctx.formats = []
    for k in (saved.kept, saved.pre):
        if isinstance(k, Checkpoint8):
            tensors += [k.codes, k.scales]
            ctx.formats.append((k.shape, k.dtype, k.format))
        else:
            tensors += [k, None]
            ctx.formats.append(None)
    ctx.save_for_backward(*tensors, saved.stats)
    ctx.saved_as = (saved.op, saved.shape, saved.dtype, saved.activation, saved.bias)


def _unpack(ctx) -> tuple[Saved, torch.Tensor | None]:
    weight, k0, k1, p0, p1, stats = ctx.saved_tensors
    kept, pre = ((t if f is None else Checkpoint8(t, s, *f)) for t, s, f in zip((k0, p0), (k1, p1), ctx.formats))
    op, shape, dtype, kind, bias = ctx.saved_as
    return Saved(op, kept, shape, dtype, pre=pre, stats=stats, activation=kind, bias=bias), weight


class _Paused:
    """torch.jit's tracing, off for as long as an autograd function runs, which
    the trace holds as one node."""

    def __enter__(self):
        self.state = torch._C._get_tracing_state()
        torch._C._set_tracing_state(None)

    def __exit__(self, *exc):
        torch._C._set_tracing_state(self.state)
        return False


def _traced() -> bool:
    return torch._C._get_tracing_state() is not None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, keep):
        with _Paused() if _traced() else _native._NOTHING:
            y, saved = linear_forward(x, weight, bias, activation=activation, residual=residual, keep=keep)
        _pack(ctx, saved, weight)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        saved, weight = _unpack(ctx)
        n = ctx.needs_input_grad
        dx, dw, db = linear_backward(grad, saved, weight, n[:3]) if any(n[:3]) else (None, None, None)
        return dx, dw, db, grad if n[3] else None, None, None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        with _Paused() if _traced() else _native._NOTHING:
            y, saved = layer_norm_forward(x, weight, bias, eps=eps, keep=keep)
        _pack(ctx, saved, weight)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        saved, weight = _unpack(ctx)
        return layer_norm_backward(grad, saved, weight, ctx.needs_input_grad[:3]) + (None, None)


class _Activation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind, keep):
        with _Paused() if _traced() else _native._NOTHING:
            y, saved = activation_forward(x, kind, keep=keep)
        _pack(ctx, saved, None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return activation_backward(grad, _unpack(ctx)[0]), None, None


def _recorded(*tensors) -> bool:
    """Whether a call goes through its autograd function: for a gradient, or for a trace."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        return True
    return _traced()


def linear(x, weight, bias=None, *, activation: str = "none", residual=None, keep: str = "full") -> torch.Tensor:
    """Differentiable ``linear_forward``; ``keep`` says how x and the
    activation's input wait for the backward pass."""
    if keep is None:
        raise ValueError("keep must say how tensors wait for the backward pass (one of 'full', 'int8', 'e4m3')")
    if not _recorded(x, weight, bias, residual):
        return linear_forward(x, weight, bias, activation=activation, residual=residual)
    return _Linear.apply(x, weight, bias, residual, activation, keep)


def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5, keep: str = "full") -> torch.Tensor:
    """Differentiable ``layer_norm_forward``."""
    if keep is None:
        raise ValueError("keep must say how tensors wait for the backward pass (one of 'full', 'int8', 'e4m3')")
    if not _recorded(x, weight, bias):
        return layer_norm_forward(x, weight, bias, eps=eps)
    return _LayerNorm.apply(x, weight, bias, eps, keep)


def activation(x, kind: str, *, keep: str = "full") -> torch.Tensor:
    """Differentiable ``activation_forward``; ``keep`` says how x waits for the
    backward pass."""
    if keep is None:
        raise ValueError("keep must say how tensors wait for the backward pass (one of 'full', 'int8', 'e4m3')")
    if not _recorded(x):
        return activation_forward(x, kind)
    return _Activation.apply(x, kind, keep)
