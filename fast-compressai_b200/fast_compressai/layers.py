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

Every call runs on the current stream of its tensors' device and allocates its
outputs and scratch from torch's caching allocator, so calls on different
streams or in different captured graphs share nothing.  Tensors that belong to
another stream need the caller's ``wait_stream`` / ``record_stream``, as with
any torch operation.  Results are bitwise reproducible: no sum depends on the
order in which CTAs finish.  To capture a backward pass into a CUDA graph, use
the explicit calls, or release eager autograd graphs of the same parameters
first (torch's own gradient accumulation ties them to the stream they were
first used on).

Arguments that do not fit raise ``ValueError`` before anything is launched.
There is no fallback: the tensors are on a CUDA device and the native library
is built.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _native

ACTIVATIONS = ("none", "relu", "gelu", "silu")
KEEPS = ("full", "int8", "e4m3")
BLOCK = 128  # channels that share a scale (FCAI_KEEP_BLOCK)

_ACT = {name: i for i, name in enumerate(ACTIVATIONS)}
_KEEP = {None: 0, "full": 1, "int8": 2, "e4m3": 3}
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_FORWARD, _BACKWARD_INPUT, _BACKWARD_WEIGHT = 0, 1, 2


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
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DTYPE:
            raise ValueError(f"a checkpoint reads back as bf16, fp16 or fp32, not {dtype}")
        dev = self.codes.device
        out = torch.empty(self.shape, dtype=dtype, device=dev)
        rows, n = self.codes.shape
        with _native.on_device(dev):
            _check(_native.lib().fcai_checkpoint_load(
                self.codes.data_ptr(), self.scales.data_ptr(), out.data_ptr(), n, rows, n, _DTYPE[dtype],
                _KEEP[self.format], _native.stream_handle(dev)))
        _native.count_launches(1)
        return out


class Saved:
    """What a forward call kept for its backward call."""

    __slots__ = ("op", "kept", "pre", "mean", "rstd", "activation", "shape", "dtype", "bias")

    def __init__(self, op, kept, shape, dtype, pre=None, mean=None, rstd=None, activation="none", bias=None):
        self.op, self.kept, self.shape, self.dtype = op, kept, shape, dtype
        self.pre, self.mean, self.rstd, self.activation, self.bias = pre, mean, rstd, activation, bias


def _check(code: int) -> None:
    if code:
        try:
            _native.check(code)
        except _native.NativeCallError as exc:
            if exc.code == _native.FCAI_ERR_INVALID:
                raise ValueError(str(exc)) from None
            raise


def _tensor(name: str, t, device=None, dtype=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")


def _rows(t: torch.Tensor, n: int) -> tuple[torch.Tensor, int, int]:
    """(matrix, rows, row stride) of ``[..., n]``; copied only if its channels
    are not contiguous or its rows overlap or have no common stride."""
    if t.is_contiguous():
        return t, t.numel() // n, n
    if t.dim() != 2:
        t = t.reshape(-1, n)
    rows, ld = t.shape[0], t.stride(0)
    if n > 1 and t.stride(1) != 1 or ld < n:
        t, ld = t.contiguous(), n
    return t, rows, ld


@lru_cache(maxsize=4096)
def _linear_workspace(device_index: int, op: int, rows: int, cin: int, cout: int, repack: int, keep: int = 0) -> int:
    return _native.lib().fcai_linear_workspace(op, rows, cin, cout, repack, keep)


def _scratch(nbytes: int, device) -> tuple[torch.Tensor | None, int]:
    if nbytes < 0:
        raise ValueError("sizes out of range")
    if nbytes == 0:
        return None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr()


def _choice(what: str, value, known) -> None:
    if value not in known:
        raise ValueError(f"unknown {what} {value!r} (one of {', '.join(map(repr, known))})")


# ------------------------------------------------------------------ activations

def _keep8(t: torch.Tensor, rows: int, n: int, ld: int, shape, keep: str, y: torch.Tensor | None = None,
           act: int = 0) -> Checkpoint8:
    """The checkpoint of a matrix, and y = act(t) in the same pass if given."""
    dev = t.device
    codes = torch.empty((rows, n), dtype=torch.uint8, device=dev)
    scales = torch.empty((rows, -(-n // BLOCK)), dtype=torch.float32, device=dev)
    _check(_native.lib().fcai_activation_forward(
        t.data_ptr(), ld, 0 if y is None else y.data_ptr(), n, codes.data_ptr(), scales.data_ptr(), rows, n,
        _DTYPE[t.dtype], act, _KEEP[keep], _native.stream_handle(dev)))
    _native.count_launches(1)
    return Checkpoint8(codes, scales, shape, t.dtype, keep)


def save_checkpoint(x: torch.Tensor, format: str = "int8") -> Checkpoint8:
    """x (``[..., channels]``, bf16, fp16 or fp32) in 8 bits."""
    _choice("checkpoint format", format, KEEPS[1:])
    _tensor("x", x)
    if x.dtype not in _DTYPE or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("a checkpoint takes [..., channels] tensors of bf16, fp16 or fp32")
    n = x.shape[-1]
    with _native.on_device(x.device):
        m, rows, ld = _rows(x, n)
        return _keep8(m, rows, n, ld, x.shape, format)


def activation_forward(x: torch.Tensor, kind: str, *, keep: str | None = None):
    """y = act(x) (``kind``: "none", "relu", "gelu" (exact) or "silu"), and the
    ``Saved`` input with ``keep`` ("full", "int8", "e4m3")."""
    _choice("activation", kind, ACTIVATIONS)
    _tensor("x", x)
    if x.dtype not in _DTYPE or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("activations take [..., channels] tensors of bf16, fp16 or fp32")
    if keep is not None:
        _choice("keep", keep, KEEPS)
    dev, n, shape = x.device, x.shape[-1], x.shape
    y = torch.empty(shape, dtype=x.dtype, device=dev)
    with _native.on_device(dev):
        m, rows, ld = _rows(x, n)
        if keep == "int8" or keep == "e4m3":
            kept = _keep8(m, rows, n, ld, shape, keep, y, _ACT[kind])
        else:
            kept = x
            _check(_native.lib().fcai_activation_forward(
                m.data_ptr(), ld, y.data_ptr(), n, 0, 0, rows, n, _DTYPE[x.dtype], _ACT[kind], 0,
                _native.stream_handle(dev)))
            _native.count_launches(1)
    if keep is None:
        return y
    return y, Saved("activation", kept, shape, x.dtype, activation=kind)


def _act_backward(g, rows, n, ldg, kept, kind, dx, bias_grad):
    """dx = g * act'(kept) and its column sums (either may be None)."""
    dev, lib = g.device, _native.lib()
    act = _ACT[kind]
    x = codes = scales = ldx = 0
    keep = 1
    if act:
        if isinstance(kept, Checkpoint8):
            codes, scales, keep = kept.codes.data_ptr(), kept.scales.data_ptr(), _KEEP[kept.format]
        else:
            m, _, ldx = _rows(kept, n)
            x = m.data_ptr()
    ws, wsp, nbytes = None, 0, 0
    if bias_grad is not None:
        nbytes = lib.fcai_activation_workspace(rows, n)
        ws, wsp = _scratch(nbytes, dev)
    _check(lib.fcai_activation_backward(
        g.data_ptr(), ldg, x, ldx, codes, scales, 0 if dx is None else dx.data_ptr(), n,
        0 if bias_grad is None else bias_grad.data_ptr(), rows, n, _DTYPE[g.dtype], act, keep, wsp, nbytes,
        _native.stream_handle(dev)))
    _native.count_launches(1 if bias_grad is None else 2)


def activation_backward(grad: torch.Tensor, saved: Saved) -> torch.Tensor:
    """dx of ``activation_forward(x, ..., keep=...)``."""
    _saved(saved, "activation")
    _grad(grad, saved.shape, saved.dtype, saved.kept)
    n = saved.shape[-1]
    dx = torch.empty(saved.shape, dtype=saved.dtype, device=grad.device)
    with _native.on_device(grad.device):
        g, rows, ldg = _rows(grad, n)
        _act_backward(g, rows, n, ldg, saved.kept, saved.activation, dx, None)
    return dx


def _saved(saved, op: str) -> None:
    if not isinstance(saved, Saved) or saved.op != op:
        raise ValueError(f"expected what {op}_forward kept")


def _grad(grad, shape, dtype, kept) -> None:
    _tensor("grad", grad, (kept.codes if isinstance(kept, Checkpoint8) else kept).device, dtype)
    if grad.shape != shape:
        raise ValueError(f"grad has shape {tuple(grad.shape)}, expected {tuple(shape)}")


# ----------------------------------------------------------------------- linear

def linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                   activation: str = "none", residual: torch.Tensor | None = None, keep: str | None = None):
    """``act(x @ weight.T + bias) + residual``; x ``[..., cin]``, weight
    ``[cout, cin]``, bias ``[cout]``, residual ``[..., cout]``, all bf16 or all
    fp16.  With ``keep`` also what ``linear_backward`` needs: x, and the
    activation's input unless there is no activation."""
    _choice("activation", activation, ACTIVATIONS)
    if keep is not None:
        _choice("keep", keep, KEEPS)
    _tensor("x", x)
    dev, dtype = x.device, x.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"linear takes bf16 or fp16, not {dtype}")
    _tensor("weight", weight, dev, dtype)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or not weight.numel():
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit")
    cout, cin = weight.shape
    out_shape = x.shape[:-1] + (cout,)
    if bias is not None:
        _tensor("bias", bias, dev, dtype)
        if bias.shape != (cout,):
            raise ValueError(f"linear: bias has shape {tuple(bias.shape)}, expected ({cout},)")
        bias = bias.contiguous()
    if residual is not None:
        _tensor("residual", residual, dev, dtype)
        if residual.shape != out_shape:
            raise ValueError(f"linear: residual has shape {tuple(residual.shape)}, expected {tuple(out_shape)}")
    with _native.on_device(dev):
        y = torch.empty(out_shape, dtype=dtype, device=dev)
        m, rows, ldx = _rows(x, cin)
        w, _, ldw = _rows(weight, cin)
        r, ldr = 0, 0
        if residual is not None:
            residual, _, ldr = _rows(residual, cout)
            r = residual.data_ptr()
        pre = codes = scales = None
        pk = 0 if activation == "none" else _KEEP[keep]  # what of the activation's input is kept
        if pk == 1:
            pre = torch.empty(out_shape, dtype=dtype, device=dev)
        elif pk:
            codes = torch.empty((rows, cout), dtype=torch.uint8, device=dev)
            scales = torch.empty((rows, -(-cout // BLOCK)), dtype=torch.float32, device=dev)
            if cout % 8 == 0:  # the codes leave with y's rows, in wide accesses
                if bias is not None and bias.data_ptr() & 15:
                    bias = bias.clone()
                if residual is not None and (r | 2 * ldr) & 15:
                    residual = residual.reshape(-1, cout).clone(memory_format=torch.contiguous_format)
                    r, ldr = residual.data_ptr(), cout
        xp, wp = m.data_ptr(), w.data_ptr()
        repack = (1 if (xp | 2 * ldx) & 15 else 0) | (2 if (wp | 2 * ldw) & 15 else 0)
        nbytes = _linear_workspace(dev.index, _FORWARD, rows, cin, cout, repack, pk)
        ws, wsp = _scratch(nbytes, dev)
        _check(_native.lib().fcai_linear_forward(
            xp, ldx, wp, ldw, 0 if bias is None else bias.data_ptr(), r, ldr, y.data_ptr(), cout,
            0 if pre is None else pre.data_ptr(), cout, 0 if codes is None else codes.data_ptr(),
            0 if codes is None else scales.data_ptr(), rows, cin, cout, _DTYPE[dtype], _ACT[activation], pk, wsp, nbytes,
            _native.stream_handle(dev)))
        _native.count_launches(1)
        if keep is None:
            return y
        kept = x
        if keep != "full":
            kept = _keep8(m, rows, cin, ldx, x.shape, keep)
            if pk:
                pre = Checkpoint8(codes, scales, out_shape, dtype, keep)
    return y, Saved("linear", kept, out_shape, dtype, pre=pre, activation=activation, bias=bias is not None)


def linear_backward(grad: torch.Tensor, saved: Saved, weight: torch.Tensor,
                    needs: tuple[bool, bool, bool] = (True, True, True)):
    """``(dx, dweight, dbias)`` of ``linear_forward(..., keep=...)`` for the
    output's gradient; the residual's gradient is ``grad`` itself.  ``needs``
    says which are computed (the others, and dbias without a bias, are None).
    The gradient at the activation's input is rounded to the tensors' type
    between the activation's derivative and the two products, which the tensor
    cores read in that type."""
    _saved(saved, "linear")
    dtype = saved.dtype
    _grad(grad, saved.shape, dtype, saved.kept)
    dev = grad.device
    _tensor("weight", weight, dev, dtype)
    x_shape = saved.kept.shape
    cin, cout = x_shape[-1], saved.shape[-1]
    if weight.shape != (cout, cin):
        raise ValueError(f"linear: weight has shape {tuple(weight.shape)}, expected ({cout}, {cin})")
    lib, code = _native.lib(), _DTYPE[dtype]
    need_x, need_w, need_b = needs[0], needs[1], needs[2] and saved.bias
    with _native.on_device(dev):
        stream = _native.stream_handle(dev)
        g, rows, ldg = _rows(grad, cout)
        db = torch.empty(cout, dtype=dtype, device=dev) if need_b else None
        if saved.activation != "none":
            dp = torch.empty((rows, cout), dtype=dtype, device=dev)
            _act_backward(g, rows, cout, ldg, saved.pre, saved.activation, dp, db)
            g, ldg = dp, cout
        elif need_b:
            _act_backward(g, rows, cout, ldg, None, "none", None, db)
        gp = g.data_ptr()
        gpack = 1 if (gp | 2 * ldg) & 15 else 0
        dx = dw = None
        if need_x:
            dx = torch.empty(x_shape, dtype=dtype, device=dev)
            w, _, ldw = _rows(weight, cin)
            wp = w.data_ptr()
            nbytes = _linear_workspace(dev.index, _BACKWARD_INPUT, rows, cin, cout,
                                       gpack | (2 if (wp | 2 * ldw) & 15 else 0))
            ws, wsp = _scratch(nbytes, dev)
            _check(lib.fcai_linear_backward_input(gp, ldg, wp, ldw, dx.data_ptr(), cin, rows, cin, cout, code, wsp,
                                                  nbytes, stream))
            _native.count_launches(1)
        if need_w:
            dw = torch.empty((cout, cin), dtype=dtype, device=dev)
            x = saved.kept.load() if isinstance(saved.kept, Checkpoint8) else saved.kept
            m, _, ldx = _rows(x, cin)
            xp = m.data_ptr()
            nbytes = _linear_workspace(dev.index, _BACKWARD_WEIGHT, rows, cin, cout,
                                       gpack | (2 if (xp | 2 * ldx) & 15 else 0))
            ws, wsp = _scratch(nbytes, dev)
            _check(lib.fcai_linear_backward_weight(gp, ldg, xp, ldx, dw.data_ptr(), cin, rows, cin, cout, code, wsp,
                                                   nbytes, stream))
            _native.count_launches(1)
    return dx, dw, db


# ------------------------------------------------------------------- layer norm

def _affine(x, weight, bias, n):
    """The norm's weight and bias, contiguous, and their type."""
    wdtype = x.dtype
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _tensor(name, t, x.device)
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise ValueError(f"layer_norm: {name} must have x's dtype or fp32")
        if t.shape != (n,):
            raise ValueError(f"layer_norm: {name} has shape {tuple(t.shape)}, expected ({n},)")
        wdtype = t.dtype
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("layer_norm: weight and bias must have one dtype")
    return (None if weight is None else weight.contiguous()), (None if bias is None else bias.contiguous()), wdtype


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                       eps: float = 1e-5, keep: str | None = None):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    (bf16, fp16 or fp32; weight and bias of x's type or fp32).  With ``keep``
    also what ``layer_norm_backward`` needs: x and each row's mean and 1 / std."""
    if keep is not None:
        _choice("keep", keep, KEEPS)
    _tensor("x", x)
    dtype = x.dtype
    if dtype not in _DTYPE or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm takes [..., channels] tensors of bf16, fp16 or fp32")
    dev, shape, n = x.device, x.shape, x.shape[-1]
    w, b, wdtype = _affine(x, weight, bias, n)
    with _native.on_device(dev):
        y = torch.empty(shape, dtype=dtype, device=dev)
        m, rows, ld = _rows(x, n)
        mean = rstd = codes = scales = None
        if keep is not None:
            stats = torch.empty((2, rows), dtype=torch.float32, device=dev)
            mean, rstd = stats[0], stats[1]
            if keep != "full":
                codes = torch.empty((rows, n), dtype=torch.uint8, device=dev)
                scales = torch.empty((rows, -(-n // BLOCK)), dtype=torch.float32, device=dev)
        _check(_native.lib().fcai_layer_norm_forward(
            m.data_ptr(), ld, 0 if w is None else w.data_ptr(), 0 if b is None else b.data_ptr(), _DTYPE[wdtype],
            y.data_ptr(), n, 0 if mean is None else mean.data_ptr(), 0 if rstd is None else rstd.data_ptr(),
            0 if codes is None else codes.data_ptr(), 0 if scales is None else scales.data_ptr(), rows, n, eps,
            _DTYPE[dtype], _KEEP[keep], _native.stream_handle(dev)))
        _native.count_launches(1)
    if keep is None:
        return y
    kept = x if codes is None else Checkpoint8(codes, scales, shape, dtype, keep)
    return y, Saved("layer_norm", kept, shape, dtype, mean=mean, rstd=rstd, bias=wdtype)


def layer_norm_backward(grad: torch.Tensor, saved: Saved, weight: torch.Tensor | None = None,
                        needs: tuple[bool, bool, bool] = (True, True, True)):
    """``(dx, dweight, dbias)`` of ``layer_norm_forward(..., keep=...)``, the
    latter two in the type the norm's weight and bias had (x's type without
    them).  ``needs`` says which are computed; the others are None."""
    _saved(saved, "layer_norm")
    dtype, shape = saved.dtype, saved.shape
    kept = saved.kept
    _grad(grad, shape, dtype, kept)
    n, dev, lib = shape[-1], grad.device, _native.lib()
    w = None
    wdtype = saved.bias
    if weight is not None:
        _tensor("weight", weight, dev, wdtype)
        if weight.shape != (n,):
            raise ValueError(f"layer_norm: weight has shape {tuple(weight.shape)}, expected ({n},)")
        w = weight.contiguous()
    if not any(needs):
        return None, None, None
    with _native.on_device(dev):
        g, rows, ldg = _rows(grad, n)
        x = codes = scales = ldx = 0
        keep = 1
        if isinstance(kept, Checkpoint8):
            codes, scales, keep = kept.codes.data_ptr(), kept.scales.data_ptr(), _KEEP[kept.format]
        else:
            m, _, ldx = _rows(kept, n)
            x = m.data_ptr()
        dx = torch.empty(shape, dtype=dtype, device=dev) if needs[0] else None
        dw = torch.empty(n, dtype=wdtype, device=dev) if needs[1] else None
        db = torch.empty(n, dtype=wdtype, device=dev) if needs[2] else None
        nbytes = lib.fcai_layer_norm_workspace(rows, n)
        ws, wsp = _scratch(nbytes, dev)
        _check(lib.fcai_layer_norm_backward(
            g.data_ptr(), ldg, x, ldx, codes, scales, saved.mean.data_ptr(), saved.rstd.data_ptr(),
            0 if w is None else w.data_ptr(), _DTYPE[wdtype], 0 if dx is None else dx.data_ptr(), n,
            0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(), rows, n, _DTYPE[dtype], keep, wsp,
            nbytes, _native.stream_handle(dev)))
        _native.count_launches(2 + (dw is not None) + (db is not None))
    return dx, dw, db


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
    ctx.save_for_backward(*tensors, saved.mean, saved.rstd)
    ctx.saved_as = (saved.op, saved.shape, saved.dtype, saved.activation, saved.bias)


def _unpack(ctx) -> tuple[Saved, torch.Tensor | None]:
    weight, k0, k1, p0, p1, mean, rstd = ctx.saved_tensors
    kept, pre = ((t if f is None else Checkpoint8(t, s, *f)) for t, s, f in zip((k0, p0), (k1, p1), ctx.formats))
    op, shape, dtype, kind, bias = ctx.saved_as
    return Saved(op, kept, shape, dtype, pre=pre, mean=mean, rstd=rstd, activation=kind, bias=bias), weight


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, keep):
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
        y, saved = activation_forward(x, kind, keep=keep)
        _pack(ctx, saved, None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return activation_backward(grad, _unpack(ctx)[0]), None, None


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def linear(x, weight, bias=None, *, activation: str = "none", residual=None, keep: str = "full") -> torch.Tensor:
    """Differentiable ``linear_forward``; ``keep`` says how x and the
    activation's input wait for the backward pass."""
    _choice("keep", keep, KEEPS)
    if not _needs_grad(x, weight, bias, residual):
        return linear_forward(x, weight, bias, activation=activation, residual=residual)
    return _Linear.apply(x, weight, bias, residual, activation, keep)


def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5, keep: str = "full") -> torch.Tensor:
    """Differentiable ``layer_norm_forward``."""
    _choice("keep", keep, KEEPS)
    if not _needs_grad(x, weight, bias):
        return layer_norm_forward(x, weight, bias, eps=eps)
    return _LayerNorm.apply(x, weight, bias, eps, keep)


def activation(x, kind: str, *, keep: str = "int8") -> torch.Tensor:
    """Differentiable ``activation_forward``; keeps x in 8 bits unless asked otherwise."""
    _choice("keep", keep, KEEPS)
    if not _needs_grad(x):
        return activation_forward(x, kind)
    return _Activation.apply(x, kind, keep)
