"""The pointwise training and serving layers of ``fast_compressai.layers``, as
workloads: what each one computes in plain torch operations, in 64 bits, and
through the package's own calls.

Three operators that work on rows of channels (the positions of a latent or
the tokens of a context model), each in the form serving uses and in the form
training uses:

``linear``      y = act(x W^T + b) + r;  dP = dy act'(p), dx = dP W,
                dW = dP^T x, db = sum dP, dr = dy
``norm``        layer norm over the channels, with dx and the reductions dw, db
``activation``  y = act(x) with x kept in 8 bits (blocks of 128 channels, one
                scale each), dx = dy act'(x kept)

Cases are dicts: "op", "rows", "cin" (and "cout"), "dtype", "train", "keep"
(what training keeps for its backward pass: "full", "int8" or "e4m3"), and the
operator's own choices.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 128
_EPS = 1e-5
_layers_module = None


def _layers():
    """The package's module; it lives in a folder beside this one."""
    global _layers_module
    if _layers_module is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "fast-compressai_b200"))
        from fast_compressai import layers

        _layers_module = layers
    return _layers_module


# --------------------------------------------------------------------- cases

def _linear(name, rows, cin, cout, dtype, act, *, residual=False, train=False, keep="full", bias=True):
    return {"name": name, "op": "linear", "rows": rows, "cin": cin, "cout": cout, "dtype": dtype, "act": act,
            "residual": residual, "bias": bias, "train": train, "keep": keep}


def _norm(name, rows, cin, dtype, *, wdtype="fp32", train=False, keep="full"):
    return {"name": name, "op": "norm", "rows": rows, "cin": cin, "dtype": dtype, "wdtype": wdtype, "train": train,
            "keep": keep}


def _activation(name, rows, cin, dtype, act, keep):
    return {"name": name, "op": "activation", "rows": rows, "cin": cin, "dtype": dtype, "act": act, "train": True,
            "keep": keep}


def listed():
    return [
        # an autoregressive context model's expanding layer at one latent position
        _linear("linear one position", 1, 4096, 4096, "bf16", "gelu"),
        # the same position of the 24 images of a batch, decoded together
        _linear("linear 24 positions", 24, 1024, 4096, "fp16", "silu"),
        # widths and rows that fit no tile and rows that are not 16-byte aligned
        _linear("linear ragged", 777, 321, 577, "fp16", "relu", residual=True),
        # a pointwise layer over the latents of 24 images of 512 x 768 (24 x 32 x 48 positions, 192 channels)
        _linear("linear latents", 36864, 192, 768, "bf16", "gelu"),
        # the largest: a long prompt through a wide layer, added to its residual stream
        _linear("linear wide", 16384, 8192, 8192, "bf16", "none", residual=True),
        # a training step of a wide layer, everything kept in its own type
        _linear("linear train", 8192, 4096, 4096, "bf16", "gelu", train=True),
        # a training step over the 24 x 64 x 96 positions of a transform's inner activations (128 channels),
        # kept in 8 bits
        _linear("linear train int8", 147456, 128, 512, "bf16", "silu", residual=True, train=True, keep="int8"),
        # the norm before a pointwise layer over the same latents, serving
        _norm("norm latents", 36864, 192, "bf16"),
        # training on long batches of a wide model
        _norm("norm train", 16384, 4096, "bf16", train=True),
        # odd width, 16-bit weights, input kept in 8 bits
        _norm("norm train ragged int8", 5003, 1021, "fp16", wdtype="fp16", train=True, keep="int8"),
        # the latent positions of one 512 x 768 image, inner width 512
        _activation("activation one image", 1536, 512, "bf16", "gelu", "int8"),
        # the inner activations of a wide layer over a long batch
        _activation("activation wide", 16384, 16384, "bf16", "silu", "e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    w = _log(rng, lo, hi)
    # half of the widths are the multiples of 8 that models use, the others whatever comes
    return max(8, w // 8 * 8) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(("linear", "linear", "norm", "activation"))
    act = rng.choice(("none", "relu", "gelu", "silu"))
    keep = rng.choice(("full", "int8", "e4m3"))
    if op == "linear":
        while True:
            rows, cin, cout = _log(rng, 1, 65536), _width(rng, 16, 8192), _width(rng, 16, 8192)
            train = rng.random() < 0.4
            if 2.0 * rows * cin * cout * (3 if train else 1) <= 1.0e12 and rows * max(cin, cout) <= 1 << 27:
                break
        c = _linear("", rows, cin, cout, rng.choice(("bf16", "fp16")), act, residual=rng.random() < 0.5, train=train,
                    keep=keep if train else "full", bias=rng.random() < 0.8)
    elif op == "norm":
        while True:
            rows, cin = _log(rng, 1, 262144), _width(rng, 8, 16384)
            if rows * cin <= 1 << 26:
                break
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        train = rng.random() < 0.6
        c = _norm("", rows, cin, dtype, wdtype=rng.choice(("fp32", dtype)), train=train, keep=keep if train else "full")
    else:
        while True:
            rows, cin = _log(rng, 1, 262144), _width(rng, 8, 32768)
            if rows * cin <= 1 << 27:
                break
        c = _activation("", rows, cin, rng.choice(("bf16", "fp16", "fp32")), rng.choice(("relu", "gelu", "silu")),
                        rng.choice(("int8", "e4m3")))
    del c["name"]
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    rows, cin = case["rows"], case["cin"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = {"case": case}
    # activations with a few channels much larger than the rest, as trained models have them
    gain = torch.where(torch.rand(cin, generator=g, device="cuda") < 0.02, 6.0, 1.0)
    if case["op"] == "linear":
        cout = case["cout"]
        s["x"] = (normal(rows, cin) * gain).to(dtype)
        s["w"] = (normal(cout, cin) / math.sqrt(cin)).to(dtype)
        s["b"] = (0.5 * normal(cout)).to(dtype) if case["bias"] else None
        s["r"] = normal(rows, cout).to(dtype) if case["residual"] else None
        if case["train"]:
            s["dy"] = normal(rows, cout).to(dtype)
    elif case["op"] == "norm":
        wdtype = _DTYPES[case["wdtype"]]
        s["x"] = (normal(rows, cin) * gain + 1.5 * normal(rows, 1)).to(dtype)
        s["w"] = (1.0 + 0.3 * normal(cin)).to(wdtype)
        s["b"] = (0.3 * normal(cin)).to(wdtype)
        if case["train"]:
            s["dy"] = normal(rows, cin).to(dtype)
    else:
        s["x"] = (1.5 * normal(rows, cin) * gain).to(dtype)
        s["dy"] = normal(rows, cin).to(dtype)
    return s


# ---------------------------------------------------------------- plain forms

def _act(p, kind):
    if kind == "relu":
        return torch.where(p < 0, torch.zeros_like(p), p)
    if kind == "gelu":
        return 0.5 * p * torch.special.erfc(p * -math.sqrt(0.5))
    if kind == "silu":
        return p / (1 + torch.exp(-p))
    return p


def _act_grad(p, kind):
    if kind == "relu":
        return (p > 0).to(p.dtype)
    if kind == "gelu":
        return 0.5 * torch.special.erfc(p * -math.sqrt(0.5)) + p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)
    if kind == "silu":
        t = 1 / (1 + torch.exp(-p))
        return t * (1 + p * (1 - t))
    return torch.ones_like(p)


def _kept(x, keep):
    """What an 8-bit checkpoint of the fp32 tensor x reads back as, in 32 bits: blocks of 128 channels, the scale
    amax * fl(1 / top) (at least the smallest normal number), codes round(x * fl(1 / scale))."""
    rows, cols = x.shape
    pad = -cols % _BLOCK
    v = torch.nn.functional.pad(x, (0, pad)).reshape(rows, -1, _BLOCK)
    amax = v.abs().amax(dim=2, keepdim=True)
    top = 127.0 if keep == "int8" else 448.0
    tiny = torch.finfo(torch.float32).tiny
    scale = (amax * torch.tensor(1.0 / top, dtype=torch.float32, device=x.device)).clamp(min=tiny)
    scale = torch.where(torch.isfinite(amax), scale, torch.full_like(scale, math.nan))
    q = (v * (torch.ones_like(scale) / scale)).clamp(-top, top)
    q = torch.round(q) if keep == "int8" else q.to(torch.float8_e4m3fn).float()
    return (q * scale).reshape(rows, cols + pad)[:, :cols]


def _linear_plain(s):
    c = s["case"]
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    p = x @ w.t()
    if s["b"] is not None:
        p = p + s["b"].float()
    y = _act(p, c["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    out = {"y": y.to(dtype)}
    if c["train"]:
        dp = s["dy"].float()
        if c["keep"] != "full":
            p = _kept(p, c["keep"])
            x = _kept(x, c["keep"]).to(dtype).float()  # a checkpoint reads back in its tensor's type
        if c["act"] != "none":
            dp = dp * _act_grad(p, c["act"])
        out["dx"] = (dp @ w).to(dtype)
        out["dw"] = (dp.t() @ x).to(dtype)
        if s["b"] is not None:
            out["db"] = dp.sum(dim=0).to(dtype)
    return out


def _norm_plain(s):
    c = s["case"]
    dtype = s["x"].dtype
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    mean = x.mean(dim=1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(dim=1, keepdim=True) + _EPS)
    out = {"y": ((x - mean) * rstd * w + b).to(dtype)}
    if c["train"]:
        dy = s["dy"].float()
        if c["keep"] != "full":
            x = _kept(x, c["keep"])
        xhat = (x - mean) * rstd
        t = dy * w
        dx = rstd * (t - t.mean(dim=1, keepdim=True) - xhat * (t * xhat).mean(dim=1, keepdim=True))
        out["dx"] = dx.to(dtype)
        out["dw"] = (dy * xhat).sum(dim=0).to(s["w"].dtype)
        out["db"] = dy.sum(dim=0).to(s["b"].dtype)
    return out


def _activation_plain(s):
    c = s["case"]
    x = s["x"].float()
    kept = _kept(x, c["keep"])
    return {"y": _act(x, c["act"]).to(s["x"].dtype),
            "dx": (s["dy"].float() * _act_grad(kept, c["act"])).to(s["x"].dtype),
            "kept": kept.to(s["x"].dtype)}


# ----------------------------------------------------------- the package's calls

def _linear_own(s):
    c = s["case"]
    L = _layers()
    if not c["train"]:
        return {"y": L.linear_forward(s["x"], s["w"], s["b"], activation=c["act"], residual=s["r"])}
    y, saved = L.linear_forward(s["x"], s["w"], s["b"], activation=c["act"], residual=s["r"], keep=c["keep"])
    dx, dw, db = L.linear_backward(s["dy"], saved, s["w"])
    out = {"y": y, "dx": dx, "dw": dw}
    if s["b"] is not None:
        out["db"] = db
    return out


def _norm_own(s):
    c = s["case"]
    L = _layers()
    if not c["train"]:
        return {"y": L.layer_norm_forward(s["x"], s["w"], s["b"], eps=_EPS)}
    y, saved = L.layer_norm_forward(s["x"], s["w"], s["b"], eps=_EPS, keep=c["keep"])
    dx, dw, db = L.layer_norm_backward(s["dy"], saved, s["w"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _activation_own(s):
    c = s["case"]
    L = _layers()
    y, saved = L.activation_forward(s["x"], c["act"], keep=c["keep"])
    return {"y": y, "dx": L.activation_backward(s["dy"], saved), "kept": saved.kept.load()}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _linear_own, "norm": _norm_own, "activation": _activation_own}[op](state)
    return {"linear": _linear_plain, "norm": _norm_plain, "activation": _activation_plain}[op](state)


# ------------------------------------------------------------------ 64 bits

def _kept64(x, keep):
    """The checkpoint's values from its definition: stored scales are 32-bit numbers, all else in 64 bits."""
    rows, cols = x.shape
    top = {"int8": 127.0, "e4m3": 448.0}[keep]
    blocks = -(-cols // _BLOCK)
    v = x.new_zeros(rows, blocks * _BLOCK)
    v[:, :cols] = x
    v = v.view(rows, blocks, _BLOCK)
    amax = v.abs().max(dim=2).values.float().double()
    inv_top = float(torch.tensor(1.0 / top, dtype=torch.float32))
    scale = (amax * inv_top).float().double().clamp(min=2.0 ** -126)[:, :, None]
    u = v / scale
    if keep == "int8":
        q = torch.clamp(torch.round(u), -top, top)
    else:
        # e4m3: 4 significant bits, exponents from -6 (subnormal steps of 2^-9 below)
        e = torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6)))
        step = torch.exp2(e - 3)
        q = torch.clamp(torch.round(u / step) * step, -top, top)
    return (q * scale).reshape(rows, blocks * _BLOCK)[:, :cols]


def _normal_cdf64(p):
    return 0.5 * torch.special.erfc(-p / math.sqrt(2.0))


def _act64(p, kind):
    return {"none": lambda: p, "relu": lambda: p.clamp(min=0), "gelu": lambda: p * _normal_cdf64(p),
            "silu": lambda: p * torch.sigmoid(p)}[kind]()


def _act_grad64(p, kind):
    if kind == "gelu":
        return _normal_cdf64(p) + p * torch.exp(-p.square() / 2) * (2 * math.pi) ** -0.5
    if kind == "silu":
        return torch.sigmoid(p) + p * torch.sigmoid(p) * torch.sigmoid(-p)
    return (p > 0).double() if kind == "relu" else torch.ones_like(p)


def exact(case, seed):
    s = prepare(case, seed)
    dtype, keep = _DTYPES[case["dtype"]], case["keep"]
    x = s["x"].double()
    if case["op"] == "activation":
        kept = _kept64(x, keep)
        return {"y": _act64(x, case["act"]), "dx": s["dy"].double().mul_(_act_grad64(kept, case["act"])), "kept": kept}
    if case["op"] == "norm":
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        std = (var + _EPS).sqrt()
        out = {"y": torch.addcmul(s["b"].double(), (x - mean) / std, s["w"].double())}
        if case["train"]:
            z = ((x if keep == "full" else _kept64(x, keep)) - mean) / std
            dy = s["dy"].double()
            dz = dy * s["w"].double()
            out["dx"] = (dz - dz.mean(1, True) - z * (dz * z).mean(1, True)) / std
            out["dw"], out["db"] = torch.einsum("rc,rc->c", dy, z), dy.sum(0)
        return out
    w = s["w"].double()
    p = torch.einsum("rk,nk->rn", x, w)
    if s["b"] is not None:
        p += s["b"].double()
    y = _act64(p, case["act"])
    out = {"y": y if s["r"] is None else y + s["r"].double()}
    if case["train"]:
        if keep != "full":
            p, x = _kept64(p, keep), _kept64(x, keep).to(dtype).double()
        dp = s["dy"].double() * _act_grad64(p, case["act"])
        out["dx"], out["dw"] = torch.einsum("rn,nk->rk", dp, w), torch.einsum("rn,rk->nk", dp, x)
        if s["b"] is not None:
            out["db"] = dp.sum(0)
    return out


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    rows, cin = case["rows"], case["cin"]
    n = rows * cin
    if case["op"] == "linear":
        cout = case["cout"]
        m = rows * cout
        weights = cin * cout + (cout if case["bias"] else 0)
        b = n + weights + m * (2 if case["residual"] else 1)
        f = 2.0 * rows * cin * cout
        if case["train"]:
            b += m + n + weights  # dy read; dx, dw and db written
            f *= 3
        return {"bytes": float(b * size), "flops": f}
    if case["op"] == "norm":
        ws = {"bf16": 2, "fp16": 2, "fp32": 4}[case["wdtype"]]
        b, f = 2 * n * size + 2 * cin * ws, 8.0 * n
        if case["train"]:
            b, f = b + 2 * n * size + 2 * cin * ws, f + 14.0 * n
        return {"bytes": float(b), "flops": f}
    return {"bytes": float(5 * n * size), "flops": 30.0 * n}  # x, dy; y, dx, the values kept
