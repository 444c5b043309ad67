"""The pointwise layers on the B200 at the edges of what they take: infinities
and values that leave the type's range, rows beside other rows, constant rows,
waits that ran out, large matrices, and calls at the same time."""

from __future__ import annotations

import ctypes
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from fast_compressai import _native, layers
from fast_compressai.layers import Checkpoint8
from tests import layers_reference as R
from tests.test_layers_gpu import _randn, _sliced

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


# ------------------------------------------------- transforms of torch around the calls

def _three_calls():
    w = _randn(64, 64, dtype=torch.bfloat16, seed=1, scale=0.1)
    return {"linear": lambda q: layers.linear(q, w, activation="gelu"),
            "linear trained": lambda q: layers.linear(q, w.clone().requires_grad_()),
            "layer_norm": lambda q: layers.layer_norm(q),
            "activation": lambda q: layers.activation(q, "silu")}


@pytest.mark.parametrize("name", ["linear", "layer_norm", "activation"])
def test_a_trace_runs_the_kernels_again(cuda_device, name):
    call = _three_calls()[name]
    x = _randn(40, 64, dtype=torch.bfloat16)
    traced = torch.jit.trace(lambda q: call(q) * 2, (x,), check_trace=False)
    z = _randn(40, 64, dtype=torch.bfloat16, seed=5).requires_grad_()
    out = traced(z)
    assert torch.equal(out, call(z) * 2)
    dy = _randn(40, 64, dtype=torch.bfloat16, seed=6)
    assert torch.equal(torch.autograd.grad(out, z, dy)[0], torch.autograd.grad(call(z) * 2, z, dy)[0])


@pytest.mark.parametrize("name", ["linear", "linear trained", "layer_norm", "activation"])
def test_transforms_of_torch_do_not_lose_anything(cuda_device, name):
    # refused, each with an error of its own
    call = _three_calls()[name]
    x = _randn(40, 64, dtype=torch.bfloat16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
            call(dual)
    for transform in (lambda: torch.vmap(call)(x[None]), lambda: torch.func.jvp(call, (x,), (x,)),
                      lambda: torch.func.grad(lambda q: call(q).float().sum())(x)):
        with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
            transform()


def test_a_function_with_a_forward_mode_of_its_own_uses_the_calls(cuda_device):
    w = _randn(48, 64, dtype=torch.bfloat16, seed=1, scale=0.1)

    class Linear(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return layers.linear_forward(x, w)

        @staticmethod
        def jvp(ctx, t):
            return layers.linear_forward(t, w)

    x, t = _randn(40, 64, dtype=torch.bfloat16), _randn(40, 64, dtype=torch.bfloat16, seed=2)
    with torch.autograd.forward_ad.dual_level():
        y = torch.autograd.forward_ad.unpack_dual(Linear.apply(torch.autograd.forward_ad.make_dual(x, t)))
    assert torch.equal(y.primal, layers.linear_forward(x, w)) and torch.equal(y.tangent, layers.linear_forward(t, w))


# ------------------------------------------------------------- rows beside other rows

# every way out of a product: narrow stores, padded copies, tiles, few rows, kept values
@pytest.mark.parametrize("rows,cout,keep", [(777, 577, None), (2001, 333, "full"), (40, 65, None), (20001, 333, None),
                                            (30, 577, None), (1000, 1030, "int8"), (2000, 512, None)])
@pytest.mark.parametrize("kind", ["relu", "gelu", "silu"])
def test_rows_do_not_depend_on_their_neighbours(cuda_device, kind, rows, cout, keep):
    x, w = _randn(rows, 72, dtype=torch.float16), _randn(cout, 72, dtype=torch.float16, seed=1, scale=0.12)
    other = x.clone()
    other[1::2] = _randn(rows, 72, dtype=torch.float16, seed=9)[1::2]
    a, b = (layers.linear_forward(v, w, activation=kind, keep=keep) for v in (x, other))
    a, b = (a, b) if keep is None else (a[0], b[0])
    assert torch.equal(a[::2], b[::2])


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("n", [7, 28, 112, 224, 448, 896, 1792, 3584, 7168, 8960])
@pytest.mark.parametrize("keep", [None, "full", "int8"])
def test_layer_norm_of_any_constant_row(cuda_device, dtype, n, keep):
    # n equal values of 8 significant bits sum without rounding in 32 bits (n < 2^14), so their mean is the value
    c = torch.arange(128, 256, device="cuda", dtype=torch.float32)
    x = torch.cat([c, c * 128]).to(dtype)[:, None].expand(-1, n).contiguous()
    y = layers.layer_norm_forward(x, keep=keep)
    y = y if keep is None else y[0]
    assert not y.any()


# ------------------------------------------------------------- waits that ran out

def test_check_reports_a_wait_that_ran_out(cuda_device):
    # as a replayed graph or a last product leaves it; the word is set here by the host
    word = _native.lib().fcai_linear_error_word()
    x, w = _randn(300, 64, dtype=torch.bfloat16), _randn(40, 64, dtype=torch.bfloat16, seed=1)
    want = layers.linear_forward(x, w)
    layers.check()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = layers.linear_forward(x, w)
    for device in (None, 0, "cuda:0", torch.device("cuda", 0)):
        graph.replay()
        word[0] = 1
        with pytest.raises(_native.NativeCallError, match="ran out"):
            layers.check(device)
        layers.check(device)  # reported once
    assert torch.equal(y, want) and torch.equal(layers.linear_forward(x, w), want)


def test_the_word_belongs_to_the_device(cuda_device):
    lib = _native.lib()
    with torch.cuda.device(0):
        address = ctypes.addressof(lib.fcai_linear_error_word().contents)
    assert ctypes.addressof(lib.fcai_linear_error_word().contents) == address  # one for all calls on a device
    for other in range(1, torch.cuda.device_count()):
        with torch.cuda.device(other):
            assert ctypes.addressof(lib.fcai_linear_error_word().contents) != address


@pytest.mark.parametrize("dtype", T3)
def test_activation_by_default_has_the_gradient_of_its_input(cuda_device, dtype):
    x, dy = _randn(33, 200, dtype=dtype, scale=3.0).requires_grad_(), _randn(33, 200, dtype=dtype, seed=5)
    got = torch.autograd.grad(layers.activation(x, "silu"), x, dy)[0]
    xd = x.detach().double()
    want = dy.double() * R.act_grad64(xd, "silu")
    e = dy.double().abs() * R.act_grad_bound(xd, "silu") + R.U32 * want.abs()
    R.check(got, want, e + R.half_step(dtype) * (want.abs() + e) + R.tiny(dtype))


# ------------------------------------------------- products kept in 8 bits

# widths that are no multiple of 16: codes by way of padded rows (from 6 Mi results on) or of fp32 values
@pytest.mark.parametrize("rows,cin,cout", [(40001, 24, 1030), (65537, 40, 520), (20000, 33, 5003), (33000, 64, 520), (12099, 64, 520),
                                           (12098, 64, 520), (6291457, 8, 1), (700001, 16, 9), (50, 24, 130001), (400000, 200, 17)])
@pytest.mark.parametrize("fmt,dtype", [("int8", torch.bfloat16), ("e4m3", torch.float16)])
@pytest.mark.parametrize("unaligned", [False, True])
def test_products_kept_in_8_bits_of_any_width(cuda_device, rows, cin, cout, fmt, dtype, unaligned):
    x, w = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1, scale=cin ** -0.5)
    b, r = _randn(cout, dtype=dtype, seed=2), _randn(rows, cout, dtype=dtype, seed=3)
    if unaligned:
        x, r = _sliced(x), _sliced(r)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y, saved = layers.linear_forward(x, w, b, activation="gelu", residual=r, keep=fmt)
    held = torch.cuda.memory_allocated() - before
    # scratch: padded copies of what is not aligned, and the codes once more or 6 Mi fp32 values
    copies = 2 * (rows + cout) * (cin + 8) + 4 * rows * (cout + 8)
    assert torch.cuda.max_memory_allocated() - before - held <= copies + max(rows * (cout + 15), 32 << 20) + (4 << 20)
    if rows * cout >= 6 << 20:  # the same epilogue as without codes
        assert torch.equal(y, layers.linear_forward(x, w, b, activation="gelu", residual=r))
    want, bound = R.linear_bound(x, w, b, r, "gelu", dtype)
    R.check(y, want, bound, "y")
    p64, _ = R.linear64(x, w, b)
    e = (cin + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    R.check(saved.pre.load(torch.float32), p64, e + R.keep8_step(p64.abs() + e, saved.pre.scales, fmt), "pre")
    # the scales are those of the values: a block's largest one has the largest code
    amax = torch.nn.functional.pad(p64.abs(), (0, -cout % 128)).reshape(rows, -1, 128).amax(2)
    top = 127 if fmt == "int8" else 448
    slack = torch.nn.functional.pad(e, (0, -cout % 128)).reshape(rows, -1, 128).amax(2) / top + amax / top * 2.0 ** -22
    R.check(saved.pre.scales, amax / top, slack, "scales")


# ------------------------------------------------- offsets past 32 bits, calls at the same time

def _tail(kept, rows):
    return Checkpoint8(kept.codes[rows].contiguous(), kept.scales[rows].contiguous(),
                       torch.Size((kept.codes[rows].shape[0], kept.codes.shape[1])), kept.dtype, kept.format)


# codes beside y, codes through padded rows, and everything through padded rows
@pytest.mark.parametrize("cout", [2064, 2056, 2057])
def test_last_rows_of_large_matrices(cuda_device, cout):
    dtype, rows, cin = torch.bfloat16, (1 << 20) + 3, 16  # 2.16e9 values
    tail = slice(rows - 300, rows)
    x, w, b = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1, scale=0.25), _randn(cout, dtype=dtype, seed=2)
    r, dy = _randn(rows, cout, dtype=dtype, seed=3), _randn(rows, cout, dtype=dtype, seed=4)
    y, saved = layers.linear_forward(x, w, b, activation="silu", residual=r, keep="int8")
    want, bound = R.linear_bound(x[tail], w, b, r[tail], "silu", dtype)
    R.check(y[tail], want, bound, "y")
    p64, _ = R.linear64(x[tail], w, b)
    e = (cin + 2) * 2.0 ** -23 * (x[tail].double().abs() @ w.double().abs().t() + b.double().abs())
    pre = _tail(saved.pre, tail).load(torch.float32)
    R.check(pre, p64, e + R.keep8_step(p64.abs() + e, saved.pre.scales[tail], "int8"), "pre")
    assert torch.equal(saved.pre.load()[tail], pre.to(dtype))
    dx = layers.linear_backward(dy, saved, w, needs=(True, False, False))[0]
    (g, e), _, _ = R.linear_grads(dy[tail], _tail(saved.kept, tail).load(), w, pre.double(), "silu", dtype)
    R.check(dx[tail], g, e, "dx")
    del r, saved, dx

    z, saved = layers.activation_forward(y, "relu", keep="int8")
    assert torch.equal(z[tail], torch.relu(y[tail]))
    kept, scales = R.keep8(y[tail], "int8")
    assert torch.equal(saved.kept.scales[tail], scales)
    assert torch.equal(_tail(saved.kept, tail).load(torch.float32), kept)
    dz = layers.activation_backward(dy, saved)
    assert torch.equal(dz[tail], torch.where(kept > 0, dy[tail], torch.zeros_like(dy[tail])))
    del z, dz, saved

    z, saved = layers.layer_norm_forward(y, keep="e4m3")
    want, bound, *_ = R.norm64(y[tail], None, None, 1e-5, dtype)
    R.check(z[tail], want, bound, "norm")
    kept, _ = R.keep8(y[tail], "e4m3")
    assert torch.equal(_tail(saved.kept, tail).load(torch.float32), kept)
    dx = layers.layer_norm_backward(dy, saved, needs=(True, False, False))[0]
    (g, e), _, _ = R.norm_grads(dy[tail], kept, y[tail], None, 1e-5, dtype, dtype)
    R.check(dx[tail], g, e, "norm dx")


def test_threads_call_at_the_same_time(cuda_device):
    x, dy = _randn(700, 200, dtype=torch.bfloat16), _randn(700, 264, dtype=torch.bfloat16, seed=5)
    w, b = _randn(264, 200, dtype=torch.bfloat16, seed=1, scale=0.07), _randn(264, dtype=torch.bfloat16, seed=2)
    g = _randn(200, dtype=torch.float32, seed=3)

    def step():
        h, s0 = layers.layer_norm_forward(x, g, keep="int8")
        y, s1 = layers.linear_forward(h, w, b, activation="gelu", keep="e4m3")
        dh, dw, db = layers.linear_backward(dy, s1, w)
        one = layers.linear_forward(x[:3], w, b)
        with pytest.raises(ValueError, match="fit"):  # a thread's message is its own
            layers.linear_forward(x[:, :8], w)
        return [y, dh, dw, db, one, *layers.layer_norm_backward(dh, s0, g)]

    first = step()
    torch.cuda.synchronize()

    def many(_):
        with torch.cuda.stream(torch.cuda.Stream()):
            results = [step() for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(a, e) for got in results for a, e in zip(got, first))

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(many, range(4)))


# ------------------------------------------------- the smallest sizes, other ways to call

@pytest.mark.parametrize("rows", [1, 2, 33, 300])
@pytest.mark.parametrize("cin,cout", [(1, 1), (1, 7), (2, 9), (3, 1), (7, 5), (1, 129)])
@pytest.mark.parametrize("keep", layers.KEEPS)
def test_linear_of_the_fewest_channels(cuda_device, rows, cin, cout, keep):
    dtype = torch.bfloat16
    x, w, b = _randn(rows, cin, dtype=dtype), _randn(cout, cin, dtype=dtype, seed=1), _randn(cout, dtype=dtype, seed=2)
    dy = _randn(rows, cout, dtype=dtype, seed=4)
    y, saved = layers.linear_forward(x, w, b, activation="silu", keep=keep)
    want, bound = R.linear_bound(x, w, b, None, "silu", dtype)
    R.check(y, want, bound, "y")
    kept = x if keep == "full" else saved.kept.load()
    pre = (saved.pre if keep == "full" else saved.pre.load(torch.float32)).double()
    for name, got, (g, e) in zip(("dx", "dw", "db"), layers.linear_backward(dy, saved, w),
                                 R.linear_grads(dy, kept, w, pre, "silu", dtype)):
        R.check(got, g, e, name)


@pytest.mark.parametrize("keep", layers.KEEPS)
def test_a_single_row_without_a_row_dimension(cuda_device, keep):
    x, w, g = _randn(1, 65, dtype=torch.bfloat16), _randn(41, 65, dtype=torch.bfloat16, seed=1, scale=0.1), _randn(65, dtype=torch.float32)

    def step(x):
        h, s0 = layers.layer_norm_forward(x, g, keep=keep)
        a, s1 = layers.activation_forward(h, "gelu", keep=keep)
        y, s2 = layers.linear_forward(a, w, activation="silu", keep=keep)
        da, dw, _ = layers.linear_backward(y, s2, w)
        dh = layers.activation_backward(da, s1)
        dx, dg, db = layers.layer_norm_backward(dh, s0, g)
        return h, a, y, da, dh, dx, dw, dg, db

    for flat, rows in zip(step(x[0]), step(x)):
        assert flat.shape == rows.shape or flat.shape == rows.shape[1:]
        assert torch.equal(flat.reshape(-1), rows.reshape(-1))


@pytest.mark.parametrize("keep", layers.KEEPS)
def test_saved_tensors_may_wait_elsewhere(cuda_device, keep):
    x, w = _randn(300, 65, dtype=torch.bfloat16).requires_grad_(), _randn(41, 65, dtype=torch.bfloat16, seed=1).requires_grad_()
    dy = _randn(300, 41, dtype=torch.bfloat16, seed=2)

    def grads():
        y = layers.linear(layers.activation(layers.layer_norm(x, keep=keep), "silu", keep=keep), w, activation="gelu", keep=keep)
        return torch.autograd.grad(y, [x, w], dy)

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_second_derivative_is_refused(cuda_device):
    x = _randn(8, 64, dtype=torch.float32).requires_grad_()
    dx = torch.autograd.grad(layers.activation(x, "silu").sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        torch.autograd.grad(dx.sum(), x)
