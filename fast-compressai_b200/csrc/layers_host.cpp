// layers_host.cpp -- the calls of fast_compressai.layers from tensors down to
// the C ABI of include/fcai_layers.h: checks, outputs and scratch from torch's
// allocator, the current stream of the tensors' device.
//
// A compiled module because these calls are often microseconds of GPU time (one
// position of a latent through a layer): checking a dozen tensor attributes and
// converting twenty arguments in Python takes 8 to 13 us a call; here a whole call,
// its launch and Python's side included, takes 4 to 5.
// Plain CPython functions over torch's C++ tensors; every C++ exception ends in
// a Python one.
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Size.h>

#include <string>

#include "../../include/fcai_layers.h"

namespace {

struct Refused {  // becomes ValueError
    std::string what;
};
struct NativeStatus {  // becomes NativeCallError
    int code;
};

[[noreturn]] void refuse(std::string what) { throw Refused{std::move(what)}; }

std::string sizes_text(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}

// The calls write their outputs past torch's dispatcher, where nothing follows what
// they do: a trace would hold their results as constants, and a forward-mode tangent
// would be lost.  Both are refused instead.  (Inside an autograd function, whose
// forward runs with forward mode off, torch looks after tangents itself.)
void check_not_traced() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    if (at::tracer::impl::is_dispatch_enabled() ||
        (Modes::any_modes_set() && Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY)))
        refuse("this call cannot be traced (torch.jit.trace takes layers.linear, layers.layer_norm and layers.activation)");
}
const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
        refuse(std::string(name) + " has a forward-mode tangent, which these calls do not carry on");
    if (!t.is_cuda()) refuse(std::string(name) + " must be on a CUDA device");
    if (t.layout() != at::kStrided || t.is_neg() || t._is_zerotensor()) refuse(std::string(name) + " must be a dense tensor");
    return t;
}
void same(const at::Tensor &t, const char *name, const at::Tensor &as) {
    if (t.device() != as.device()) refuse(std::string(name) + " is on " + t.device().str() + ", expected " + as.device().str());
    if (t.scalar_type() != as.scalar_type())
        refuse(std::string(name) + " has dtype " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(as.scalar_type()));
}
int dtype_code(const at::Tensor &t, const char *what) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return FCAI_DTYPE_BF16;
        case at::kHalf: return FCAI_DTYPE_F16;
        case at::kFloat: return FCAI_DTYPE_F32;
        default: refuse(std::string(what) + " takes bf16, fp16 or fp32 tensors, not " + c10::toString(t.scalar_type()));
    }
}
int64_t channels(const at::Tensor &t, const char *what) {
    if (t.dim() < 1 || t.size(-1) < 1) refuse(std::string(what) + " takes [..., channels] tensors");
    if (t.size(-1) > (1 << 24)) refuse(std::string(what) + ": too many channels");
    return t.size(-1);
}
void status(int code) {
    if (code) throw NativeStatus{code};
}

// [..., n] as rows of channels; copied only if its channels are not contiguous
// or its rows overlap or have no common stride.
struct Rows {
    at::Tensor hold;
    const void *p;
    int64_t ld, rows;
};
Rows rows_of(const at::Tensor &t, int64_t n) {
    if (t.is_contiguous()) return {t, t.data_ptr(), n, t.numel() / n};
    at::Tensor m = t.dim() == 2 ? t : t.reshape({-1, n});
    if ((n > 1 && m.stride(1) != 1) || m.stride(0) < n) m = m.contiguous();
    const int64_t rows = m.size(0), ld = m.stride(0);
    const void *p = m.data_ptr();
    return {std::move(m), p, ld < n ? n : ld, rows};
}
bool unaligned(const void *p, int64_t ld) { return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(2 * ld)) & 15) != 0; }

fcai_stream_t stream_of(const at::Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// A contiguous tensor on like's device, straight from the allocator (the
// dispatcher costs as much again); the device is current.
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor &like, at::ScalarType type) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor &like) { return fresh(sizes, like, like.scalar_type()); }
// Memory for one call's kernels; back to the current stream's pool when it goes out of scope.
struct Scratch {
    c10::DataPtr p;
    void *get() const { return p.get(); }
};
Scratch scratch(int64_t bytes) {
    if (bytes < 0) refuse("sizes out of range");
    return {bytes ? c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes) : c10::DataPtr()};
}
void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Codes {
    at::Tensor codes, scales;
};
Codes new_codes(const at::Tensor &like, int64_t rows, int64_t n) {
    return {fresh({rows, n}, like, at::kByte),
            fresh({rows, (n + FCAI_KEEP_BLOCK - 1) / FCAI_KEEP_BLOCK}, like, at::kFloat)};
}
Codes save8(const at::Tensor &like, const Rows &m, int64_t n, int keep, void *y = nullptr, int act = 0) {
    Codes c = new_codes(like, m.rows, n);
    status(fcai_activation_forward(m.p, m.ld, y, n, c.codes.data_ptr(), c.scales.data_ptr<float>(), m.rows, (int)n,
                                   dtype_code(like, "a checkpoint"), act, keep, stream_of(like)));
    return c;
}

long integer(PyObject *o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse("an integer is expected");
    }
    return v;
}
PyObject *wrap(const at::Tensor &t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
template <typename... Ts>
PyObject *wrap_all(const Ts &...ts) {
    PyObject *out = PyTuple_New(sizeof...(ts));
    if (!out) return nullptr;
    Py_ssize_t i = 0;
    bool ok = true;
    auto put = [&](const at::Tensor &t) {
        PyObject *o = ok ? wrap(t) : nullptr;
        if (!o) ok = false;
        else PyTuple_SET_ITEM(out, i++, o);
    };
    (put(ts), ...);
    if (!ok) {
        Py_DECREF(out);
        return nullptr;
    }
    return out;
}

// Runs a call; C++ exceptions become Python ones.
template <typename F>
PyObject *guarded(Py_ssize_t n, Py_ssize_t want, F &&f) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
        return nullptr;
    }
    try {
        check_not_traced();
        const c10::AutoGradMode no_graph(false);  // a copy made here is no operation of the caller's
        return f();
    } catch (const Refused &r) {
        PyErr_SetString(PyExc_ValueError, r.what.c_str());
    } catch (const NativeStatus &s) {
        const std::string msg = fcai_last_error();
        if (s.code == FCAI_ERR_INVALID) {
            PyErr_SetString(PyExc_ValueError, msg.c_str());
        } else {
            PyObject *mod = PyImport_ImportModule("fast_compressai._native");
            PyObject *cls = mod ? PyObject_GetAttrString(mod, "NativeCallError") : nullptr;
            PyObject *exc = cls ? PyObject_CallFunction(cls, "is", s.code, msg.c_str()) : nullptr;
            if (exc) PyErr_SetObject(cls, exc);
            Py_XDECREF(exc);
            Py_XDECREF(cls);
            Py_XDECREF(mod);
        }
    } catch (const c10::OutOfMemoryError &e) {
        PyObject *mod = PyImport_ImportModule("torch");
        PyObject *cls = mod ? PyObject_GetAttrString(mod, "OutOfMemoryError") : nullptr;
        PyErr_SetString(cls ? cls : PyExc_RuntimeError, e.what_without_backtrace());
        Py_XDECREF(cls);
        Py_XDECREF(mod);
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// save8(x, keep) -> (codes, scales)
PyObject *py_save8(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 2, [&] {
        const at::Tensor &x = tensor(a[0], "x");
        dtype_code(x, "a checkpoint");
        const int64_t c = channels(x, "a checkpoint");
        const c10::cuda::CUDAGuard guard(x.device());
        const Codes k = save8(x, rows_of(x, c), c, (int)integer(a[1]));
        return wrap_all(k.codes, k.scales);
    });
}

// What a backward call reads: a tensor, or codes and scales.
struct Kept {
    Rows m{};
    const void *codes = nullptr;
    const float *scales = nullptr;
    int keep = FCAI_KEEP_FULL;
};
Kept kept_of(PyObject *x, PyObject *scales, int keep, int64_t n, const at::Tensor &as) {
    Kept k;
    const at::Tensor &t = tensor(x, "what was kept");
    if (t.device() != as.device()) refuse("what was kept is on " + t.device().str() + ", expected " + as.device().str());
    if (keep >= FCAI_KEEP_INT8) {
        const at::Tensor &s = tensor(scales, "the scales kept");
        if (t.scalar_type() != at::kByte || s.scalar_type() != at::kFloat || t.dim() != 2 || t.size(1) != n || !t.is_contiguous() ||
            !s.is_contiguous() || s.numel() != t.size(0) * ((n + FCAI_KEEP_BLOCK - 1) / FCAI_KEEP_BLOCK) || s.device() != t.device())
            refuse("the checkpoint's codes and scales do not fit each other");
        k.codes = t.data_ptr();
        k.scales = s.data_ptr<float>();
        k.m.rows = t.size(0);
        k.keep = keep;
    } else {
        if (t.dim() < 1 || t.size(-1) != n) refuse("what was kept does not fit the gradient");
        same(t, "what was kept", as);
        k.m = rows_of(t, n);
    }
    return k;
}

// load8(codes, scales, keep, like or None, dtype code, shape) -> values
PyObject *py_load8(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 5, [&] {
        const at::Tensor &codes = tensor(a[0], "codes");
        const int keep = (int)integer(a[2]), dtype = (int)integer(a[3]);
        if (codes.dim() != 2) refuse("codes are [rows, channels]");
        const int64_t c = codes.size(1);
        const c10::cuda::CUDAGuard guard(codes.device());
        const Kept k = kept_of(a[0], a[1], keep, c, codes);
        std::vector<int64_t> shape;
        if (!PyTuple_Check(a[4])) refuse("a shape is expected");
        int64_t total = 1;
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[4]); ++i) {
            shape.push_back(integer(PyTuple_GET_ITEM(a[4], i)));
            total *= shape.back();
        }
        if (total != codes.numel() || shape.empty() || shape.back() != c) refuse("the shape does not fit the codes");
        const at::ScalarType types[3] = {at::kBFloat16, at::kHalf, at::kFloat};
        if (dtype < 0 || dtype > 2) refuse("unknown dtype");
        at::Tensor out = fresh(shape, codes, types[dtype]);
        status(fcai_checkpoint_load(k.codes, k.scales, out.data_ptr(), c, k.m.rows, (int)c, dtype, keep, stream_of(codes)));
        return wrap(out);
    });
}

// activation_forward(x, act, keep) -> y, or (y, codes, scales) for an 8-bit keep
PyObject *py_activation_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 3, [&] {
        const at::Tensor &x = tensor(a[0], "x");
        const int act = (int)integer(a[1]), keep = (int)integer(a[2]), dtype = dtype_code(x, "an activation");
        const int64_t c = channels(x, "an activation");
        const c10::cuda::CUDAGuard guard(x.device());
        const Rows m = rows_of(x, c);
        at::Tensor y = fresh(x.sizes(), x);
        if (keep >= FCAI_KEEP_INT8) {
            const Codes k = save8(x, m, c, keep, y.data_ptr(), act);
            return wrap_all(y, k.codes, k.scales);
        }
        status(fcai_activation_forward(m.p, m.ld, y.data_ptr(), c, nullptr, nullptr, m.rows, (int)c, dtype, act, FCAI_KEEP_NONE,
                                       stream_of(x)));
        return wrap(y);
    });
}

// dx = g * act'(kept) and its column sums (either may be undefined)
void act_backward(const at::Tensor &like, const Rows &g, int64_t n, const Kept &k, int act, const at::Tensor &dx, const at::Tensor &sums,
                  int64_t lddx) {
    Scratch ws;
    int64_t bytes = 0;
    if (sums.defined()) {
        bytes = fcai_activation_workspace(g.rows, (int)n);
        ws = scratch(bytes);
    }
    status(fcai_activation_backward(g.p, g.ld, k.m.p, k.m.ld, k.codes, k.scales, ptr(dx), lddx, ptr(sums), g.rows, (int)n,
                                    dtype_code(like, "an activation"), act, k.keep, ws.get(), bytes, stream_of(like)));
}

// activation_backward(grad, kept or codes, scales, keep, act) -> dx
PyObject *py_activation_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 5, [&] {
        const at::Tensor &grad = tensor(a[0], "grad");
        const int keep = (int)integer(a[3]), act = (int)integer(a[4]);
        const int64_t c = channels(grad, "an activation");
        const c10::cuda::CUDAGuard guard(grad.device());
        const Rows g = rows_of(grad, c);
        const Kept k = kept_of(a[1], a[2], keep, c, grad);
        if (k.m.rows != g.rows) refuse("grad does not fit what was kept");
        at::Tensor dx = fresh(grad.sizes(), grad);
        act_backward(grad, g, c, k, act, dx, at::Tensor(), c);
        return wrap(dx);
    });
}

void check_linear(const at::Tensor &x, const at::Tensor &w) {
    if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf)
        refuse(std::string("linear takes bf16 or fp16, not ") + c10::toString(x.scalar_type()));
    same(w, "weight", x);
    if (w.dim() != 2 || w.numel() == 0 || w.size(0) > (1 << 24) || w.size(1) > (1 << 24))
        refuse("linear: weight must be [cout, cin], got " + sizes_text(w.sizes()));
}

// linear_forward(x, weight, bias, residual, act, keep)
//   -> y                                                keep none
//   -> (y, pre or None)                                 keep full
//   -> (y, x codes, x scales, codes or None, scales or None)  keep in 8 bits
PyObject *py_linear_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 6, [&] {
        const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "weight");
        const int act = (int)integer(a[4]), keep = (int)integer(a[5]);
        check_linear(x, w);
        const int64_t cout = w.size(0), cin = w.size(1);
        if (x.dim() < 1 || x.size(-1) != cin) refuse("linear: x " + sizes_text(x.sizes()) + " and weight " + sizes_text(w.sizes()) + " do not fit");
        at::DimVector shape(x.sizes().begin(), x.sizes().end());
        shape.back() = cout;
        const c10::cuda::CUDAGuard guard(x.device());
        at::Tensor bias;
        if (a[2] != Py_None) {
            bias = tensor(a[2], "bias");
            same(bias, "bias", x);
            if (bias.dim() != 1 || bias.size(0) != cout) refuse("linear: bias has shape " + sizes_text(bias.sizes()) + ", expected " + sizes_text({cout}));
            bias = bias.contiguous();
        }
        Rows r{};
        if (a[3] != Py_None) {
            const at::Tensor &res = tensor(a[3], "residual");
            same(res, "residual", x);
            if (res.sizes() != at::IntArrayRef(shape)) refuse("linear: residual has shape " + sizes_text(res.sizes()) + ", expected " + sizes_text(shape));
            r = rows_of(res, cout);
        }
        const Rows m = rows_of(x, cin), wm = rows_of(w, cin);
        at::Tensor y = fresh(shape, x), pre;
        // pre: the activation's input rounded to the type, as keep "full" says; padded rows, which leave the kernel (and enter
        // the backward pass) in wide accesses
        const int64_t ldpre = (cout + 7) / 8 * 8;
        Codes k;
        const int kp = act == FCAI_ACT_NONE ? FCAI_KEEP_NONE : keep;  // what of the activation's input is kept
        if (kp == FCAI_KEEP_FULL) pre = fresh({m.rows, ldpre}, x);
        if (kp >= FCAI_KEEP_INT8) {
            k = new_codes(x, m.rows, cout);
            if (cout % 8 == 0) {  // the codes leave with y's rows, in wide accesses
                if (bias.defined() && unaligned(bias.data_ptr(), 0)) bias = bias.clone();
                if (r.p && unaligned(r.p, r.ld)) {
                    at::Tensor copy = r.hold.reshape({-1, cout}).clone(at::MemoryFormat::Contiguous);
                    const void *p = copy.data_ptr();
                    r = Rows{std::move(copy), p, cout, m.rows};
                }
            }
        }
        const int repack = (unaligned(m.p, m.ld) ? 1 : 0) | (unaligned(wm.p, wm.ld) ? 2 : 0) | (unaligned(y.data_ptr(), cout) ? 4 : 0) |
                           (r.p && unaligned(r.p, r.ld) ? 8 : 0) | (bias.defined() && unaligned(bias.data_ptr(), cout) ? 16 : 0);
        const int64_t bytes = fcai_linear_workspace(FCAI_LINEAR_FORWARD, m.rows, (int)cin, (int)cout, repack, kp);
        const Scratch ws = scratch(bytes);
        status(fcai_linear_forward(m.p, m.ld, wm.p, wm.ld, ptr(bias), r.p, r.ld, y.data_ptr(), cout, ptr(pre), ldpre, ptr(k.codes),
                                   static_cast<float *>(ptr(k.scales)), m.rows, (int)cin, (int)cout, dtype_code(x, "linear"), act, kp,
                                   ws.get(), bytes, stream_of(x)));
        if (keep == FCAI_KEEP_NONE) return wrap(y);
        if (keep == FCAI_KEEP_FULL) return wrap_all(y, pre.defined() && ldpre != cout ? pre.narrow(1, 0, cout) : pre);
        const Codes kx = save8(x, m, cin, keep);
        return wrap_all(y, kx.codes, kx.scales, k.codes, k.scales);
    });
}

// linear_backward(grad, weight, x or codes, scales, pre or codes, scales, keep, act, needs, shape of x)
//   -> (dx, dweight, dbias); needs: bits 0, 1, 2
PyObject *py_linear_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 9, [&] {
        const at::Tensor &grad = tensor(a[0], "grad"), &w = tensor(a[1], "weight");
        check_linear(grad, w);
        const int keep = (int)integer(a[6]), act = (int)integer(a[7]), needs = (int)integer(a[8]);
        const int64_t cout = w.size(0), cin = w.size(1);
        if (grad.dim() < 1 || grad.size(-1) != cout) refuse("linear: grad " + sizes_text(grad.sizes()) + " and weight " + sizes_text(w.sizes()) + " do not fit");
        const c10::cuda::CUDAGuard guard(grad.device());
        const int dtype = dtype_code(grad, "linear");
        const fcai_stream_t st = stream_of(grad);
        Rows g = rows_of(grad, cout);
        const Kept x = kept_of(a[2], a[3], keep, cin, grad);
        if (x.m.rows != g.rows) refuse("linear: grad does not fit what was kept");
        at::Tensor dx, dw, db, dp;
        if (needs & 4) db = fresh({cout}, grad);
        if (act != FCAI_ACT_NONE) {
            const Kept p = kept_of(a[4], a[5], keep, cout, grad);
            if (p.m.rows != g.rows) refuse("linear: grad does not fit what was kept");
            // dp is rounded to the type: the tensor cores read it in that type.  dx and dw then have the square root of 2 of
            // the error that exact operands would leave (0.0024 against 0.0017 relative in bf16); db is summed before it.
            const int64_t ld = (cout + 7) / 8 * 8;  // rows that the products read without a copy
            dp = fresh({g.rows, ld}, grad);
            act_backward(grad, g, cout, p, act, dp, db, ld);
            g = Rows{dp, dp.data_ptr(), ld, g.rows};
        } else if (needs & 4) {
            act_backward(grad, g, cout, Kept{}, FCAI_ACT_NONE, at::Tensor(), db, cout);
        }
        const int gpack = unaligned(g.p, g.ld) ? 1 : 0;
        if (needs & 1) {
            at::DimVector shape(grad.sizes().begin(), grad.sizes().end());
            shape.back() = cin;
            dx = fresh(shape, grad);
            const Rows wm = rows_of(w, cin);
            const int64_t bytes = fcai_linear_workspace(FCAI_LINEAR_BACKWARD_INPUT, g.rows, (int)cin, (int)cout,
                                                        gpack | (unaligned(wm.p, wm.ld) ? 2 : 0) | (unaligned(dx.data_ptr(), cin) ? 4 : 0), 0);
            const Scratch ws = scratch(bytes);
            status(fcai_linear_backward_input(g.p, g.ld, wm.p, wm.ld, dx.data_ptr(), cin, g.rows, (int)cin, (int)cout, dtype, ws.get(),
                                              bytes, st));
        }
        if (needs & 2) {
            dw = fresh({cout, cin}, grad);
            Rows m = x.m;
            if (keep >= FCAI_KEEP_INT8) {
                const int64_t ld = (cin + 7) / 8 * 8;
                at::Tensor v = fresh({x.m.rows, ld}, grad);
                status(fcai_checkpoint_load(x.codes, x.scales, v.data_ptr(), ld, x.m.rows, (int)cin, dtype, keep, st));
                const void *p = v.data_ptr();
                m = Rows{std::move(v), p, ld, x.m.rows};
            }
            const int64_t bytes = fcai_linear_workspace(FCAI_LINEAR_BACKWARD_WEIGHT, g.rows, (int)cin, (int)cout,
                                                        gpack | (unaligned(m.p, m.ld) ? 2 : 0) | (unaligned(dw.data_ptr(), cin) ? 4 : 0), 0);
            const Scratch ws = scratch(bytes);
            status(fcai_linear_backward_weight(g.p, g.ld, m.p, m.ld, dw.data_ptr(), cin, g.rows, (int)cin, (int)cout, dtype, ws.get(),
                                               bytes, st));
        }
        return wrap_all(dx, dw, db);
    });
}

at::Tensor affine(PyObject *o, const char *name, const at::Tensor &x, int64_t n) {
    if (o == Py_None) return at::Tensor();
    const at::Tensor &t = tensor(o, name);
    if (t.device() != x.device()) refuse(std::string(name) + " is on " + t.device().str() + ", expected " + x.device().str());
    if (t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat)
        refuse(std::string("layer_norm: ") + name + " must have x's dtype or fp32");
    if (t.dim() != 1 || t.size(0) != n) refuse(std::string("layer_norm: ") + name + " has shape " + sizes_text(t.sizes()) + ", expected " + sizes_text({n}));
    return t.contiguous();
}

// layer_norm_forward(x, weight, bias, eps, keep)
//   -> y, or (y, stats), or (y, stats, codes, scales)
PyObject *py_layer_norm_forward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 5, [&] {
        const at::Tensor &x = tensor(a[0], "x");
        const int dtype = dtype_code(x, "layer_norm"), keep = (int)integer(a[4]);
        const int64_t c = channels(x, "layer_norm");
        const double eps = PyFloat_AsDouble(a[3]);
        if (eps == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            refuse("layer_norm: eps must be a number");
        }
        const c10::cuda::CUDAGuard guard(x.device());
        const at::Tensor w = affine(a[1], "weight", x, c), b = affine(a[2], "bias", x, c);
        if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) refuse("layer_norm: weight and bias must have one dtype");
        const at::Tensor &any = w.defined() ? w : b;
        const int wdtype = any.defined() ? dtype_code(any, "layer_norm") : dtype;
        const Rows m = rows_of(x, c);
        at::Tensor y = fresh(x.sizes(), x), stats;
        Codes k;
        float *mean = nullptr, *rstd = nullptr;
        if (keep != FCAI_KEEP_NONE) {
            stats = fresh({2, m.rows}, x, at::kFloat);
            mean = stats.data_ptr<float>();
            rstd = mean + m.rows;
        }
        if (keep >= FCAI_KEEP_INT8) k = new_codes(x, m.rows, c);
        status(fcai_layer_norm_forward(m.p, m.ld, ptr(w), ptr(b), wdtype, y.data_ptr(), c, mean, rstd, ptr(k.codes),
                                       static_cast<float *>(ptr(k.scales)), m.rows, (int)c, (float)eps, dtype, keep, stream_of(x)));
        if (keep == FCAI_KEEP_NONE) return wrap(y);
        if (keep == FCAI_KEEP_FULL) return wrap_all(y, stats);
        return wrap_all(y, stats, k.codes, k.scales);
    });
}

// layer_norm_backward(grad, x or codes, scales, stats, weight, keep, needs, weights are fp32)
//   -> (dx, dweight, dbias)
PyObject *py_layer_norm_backward(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 8, [&] {
        const at::Tensor &grad = tensor(a[0], "grad"), &stats = tensor(a[3], "statistics");
        const int dtype = dtype_code(grad, "layer_norm"), keep = (int)integer(a[5]), needs = (int)integer(a[6]);
        const int wdtype = integer(a[7]) ? FCAI_DTYPE_F32 : dtype;
        const int64_t c = channels(grad, "layer_norm");
        const c10::cuda::CUDAGuard guard(grad.device());
        const Rows g = rows_of(grad, c);
        const Kept x = kept_of(a[1], a[2], keep, c, grad);
        if (x.m.rows != g.rows || stats.scalar_type() != at::kFloat || stats.numel() != 2 * g.rows || !stats.is_contiguous() ||
            stats.device() != grad.device())
            refuse("layer_norm: grad does not fit what was kept");
        const at::Tensor w = affine(a[4], "weight", grad, c);
        if (w.defined() && dtype_code(w, "layer_norm") != wdtype) refuse("layer_norm: weight has another dtype than in the forward call");
        const at::ScalarType wt = wdtype == FCAI_DTYPE_F32 ? at::kFloat : grad.scalar_type();
        at::Tensor dx, dw, db;
        if (needs & 1) dx = fresh(grad.sizes(), grad);
        if (needs & 2) dw = fresh({c}, grad, wt);
        if (needs & 4) db = fresh({c}, grad, wt);
        if (needs & 7) {
            const int64_t bytes = fcai_layer_norm_workspace(g.rows, (int)c);
            const Scratch ws = scratch(bytes);
            const float *mean = stats.data_ptr<float>();
            status(fcai_layer_norm_backward(g.p, g.ld, x.m.p, x.m.ld, x.codes, x.scales, mean, mean + g.rows, ptr(w), wdtype, ptr(dx), c,
                                            ptr(dw), ptr(db), g.rows, (int)c, dtype, x.keep, ws.get(), bytes, stream_of(grad)));
        }
        return wrap_all(dx, dw, db);
    });
}

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(save8), ENTRY(load8), ENTRY(activation_forward), ENTRY(activation_backward), ENTRY(linear_forward),
                         ENTRY(linear_backward), ENTRY(layer_norm_forward), ENTRY(layer_norm_backward), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layers_host", "Calls of fast_compressai.layers into libfcai_b200.so", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyMODINIT_FUNC PyInit__layers_host() { return PyModule_Create(&module); }
