// Python binding of the network operators: argument checks, output tensors, autograd nodes and
// the calls of the C entry points (include/rune_b200.h), all in C++ because a decoding step or a
// small training step spends longer in Python than on the GPU (B200 box: a 1 x 4096 norm with its
// residual 18 us through ctypes, a float32 norm step with gradients 130 us).
//
// The module is loaded by rune_b200/ops.py, which hands it the entry points' addresses (bind).
// Wrong arguments raise ValueError, failures of the library its own exceptions.

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <sstream>
#include <stdexcept>
#include <string>

#include "../../include/rune_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&rune_rms_norm) norm;
    decltype(&rune_rms_norm_backward) norm_bwd;
    decltype(&rune_rms_norm_backward_workspace) norm_bwd_ws;
    decltype(&rune_linear) linear;
    decltype(&rune_linear_workspace) linear_ws;
    decltype(&rune_linear_backward) linear_bwd;
    decltype(&rune_linear_backward_workspace) linear_bwd_ws;
    decltype(&rune_pad_rows) pad_rows;
    decltype(&rune_last_error) last_error;
} api;
PyObject* g_raise = nullptr;        // runtime.library.check's exceptions by status
int64_t g_recompute_inputs = 0;     // rune_b200.ops.RECOMPUTE_INPUTS

// A status of the library other than RUNE_OK.
struct Failure : std::runtime_error {
    int status;
    Failure(int s, const char* message) : std::runtime_error(message), status(s) {}
};
void check(int status) {
    if (status != RUNE_OK) throw Failure(status, api.last_error());
}

// Sets Python's exception for e. With the interpreter's lock.
void set_python_error(const Failure& e) {
    if (g_raise) {
        PyObject* r = PyObject_CallFunction(g_raise, "is", e.status, e.what());
        Py_XDECREF(r);
    }
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
}

// A node's backward on one of autograd's threads: its Failure goes to the caller of backward() as
// the same Python exception, which torch carries over, instead of a plain RuntimeError.
template <typename Fn>
variable_list in_backward(Fn&& fn) {
    try {
        return fn();
    } catch (const Failure& e) {
        const PyGILState_STATE lock = PyGILState_Ensure();
        set_python_error(e);
        python_error carried;
        carried.persist();
        PyGILState_Release(lock);
        throw carried;
    }
}

template <typename... Parts>
[[noreturn]] void bad(const Parts&... parts) {
    std::ostringstream s;
    (s << ... << parts);
    throw std::invalid_argument(s.str());
}

std::string name_of(ScalarType t) {
    switch (t) {
        case ScalarType::Float: return "torch.float32";
        case ScalarType::Half: return "torch.float16";
        case ScalarType::BFloat16: return "torch.bfloat16";
        case ScalarType::Float8_e4m3fn: return "torch.float8_e4m3fn";
        default: return c10::toString(t);
    }
}

int code_of(ScalarType t) {
    switch (t) {
        case ScalarType::Float: return RUNE_F32;
        case ScalarType::Half: return RUNE_F16;
        case ScalarType::BFloat16: return RUNE_BF16;
        default: return RUNE_E4M3;
    }
}

void check_tensor(const Tensor& t, const char* name, ScalarType dtype, at::IntArrayRef shape,
                  const Tensor& x) {
    if (t.scalar_type() != dtype)
        bad(name, " must be ", name_of(dtype), ", not ", name_of(t.scalar_type()), ".");
    if (t.sizes() != shape) bad(name, " must have shape ", shape, ", not ", t.sizes(), ".");
    if (t.device() != x.device()) bad(name, " must be on ", x.device(), ", not ", t.device(), ".");
}

void check_cuda(const Tensor& x) {
    if (!x.defined() || !x.is_cuda()) bad("x must be a CUDA tensor; there is no CPU path.");
}

// A tensor as rows of its last axis with unit column stride, copied only where no view has one.
struct Rows {
    Tensor t;
    int64_t n = 0, ld = 0;
    Rows() = default;
    explicit Rows(const Tensor& from) : t(from) {
        if (!from.defined()) return;
        const int64_t width = from.size(-1);
        if (!from.is_contiguous()) {
            if (t.dim() != 2) t = t.reshape({-1, width});
            if ((t.stride(1) != 1 && width > 1) || (t.stride(0) < width && t.size(0) > 1))
                t = t.contiguous();
            n = t.size(0), ld = t.stride(0);
        } else {
            n = from.numel() / width, ld = width;
        }
    }
    const void* p() const { return t.defined() ? t.data_ptr() : nullptr; }
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor empty_like_type(const Tensor& x, at::IntArrayRef shape, ScalarType t) {
    return at::empty(shape, x.options().dtype(t).requires_grad(false));
}
void* stream_of(const Tensor& x) {
    return c10::cuda::getCurrentCUDAStream(x.get_device()).stream();
}
// optional arguments of autograd nodes; an absent one has no place among the inputs' gradients
std::optional<Tensor> given(const Tensor& t) {
    return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Scratch of the bytes that `query` asks for.
template <typename Args, typename Query>
Tensor scratch(Query query, Args& args, const Tensor& x) {
    int64_t bytes = 0;
    check(query(&args, &bytes));
    Tensor ws;
    if (bytes > 0) {
        ws = empty_like_type(x, {bytes}, ScalarType::Byte);
        args.workspace = ws.data_ptr();
        args.workspace_bytes = bytes;
    }
    return ws;
}

// What follows tensors through torch's own operators does not see these: a tangent would be
// lost, and a trace would keep the empty output and no kernel that fills it.
void no_transforms(std::initializer_list<const Tensor*> inputs) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
        for (const Tensor* t : inputs)
            if (t->defined() && t->_fw_grad(/*level=*/0).defined())
                throw std::runtime_error(
                    "the operators of rune_b200.ops have no forward-mode derivative.");
    if (at::tracer::impl::is_dispatch_enabled() ||
        (TorchDispatchModeTLS::any_modes_set() &&
         (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) ||
          TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE))))
        throw std::runtime_error("the operators of rune_b200.ops cannot be traced.");
}

void first_order_only(const variable_list& grads) {
    if (at::GradMode::is_enabled())  // create_graph=True
        throw std::runtime_error("the operators of rune_b200.ops have no second derivative.");
    for (const Tensor& g : grads) no_transforms({&g});
}

// ------------------------------------------------------------------------------------ norm
struct NormOut {
    Tensor y, h, scale, rstd;
};

NormOut norm_call(const Tensor& x, const Tensor& weight, const Tensor& residual, double eps,
                  ScalarType out, bool want_rstd) {
    NormOut o;
    const Rows rx(x), rr(residual);
    rune_norm_args a{};
    a.rows = rx.n, a.width = x.size(-1);
    a.x_stride = rx.ld, a.residual_stride = rr.ld;
    a.device = x.get_device();
    a.dtype = code_of(x.scalar_type());
    a.weight_dtype = weight.defined() ? code_of(weight.scalar_type()) : a.dtype;
    a.out_dtype = code_of(out);
    a.eps = (float)eps;
    o.y = empty_like_type(x, x.sizes(), out);
    if (residual.defined()) o.h = empty_like_type(x, x.sizes(), x.scalar_type());
    if (out == ScalarType::Float8_e4m3fn)
        o.scale = empty_like_type(x, x.sizes().slice(0, x.dim() - 1), ScalarType::Float);
    if (want_rstd) o.rstd = empty_like_type(x, {rx.n}, ScalarType::Float);
    a.x = rx.p(), a.residual = rr.p(), a.weight = ptr(weight);
    a.y = ptr(o.y), a.h = ptr(o.h);
    a.scale = (float*)ptr(o.scale), a.rstd = (float*)ptr(o.rstd);
    check(api.norm(&a, stream_of(x)));
    return o;
}

struct NormFn : torch::autograd::Function<NormFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                                 const std::optional<Tensor>& residual_, double eps) {
        const Tensor residual = residual_.value_or(Tensor());
        NormOut o = norm_call(x, weight, residual, eps, x.scalar_type(), true);
        // both addends and not their rounded sum, whose error would reach dweight
        ctx->save_for_backward({x, weight, residual, o.rstd});
        ctx->set_materialize_grads(false);
        if (residual.defined()) return {o.y, o.h};
        return {o.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return in_backward([&] { return gradients(ctx, grads); });
    }
    static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
        first_order_only(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &residual = saved[2];
        const Tensor dh_in = grads.size() > 1 ? grads[1] : Tensor();
        const bool has_res = residual.defined();
        if (!grads[0].defined())  // only the residual stream has a gradient
            return {dh_in, Tensor(), has_res ? dh_in : Tensor(), Tensor()};
        const Rows rx(x), rr(residual), dy(grads[0]), dh(dh_in);
        const bool need_w = ctx->needs_input_grad(1);
        Tensor dx = empty_like_type(x, x.sizes(), x.scalar_type()), dw;
        if (need_w) dw = empty_like_type(weight, weight.sizes(), weight.scalar_type());
        rune_norm_grad_args a{};
        a.rows = rx.n, a.width = x.size(-1);
        a.x_stride = rx.ld, a.residual_stride = rr.ld, a.dy_stride = dy.ld, a.dh_stride = dh.ld;
        a.device = x.get_device();
        a.dtype = code_of(x.scalar_type()), a.weight_dtype = code_of(weight.scalar_type());
        a.x = rx.p(), a.residual = rr.p(), a.weight = ptr(weight);
        a.rstd = (const float*)ptr(saved[3]);
        a.dy = dy.p(), a.dh = dh.p();
        a.dx = ptr(dx), a.dweight = ptr(dw);
        const Tensor ws = scratch(api.norm_bwd_ws, a, x);
        check(api.norm_bwd(&a, stream_of(x)));
        return {dx, dw, has_res ? dx : Tensor(), Tensor()};
    }
};

void check_norm(const Tensor& x, Tensor& weight, const Tensor& residual) {
    check_cuda(x);
    const ScalarType t = x.scalar_type();
    if (t != ScalarType::Float && t != ScalarType::Half && t != ScalarType::BFloat16)
        bad("rms_norm takes float32, float16 or bfloat16 rows, not ", name_of(t), ".");
    if (x.dim() == 0 || x.size(-1) == 0)
        bad("x needs at least one axis, and its last one cannot be empty.");
    if (weight.defined()) {
        check_tensor(weight, "weight", weight.scalar_type() == t ? t : ScalarType::Float,
                     {x.size(-1)}, x);
        weight = weight.contiguous();
    }
    if (residual.defined()) check_tensor(residual, "residual", t, x.sizes(), x);
}

// ---------------------------------------------------------------------------------- linear
// A copy of the rows of t that start on 16 bytes each: a view of a padded buffer.
Tensor padded(const Tensor& t) {
    const Rows r(t);
    const int64_t width = t.size(-1), eb = t.element_size();
    const int64_t line = (width * eb + 15) / 16 * 16;
    Tensor buffer = empty_like_type(t, {r.n, line / eb}, t.scalar_type());
    check(api.pad_rows(t.get_device(), r.n, width * eb, r.ld * eb, r.p(), line, ptr(buffer),
                       stream_of(t)));
    return buffer.narrow(1, 0, width);
}

// t, or its padded copy where the products could not read it in place (for both passes at once)
Tensor in_place(const Tensor& t) {
    if (t.dim() != 2 || t.stride(1) != 1 || t.size(0) < 2) return t;
    const int64_t eb = t.element_size();
    const bool ready = t.stride(0) * eb % 16 == 0 && t.stride(0) >= t.size(1) &&
                       reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    return ready ? t : padded(t);
}

struct LinearOut {
    Tensor y, z;
};

LinearOut linear_call(const Tensor& x, const Tensor& weight, const Tensor& bias,
                      const Tensor& residual, const Tensor& x_scale, const Tensor& w_scale,
                      int64_t act, bool gated, ScalarType out, bool want_z) {
    LinearOut o;
    const Rows rx(x), rw(weight), rr(residual);
    const int64_t n_all = weight.size(0);
    rune_linear_args a{};
    a.rows = rx.n, a.inputs = x.size(-1), a.outputs = gated ? n_all / 2 : n_all;
    a.x_stride = rx.ld, a.weight_stride = rw.ld, a.residual_stride = rr.ld;
    a.device = x.get_device();
    a.dtype = code_of(x.scalar_type()), a.out_dtype = code_of(out);
    a.activation = (int32_t)act, a.gated = gated;
    c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = a.outputs;
    o.y = empty_like_type(x, shape, out);
    if (want_z)
        o.z = empty_like_type(x, {rx.n, gated ? 2 : 1, (a.outputs + 3) / 4 * 4}, ScalarType::Float);
    a.x = rx.p(), a.weight = rw.p(), a.bias = ptr(bias), a.residual = rr.p();
    a.x_scale = (const float*)ptr(x_scale), a.weight_scale = (const float*)ptr(w_scale);
    a.y = ptr(o.y), a.saved = (float*)ptr(o.z);
    int status = api.linear(&a, stream_of(x));
    if (status == RUNE_ERR_RETRY) {  // this call needs scratch
        const Tensor ws = scratch(api.linear_ws, a, x);
        status = api.linear(&a, stream_of(x));
    }
    check(status);
    return o;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& weight_,
                          const std::optional<Tensor>& bias_,
                          const std::optional<Tensor>& residual, int64_t act, bool gated) {
        const Tensor bias = bias_.value_or(Tensor());
        const bool again = wants_grad(x_) || wants_grad(weight_) || wants_grad(bias);
        const bool save = act != RUNE_ACT_NONE && x_.size(-1) > g_recompute_inputs && again;
        const Tensor x = again ? in_place(x_) : x_, weight = again ? in_place(weight_) : weight_;
        LinearOut o = linear_call(x, weight, bias, residual.value_or(Tensor()), Tensor(), Tensor(),
                                  act, gated, x.scalar_type(), save);
        ctx->save_for_backward({x, weight, bias, o.z});
        ctx->saved_data["act"] = act;
        ctx->saved_data["gated"] = gated;
        ctx->saved_data["residual"] = residual.has_value();
        return o.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return in_backward([&] { return gradients(ctx, grads); });
    }
    static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
        first_order_only(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2];
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        const bool need_b = bias.defined() && ctx->needs_input_grad(2);
        Tensor dx, dw, db;
        if (need_x || need_w || need_b) {
            const Rows rx(x), rw(weight), dy(grads[0]);
            rune_linear_grad_args a{};
            a.rows = rx.n, a.inputs = x.size(-1), a.outputs = grads[0].size(-1);
            a.x_stride = rx.ld, a.weight_stride = rw.ld, a.dy_stride = dy.ld;
            a.device = x.get_device();
            a.dtype = code_of(x.scalar_type());
            a.activation = (int32_t)ctx->saved_data["act"].toInt();
            a.gated = ctx->saved_data["gated"].toBool();
            if (need_x) dx = empty_like_type(x, x.sizes(), x.scalar_type());
            if (need_w) dw = empty_like_type(weight, weight.sizes(), weight.scalar_type());
            if (need_b) db = empty_like_type(bias, bias.sizes(), bias.scalar_type());
            a.x = rx.p(), a.weight = rw.p(), a.bias = ptr(bias), a.dy = dy.p();
            a.saved = (const float*)ptr(saved[3]);
            a.dx = ptr(dx), a.dweight = ptr(dw), a.dbias = ptr(db);
            const Tensor ws = scratch(api.linear_bwd_ws, a, x);
            check(api.linear_bwd(&a, stream_of(x)));
        }
        const bool residual = ctx->saved_data["residual"].toBool();
        return {dx, dw, db, residual ? grads[0] : Tensor(), Tensor(), Tensor()};
    }
};

Tensor layer(const Tensor& x, const Tensor& weight, Tensor bias, const Tensor& residual,
             Tensor x_scale, Tensor w_scale, int64_t act, bool gated, int out_code) {
    no_transforms({&x, &weight, &bias, &residual, &x_scale, &w_scale});
    check_cuda(x);
    const ScalarType t = x.scalar_type();
    const bool fp8 = t == ScalarType::Float8_e4m3fn;
    if (!fp8 && t != ScalarType::Half && t != ScalarType::BFloat16)
        bad("x must be float16, bfloat16 or float8_e4m3fn, not ", name_of(t), ".");
    if (!weight.defined() || x.dim() == 0 || x.size(-1) == 0 || weight.dim() != 2 ||
        weight.size(0) == 0)
        bad("x needs a last axis and weight two axes, none of them empty.");
    const int64_t n_all = weight.size(0), outputs = gated ? n_all / 2 : n_all;
    if (gated && n_all % 2)
        bad("weight of a gated layer has the gate's rows, then as many for the other factor; ",
            n_all, " rows are odd.");
    check_tensor(weight, "weight", t, {n_all, x.size(-1)}, x);
    ScalarType out = t;
    if (fp8) {
        out = out_code == RUNE_F16 ? ScalarType::Half : ScalarType::BFloat16;
        if (out_code == RUNE_F32 || out_code == RUNE_E4M3)
            bad("out_dtype must be float16 or bfloat16.");
        if (!x_scale.defined() || !w_scale.defined())
            bad("float8_e4m3fn operands need x_scale and weight_scale.");
        check_tensor(x_scale, "x_scale", ScalarType::Float, x.sizes().slice(0, x.dim() - 1), x);
        check_tensor(w_scale, "weight_scale", ScalarType::Float, {n_all}, x);
        x_scale = x_scale.contiguous(), w_scale = w_scale.contiguous();
    } else {
        if (out_code >= 0 && out_code != code_of(t))
            bad("out_dtype of ", name_of(t), " operands is ", name_of(t), ".");
        if (x_scale.defined() || w_scale.defined())
            bad("x_scale and weight_scale go with float8_e4m3fn operands.");
    }
    if (bias.defined()) {
        check_tensor(bias, "bias", out, {n_all}, x);
        bias = bias.contiguous();
    }
    if (residual.defined()) {
        c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = outputs;
        check_tensor(residual, "residual", out, shape, x);
    }
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() ||
                                       wants_grad(bias) || wants_grad(residual) ||
                                       wants_grad(x_scale) || wants_grad(w_scale))) {
        if (fp8)
            bad("float8_e4m3fn operands have no gradient; call under torch.no_grad().");
        return LinearFn::apply(x, weight, given(bias), given(residual), act, gated);
    }
    return linear_call(x, weight, bias, residual, x_scale, w_scale, act, gated, out, false).y;
}

// ---------------------------------------------------------------------------------- Python
Tensor tensor_arg(PyObject* o, const char* name) {
    if (o == Py_None) return Tensor();
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s must be a torch.Tensor, not %s", name,
                     Py_TYPE(o)->tp_name);
        throw 0;
    }
    return THPVariable_Unpack(o);
}

// fn() with its exceptions turned into Python's
template <typename Fn>
PyObject* guarded(Fn&& fn) {
    try {
        return fn();
    } catch (const Failure& e) {
        set_python_error(e);
    } catch (python_error& e) {  // raised in Python, by a hook on what a node saves
        e.restore();
    } catch (const std::invalid_argument& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (int) {  // a Python error is set
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown failure");
    }
    return nullptr;
}

PyObject* pack(const Tensor& a, const Tensor& b, const Tensor& c) {
    const int n = 1 + b.defined() + c.defined();
    PyObject* t = PyTuple_New(n);
    if (!t) throw 0;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
    if (b.defined()) PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
    if (c.defined()) PyTuple_SET_ITEM(t, n - 1, THPVariable_Wrap(c));
    return t;
}

bool count_is(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
    return false;
}

// rms_norm(x, weight, residual, eps): y, or (y, h)
PyObject* py_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!count_is(n, 4)) return nullptr;
    return guarded([&] {
        const Tensor x = tensor_arg(args[0], "x"), res = tensor_arg(args[2], "residual");
        Tensor w = tensor_arg(args[1], "weight");
        const double eps = PyFloat_AsDouble(args[3]);
        if (PyErr_Occurred()) throw 0;
        no_transforms({&x, &w, &res});
        if (!w.defined()) bad("rms_norm needs a weight.");
        check_norm(x, w, res);
        if (at::GradMode::is_enabled() &&
            (x.requires_grad() || w.requires_grad() || wants_grad(res))) {
            const variable_list got = NormFn::apply(x, w, given(res), eps);
            return res.defined() ? pack(got[0], got[1], Tensor()) : THPVariable_Wrap(got[0]);
        }
        const NormOut o = norm_call(x, w, res, eps, x.scalar_type(), false);
        return res.defined() ? pack(o.y, o.h, Tensor()) : THPVariable_Wrap(o.y);
    });
}

// to_fp8(x, weight or None, residual, eps): (q, scale), or (q, scale, h)
PyObject* py_to_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!count_is(n, 4)) return nullptr;
    return guarded([&] {
        const Tensor x = tensor_arg(args[0], "x"), res = tensor_arg(args[2], "residual");
        Tensor w = tensor_arg(args[1], "weight");
        const double eps = PyFloat_AsDouble(args[3]);
        if (PyErr_Occurred()) throw 0;
        no_transforms({&x, &w, &res});
        check_norm(x, w, res);
        if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(w) || wants_grad(res)))
            bad("8-bit outputs have no gradient; call under torch.no_grad().");
        const NormOut o = norm_call(x, w, res, eps, ScalarType::Float8_e4m3fn, false);
        return pack(o.y, o.scale, o.h);
    });
}

// padded(t): a copy of its rows, padded to 16 bytes each
PyObject* py_padded(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!count_is(n, 1)) return nullptr;
    return guarded([&] {
        const Tensor t = tensor_arg(args[0], "t");
        no_transforms({&t});
        if (!t.defined() || !t.is_cuda()) bad("t must be a CUDA tensor; there is no CPU path.");
        if (t.dim() != 2 || t.size(1) == 0) bad("t needs two axes, the last one not empty.");
        if (at::GradMode::is_enabled() && t.requires_grad())
            bad("a padded copy has no gradient; call under torch.no_grad().");
        return THPVariable_Wrap(padded(t));
    });
}

// layer(x, weight, bias, residual, x_scale, weight_scale, activation, gated, out code): y
PyObject* py_layer(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (!count_is(n, 9)) return nullptr;
    return guarded([&] {
        const long act = PyLong_AsLong(args[6]), gated = PyLong_AsLong(args[7]);
        const long out = PyLong_AsLong(args[8]);
        if (PyErr_Occurred()) throw 0;
        return THPVariable_Wrap(layer(tensor_arg(args[0], "x"), tensor_arg(args[1], "weight"),
                                      tensor_arg(args[2], "bias"),
                                      tensor_arg(args[3], "residual"),
                                      tensor_arg(args[4], "x_scale"),
                                      tensor_arg(args[5], "weight_scale"), act, gated != 0,
                                      (int)out));
    });
}

// bind(addresses of the entry points in Api's order, raise(status, message), recompute inputs)
PyObject* py_bind(PyObject*, PyObject* args) {
    PyObject *list, *raise;
    long long inputs;
    if (!PyArg_ParseTuple(args, "O!OL", &PyTuple_Type, &list, &raise, &inputs)) return nullptr;
    constexpr Py_ssize_t kEntries = sizeof(Api) / sizeof(void*);
    if (PyTuple_GET_SIZE(list) != kEntries) {
        PyErr_SetString(PyExc_ValueError, "wrong number of entry points");
        return nullptr;
    }
    void* entry[kEntries];
    for (Py_ssize_t i = 0; i < kEntries; ++i) {
        entry[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(list, i));
        if (!entry[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
            return nullptr;
        }
    }
    static_assert(sizeof(api) == sizeof(entry), "entry points only");
    memcpy(static_cast<void*>(&api), entry, sizeof(api));
    Py_INCREF(raise);
    Py_XSETREF(g_raise, raise);
    g_recompute_inputs = inputs;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, "Take the library's entry points."},
    {"rms_norm", reinterpret_cast<PyCFunction>(py_rms_norm), METH_FASTCALL, nullptr},
    {"to_fp8", reinterpret_cast<PyCFunction>(py_to_fp8), METH_FASTCALL, nullptr},
    {"padded", reinterpret_cast<PyCFunction>(py_padded), METH_FASTCALL, nullptr},
    {"layer", reinterpret_cast<PyCFunction>(py_layer), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&module); }
