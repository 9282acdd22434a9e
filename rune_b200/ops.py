"""Network operators in mixed precision, with gradients: normalisation, linear and gated layers.

The layers of the Möbius networks (rune/mobius/layers.py:26-67) as differentiable operators on
CUDA tensors, for training, distilling or serving networks beside the engine's float32 inference:

* ``rms_norm`` / ``rms_norm_fp8``: root-mean-square norm with the residual's addition; the
  second leaves its rows in 8 bits (e4m3) with a scale per row.
* ``linear``: ``act(x W^T + b) + residual`` in one kernel; 16-bit operands, or e4m3 with scales.
* ``gated_linear``: ``act(x Wg^T + bg) * (x Wu^T + bu)`` in one kernel.
* ``quantize_fp8``: rows to e4m3 with a scale per row (weights once, activations per call).

Every function works on the last axis of its input, takes row-strided views, runs on the current
stream of the tensors' device without synchronising it, and returns new tensors. Wrong types,
shapes or devices raise ``ValueError``; failures of the GPU raise ``RuneError``. Sums and
statistics are float32; results are rounded once. Equal inputs give equal bits.
"""

from __future__ import annotations

from ctypes import byref, c_int64

import torch

from .runtime import library as L

__all__ = ["gated_linear", "linear", "quantize_fp8", "rms_norm", "rms_norm_fp8"]

_CODES = {torch.float32: L.RUNE_F32, torch.float16: L.RUNE_F16, torch.bfloat16: L.RUNE_BF16,
          torch.float8_e4m3fn: L.RUNE_E4M3}
_ACTS = {None: L.RUNE_ACT_NONE, **L.RUNE_ACT}

# Largest input width at which the backward pass of an activated layer recomputes z = x W^T + b
# instead of reading a float32 copy that the forward saved. Per value of z the copy costs 8 bytes
# of traffic, the product 2 * inputs operations.
RECOMPUTE_INPUTS = 512


def _stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


def _activation(name):
    try:
        return _ACTS[name]
    except (KeyError, TypeError):
        key = str(name).strip().lower()
        if key in _ACTS:
            return _ACTS[key]
        raise ValueError(f"Unsupported activation {name!r}; choose one of "
                         f"{', '.join(sorted(L.RUNE_ACT))} or None.") from None


def _rows(t, name):
    """(`t`, rows, stride): `t` as rows of its last axis with unit column stride, copied only
    where no view has one."""
    shape = t.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{name} needs at least one axis, and its last one cannot be empty.")
    width = shape[-1]
    if t.is_contiguous():
        return t, t.numel() // width, width
    if len(shape) != 2:
        t = t.reshape(-1, width)
    step, unit = t.stride()
    if (unit != 1 and width > 1) or (step < width and t.shape[0] > 1):
        t = t.contiguous()
        step = width
    return t, t.shape[0], step


def _check(t, name, dtype, shape, x):
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}.")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}.")
    if t.get_device() != x.get_device():
        raise ValueError(f"{name} must be on {x.device}, not {t.device}.")


def _cuda(t, name):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor; there is no CPU path.")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _workspace(lib, query, args, like):
    """Scratch of the bytes that `query` asks for (None where it needs none)."""
    need = c_int64(0)
    L.check(lib, query(args, byref(need)))
    n = need.value
    return (like.new_empty(n, dtype=torch.uint8), n) if n else (None, 0)


def _first_order_only():
    if torch.is_grad_enabled():  # create_graph=True
        raise RuntimeError("the operators of rune_b200.ops have no second derivative.")


# ------------------------------------------------------------------------------------ norm
def _norm_call(x, weight, residual, eps, out_dtype, want_rstd):
    """(y, h, scale, rstd) of the rows of x; h is None without a residual."""
    lib = L.load_library()
    shape, dtype, index = x.shape, x.dtype, x.get_device()
    x, rows, ld = _rows(x, "x")
    h = scale = rstd = None
    res_ptr = ld_res = h_ptr = 0
    if residual is not None:
        res, _, ld_res = _rows(residual, "residual")
        res_ptr = res.data_ptr()
        h = x.new_empty(shape)
        h_ptr = h.data_ptr()
    y = x.new_empty(shape, dtype=out_dtype)
    if out_dtype is torch.float8_e4m3fn:
        scale = x.new_empty(shape[:-1], dtype=torch.float32)
    if want_rstd:
        rstd = x.new_empty(rows, dtype=torch.float32)
    code = _CODES[dtype]
    status = lib.rune_rms_norm(L.NORM_ARGS.pack(
        rows, shape[-1], ld, ld_res, index, code,
        code if weight is None else _CODES[weight.dtype], _CODES[out_dtype], eps, 0,
        x.data_ptr(), res_ptr, _ptr(weight), y.data_ptr(), h_ptr, _ptr(scale), _ptr(rstd)),
        _stream(index))
    if status:
        L.check(lib, status)
    return y, h, scale, rstd


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, _, rstd = _norm_call(x, weight, residual, eps, x.dtype, True)
        # both addends and not their rounded sum, whose error would reach dweight
        ctx.save_for_backward(x, residual, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        _first_order_only()
        x, residual, weight, rstd = ctx.saved_tensors
        _, need_w, with_res, _ = ctx.needs_input_grad
        if dy is None:  # only the residual stream has a gradient
            return dh, None, dh if with_res else None, None
        lib = L.load_library()
        width, index = x.shape[-1], x.get_device()
        dx = x.new_empty(x.shape)
        x, rows, ld = _rows(x, "x")
        ld_res = 0
        if residual is not None:
            residual, _, ld_res = _rows(residual, "residual")
        dy, _, ld_dy = _rows(dy, "dy")
        ld_dh = 0
        if dh is not None:
            dh, _, ld_dh = _rows(dh, "dh")
        dw = torch.empty_like(weight) if need_w else None

        def args(ws, size):
            return L.NORM_GRAD_ARGS.pack(
                rows, width, ld, ld_res, ld_dy, ld_dh, index, _CODES[x.dtype],
                _CODES[weight.dtype], 0, x.data_ptr(), _ptr(residual), weight.data_ptr(),
                rstd.data_ptr(), dy.data_ptr(), _ptr(dh), dx.data_ptr(), _ptr(dw), _ptr(ws), size)

        ws = _workspace(lib, lib.rune_rms_norm_backward_workspace, args(None, 0), x)
        L.check(lib, lib.rune_rms_norm_backward(args(*ws), _stream(index)))
        return dx, dw, dx if with_res else None, None


def _norm_inputs(x, weight, residual):
    _cuda(x, "x")
    dtype = x.dtype
    if dtype not in _CODES or dtype is torch.float8_e4m3fn:
        raise ValueError(f"rms_norm takes float32, float16 or bfloat16 rows, not {dtype}.")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError("x needs at least one axis, and its last one cannot be empty.")
    if weight is not None:
        _check(weight, "weight", dtype if weight.dtype is dtype else torch.float32, shape[-1:],
               x)
        weight = weight.contiguous()
    if residual is not None:
        _check(residual, "residual", dtype, shape, x)
    return weight


def rms_norm(x, weight, residual=None, eps=1.0e-8):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last axis, ``h = x + residual``.

    x and residual: float32, float16 or bfloat16 of one shape; weight [width]: their type or
    float32. Returns y, and with a residual ``(y, h)``: h is the residual stream for what
    follows. Differentiable in x, weight and residual.
    """
    weight = _norm_inputs(x, weight, residual)
    if (x.requires_grad or weight.requires_grad
            or (residual is not None and residual.requires_grad)) and torch.is_grad_enabled():
        return _RMSNorm.apply(x, weight, residual, float(eps))
    y, h, _, _ = _norm_call(x, weight, residual, eps, x.dtype, False)
    return y if residual is None else (y, h)


def _to_fp8(x, weight, residual, eps):
    for t in (x, weight, residual):
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError("8-bit outputs have no gradient; call under torch.no_grad().")
    weight = _norm_inputs(x, weight, residual)
    q, h, scale, _ = _norm_call(x, weight, residual, eps, torch.float8_e4m3fn, False)
    return (q, scale) if residual is None else (q, scale, h)


def rms_norm_fp8(x, weight, residual=None, eps=1.0e-8):
    """``rms_norm`` with its rows in 8 bits: ``(q, scale)``, and with a residual
    ``(q, scale, h)``. q (float8_e4m3fn) stands for ``q * scale``; a row's scale maps its largest
    magnitude to 448 and is 1 for a row of zeros. Not differentiable.
    """
    return _to_fp8(x, weight, residual, eps)


def quantize_fp8(x):
    """Rows of x as float8_e4m3fn with a scale per row, ``(q, scale)``: x is about ``q * scale``.

    For the weights of an 8-bit ``linear`` or ``gated_linear`` (once) and for activations that no
    ``rms_norm_fp8`` precedes. Not differentiable.
    """
    return _to_fp8(x, None, None, 0.0)


# ---------------------------------------------------------------------------------- linear
def _linear_call(x, weight, bias, residual, x_scale, w_scale, act, gated, out_dtype, want_z):
    """(y, z) of the rows of x; z is the float32 pre-activation where it is asked for."""
    lib = L.load_library()
    shape, index = x.shape, x.get_device()
    inputs, n_all = shape[-1], weight.shape[0]
    outputs = n_all // 2 if gated else n_all
    x, rows, ld = _rows(x, "x")
    w, _, ld_w = _rows(weight, "weight")
    res_ptr = ld_res = 0
    if residual is not None:
        residual, _, ld_res = _rows(residual, "residual")
        res_ptr = residual.data_ptr()
    y = x.new_empty((*shape[:-1], outputs), dtype=out_dtype)
    z = x.new_empty((rows, n_all), dtype=torch.float32) if want_z else None
    pack, stream = L.LINEAR_ARGS.pack, _stream(index)
    head = (rows, inputs, outputs, ld, ld_w, ld_res, index, _CODES[x.dtype], _CODES[out_dtype],
            act, gated, 0, x.data_ptr(), w.data_ptr(), _ptr(bias), res_ptr, _ptr(x_scale),
            _ptr(w_scale), y.data_ptr(), _ptr(z))
    args = pack(*head, 0, 0)
    status = lib.rune_linear(args, stream)
    if status == L.RUNE_ERR_RETRY:  # this call needs scratch
        ws, size = _workspace(lib, lib.rune_linear_workspace, args, x)
        status = lib.rune_linear(pack(*head, ws.data_ptr(), size), stream)
    if status:
        L.check(lib, status)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, gated):
        needs = ctx.needs_input_grad
        save = act != L.RUNE_ACT_NONE and x.shape[-1] > RECOMPUTE_INPUTS and any(needs[:3])
        y, z = _linear_call(x, weight, bias, residual, None, None, act, gated, x.dtype, save)
        ctx.save_for_backward(x, weight, bias, z)
        ctx.act, ctx.gated = act, gated
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_order_only()
        x, weight, bias, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            lib = L.load_library()
            index, outputs = x.get_device(), dy.shape[-1]
            if need_x:
                dx = x.new_empty(x.shape)
            if need_w:
                dw = weight.new_empty(weight.shape)
            if need_b:
                db = bias.new_empty(bias.shape)
            x, rows, ld = _rows(x, "x")
            w, _, ld_w = _rows(weight, "weight")
            g, _, ld_g = _rows(dy, "dy")

            def args(ws, size):
                return L.LINEAR_GRAD_ARGS.pack(
                    rows, x.shape[-1], outputs, ld, ld_w, ld_g, index, _CODES[x.dtype], ctx.act,
                    ctx.gated, x.data_ptr(), w.data_ptr(), _ptr(bias), g.data_ptr(), _ptr(z),
                    _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), size)

            ws = _workspace(lib, lib.rune_linear_backward_workspace, args(None, 0), x)
            L.check(lib, lib.rune_linear_backward(args(*ws), _stream(index)))
        return dx, dw, db, dy if need_r else None, None, None


def _layer(x, weight, bias, residual, x_scale, w_scale, act, gated, out_dtype):
    _cuda(x, "x")
    dtype, shape = x.dtype, x.shape
    fp8 = dtype is torch.float8_e4m3fn
    if not fp8 and dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"x must be float16, bfloat16 or float8_e4m3fn, not {dtype}.")
    if not shape or shape[-1] == 0 or weight.dim() != 2 or weight.shape[0] == 0:
        raise ValueError("x needs a last axis and weight two axes, none of them empty.")
    n_all = weight.shape[0]
    if gated and n_all % 2:
        raise ValueError("weight of a gated layer has the gate's rows, then as many for the "
                         f"other factor; {n_all} rows are odd.")
    _check(weight, "weight", dtype, (n_all, shape[-1]), x)
    outputs = n_all // 2 if gated else n_all
    if fp8:
        out = torch.bfloat16 if out_dtype is None else out_dtype
        if out is not torch.bfloat16 and out is not torch.float16:
            raise ValueError(f"out_dtype must be float16 or bfloat16, not {out}.")
        if x_scale is None or w_scale is None:
            raise ValueError("float8_e4m3fn operands need x_scale and weight_scale.")
        _check(x_scale, "x_scale", torch.float32, shape[:-1], x)
        _check(w_scale, "weight_scale", torch.float32, (n_all,), x)
        x_scale, w_scale = x_scale.contiguous(), w_scale.contiguous()
    else:
        out = dtype
        if out_dtype is not None and out_dtype is not dtype:
            raise ValueError(f"out_dtype of {dtype} operands is {dtype}.")
        if x_scale is not None or w_scale is not None:
            raise ValueError("x_scale and weight_scale go with float8_e4m3fn operands.")
    if bias is not None:
        _check(bias, "bias", out, (n_all,), x)
        bias = bias.contiguous()
    if residual is not None:
        _check(residual, "residual", out, (*shape[:-1], outputs), x)
    if (x.requires_grad or weight.requires_grad
            or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad)) and torch.is_grad_enabled():
        if fp8:
            raise ValueError("float8_e4m3fn operands have no gradient; call under "
                             "torch.no_grad().")
        return _Linear.apply(x, weight, bias, residual, act, int(gated))
    return _linear_call(x, weight, bias, residual, x_scale, w_scale, act, int(gated), out,
                        False)[0]


def linear(x, weight, bias=None, activation=None, residual=None, *, x_scale=None,
           weight_scale=None, out_dtype=None):
    """``act(x weight^T + bias) + residual`` over the last axis.

    x [..., inputs] and weight [outputs, inputs]: float16 or bfloat16, differentiable with bias
    [outputs] and residual [..., outputs] of the same type. Or both float8_e4m3fn with float32
    x_scale [...] and weight_scale [outputs] (forward only); out_dtype (bfloat16, or float16) is
    then the type of bias, residual and result. activation: "tanh", "silu", "gelu" (erf) or None.
    """
    return _layer(x, weight, bias, residual, x_scale, weight_scale, _activation(activation),
                  False, out_dtype)


def gated_linear(x, weight, bias=None, activation="silu", *, x_scale=None, weight_scale=None,
                 out_dtype=None):
    """``act(x Wg^T + bg) * (x Wu^T + bu)`` over the last axis, weight = [Wg; Wu].

    weight [2 * outputs, inputs] and bias [2 * outputs] hold the gate's rows first. Types,
    gradients and e4m3 operands as in ``linear``.
    """
    act = _activation(activation)
    if act == L.RUNE_ACT_NONE:
        raise ValueError("gated_linear needs an activation.")
    return _layer(x, weight, bias, None, x_scale, weight_scale, act, True, out_dtype)
