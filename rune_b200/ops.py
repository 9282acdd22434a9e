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
from torch.autograd.function import once_differentiable

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
    """`t` as [rows, width] with unit column stride (copied only where no view has one)."""
    shape = t.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{name} needs at least one axis, and its last one cannot be empty.")
    if len(shape) != 2:
        t = t.reshape(-1, shape[-1])
    step, unit = t.stride()
    if (unit != 1 and shape[-1] > 1) or (step < shape[-1] and t.shape[0] > 1):
        t = t.contiguous()
    return t


def _check(t, name, dtype, shape, device):
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}.")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}.")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, not {t.device}.")


def _cuda(t, name):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor; there is no CPU path.")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _workspace(lib, query, args, device):
    """Scratch of the bytes that `query` asks for (None where it needs none)."""
    need = c_int64(0)
    L.check(lib, query(args, byref(need)))
    n = need.value
    return (torch.empty(n, dtype=torch.uint8, device=device), n) if n else (None, 0)


# ------------------------------------------------------------------------------------ norm
def _norm_call(x, weight, residual, eps, out_dtype, want_rstd):
    """(y, h, scale, rstd) of rows x; h is x itself without a residual."""
    lib = L.load_library()
    rows, width = x.shape
    dev = x.device
    y = torch.empty((rows, width), dtype=out_dtype, device=dev)
    h = scale = rstd = None
    if residual is not None:
        h = torch.empty((rows, width), dtype=x.dtype, device=dev)
    if out_dtype is torch.float8_e4m3fn:
        scale = torch.empty(rows, dtype=torch.float32, device=dev)
    if want_rstd:
        rstd = torch.empty(rows, dtype=torch.float32, device=dev)
    code = _CODES[x.dtype]
    args = L.NORM_ARGS.pack(
        rows, width, x.stride(0), 0 if residual is None else residual.stride(0), dev.index, code,
        code if weight is None else _CODES[weight.dtype], _CODES[out_dtype], eps, 0,
        x.data_ptr(), _ptr(residual), _ptr(weight), y.data_ptr(), _ptr(h), _ptr(scale),
        _ptr(rstd))
    L.check(lib, lib.rune_rms_norm(args, _stream(dev.index)))
    return y, x if h is None else h, scale, rstd


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, _, rstd = _norm_call(x, weight, residual, eps, x.dtype, True)
        ctx.save_for_backward(h, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        with_res = ctx.needs_input_grad[2]
        if dy is None:  # only the residual stream has a gradient
            return dh, None, dh, None
        lib = L.load_library()
        rows, width = h.shape
        dev = h.device
        dy = _rows(dy, "dy")
        if dh is not None:
            dh = _rows(dh, "dh")
        dx = torch.empty((rows, width), dtype=h.dtype, device=dev)
        dw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None

        def args(ws, size):
            return L.NORM_GRAD_ARGS.pack(
                rows, width, h.stride(0), dy.stride(0), 0 if dh is None else dh.stride(0),
                dev.index, _CODES[h.dtype], _CODES[weight.dtype], 0, h.data_ptr(),
                weight.data_ptr(), rstd.data_ptr(), dy.data_ptr(), _ptr(dh), dx.data_ptr(),
                _ptr(dw), _ptr(ws), size)

        ws = _workspace(lib, lib.rune_rms_norm_backward_workspace, args(None, 0), dev)
        L.check(lib, lib.rune_rms_norm_backward(args(*ws), _stream(dev.index)))
        return dx, dw, dx if with_res else None, None


def _norm_inputs(x, weight, residual):
    _cuda(x, "x")
    dtype = x.dtype
    if dtype not in _CODES or dtype is torch.float8_e4m3fn:
        raise ValueError(f"rms_norm takes float32, float16 or bfloat16 rows, not {dtype}.")
    width = x.shape[-1:]
    if weight is not None:
        _check(weight, "weight", dtype if weight.dtype is dtype else torch.float32, width,
               x.device)
        weight = weight.contiguous()
    if residual is not None:
        _check(residual, "residual", dtype, x.shape, x.device)
        residual = _rows(residual, "residual")
    return _rows(x, "x"), weight, residual


def rms_norm(x, weight, residual=None, eps=1.0e-8):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last axis, ``h = x + residual``.

    x and residual: float32, float16 or bfloat16 of one shape; weight [width]: their type or
    float32. Returns y, and with a residual ``(y, h)``: h is the residual stream for what
    follows. Differentiable in x, weight and residual.
    """
    shape = x.shape
    rows, weight, res = _norm_inputs(x, weight, residual)
    if torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad
            or (residual is not None and residual.requires_grad)):
        got = _RMSNorm.apply(rows, weight, res, float(eps))
        y, h = got if residual is not None else (got, None)
    else:
        y, h, _, _ = _norm_call(rows, weight, res, float(eps), x.dtype, False)
    if residual is None:
        return y.view(shape)
    return y.view(shape), h.view(shape)


def _to_fp8(x, weight, residual, eps):
    for t in (x, weight, residual):
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError("8-bit outputs have no gradient; call under torch.no_grad().")
    shape = x.shape
    rows, weight, res = _norm_inputs(x, weight, residual)
    q, h, scale, _ = _norm_call(rows, weight, res, float(eps), torch.float8_e4m3fn, False)
    got = q.view(shape), scale.view(shape[:-1])
    return got if residual is None else (*got, h.view(shape))


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
    """(y, z) of rows x; z is the float32 pre-activation where it is asked for."""
    lib = L.load_library()
    rows, inputs = x.shape
    outputs = weight.shape[0] // 2 if gated else weight.shape[0]
    dev = x.device
    y = torch.empty((rows, outputs), dtype=out_dtype, device=dev)
    z = None
    if want_z:
        z = torch.empty((rows, weight.shape[0]), dtype=torch.float32, device=dev)

    def args(ws, size):
        return L.LINEAR_ARGS.pack(
            rows, inputs, outputs, x.stride(0), weight.stride(0),
            0 if residual is None else residual.stride(0), dev.index, _CODES[x.dtype],
            _CODES[out_dtype], act, gated, 0, x.data_ptr(), weight.data_ptr(), _ptr(bias),
            _ptr(residual), _ptr(x_scale), _ptr(w_scale), y.data_ptr(), _ptr(z), _ptr(ws), size)

    ws = _workspace(lib, lib.rune_linear_workspace, args(None, 0), dev)
    L.check(lib, lib.rune_linear(args(*ws), _stream(dev.index)))
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, gated):
        needs = ctx.needs_input_grad
        save = act != L.RUNE_ACT_NONE and x.shape[1] > RECOMPUTE_INPUTS and any(needs[:3])
        y, z = _linear_call(x, weight, bias, residual, None, None, act, gated, x.dtype, save)
        ctx.save_for_backward(x, weight, bias, z)
        ctx.act, ctx.gated = act, gated
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            lib = L.load_library()
            dev = x.device
            rows, inputs = x.shape
            g = _rows(dy, "dy")
            if need_x:
                dx = torch.empty((rows, inputs), dtype=x.dtype, device=dev)
            if need_w:
                dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev)
            if need_b:
                db = torch.empty(bias.shape, dtype=bias.dtype, device=dev)

            def args(ws, size):
                return L.LINEAR_GRAD_ARGS.pack(
                    rows, inputs, dy.shape[1], x.stride(0), weight.stride(0), g.stride(0),
                    dev.index, _CODES[x.dtype], ctx.act, ctx.gated, x.data_ptr(),
                    weight.data_ptr(), _ptr(bias), g.data_ptr(), _ptr(z), _ptr(dx), _ptr(dw),
                    _ptr(db), _ptr(ws), size)

            ws = _workspace(lib, lib.rune_linear_backward_workspace, args(None, 0), dev)
            L.check(lib, lib.rune_linear_backward(args(*ws), _stream(dev.index)))
        return dx, dw, db, dy if need_r else None, None, None


def _layer(x, weight, bias, residual, x_scale, w_scale, act, gated, out_dtype):
    _cuda(x, "x")
    dtype, dev, shape = x.dtype, x.device, x.shape
    fp8 = dtype is torch.float8_e4m3fn
    if not fp8 and dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"x must be float16, bfloat16 or float8_e4m3fn, not {dtype}.")
    if not shape or shape[-1] == 0 or weight.dim() != 2 or weight.shape[0] == 0:
        raise ValueError("x needs a last axis and weight two axes, none of them empty.")
    n_all = weight.shape[0]
    if gated and n_all % 2:
        raise ValueError("weight of a gated layer has the gate's rows, then as many for the "
                         f"other factor; {n_all} rows are odd.")
    _check(weight, "weight", dtype, (n_all, shape[-1]), dev)
    outputs = n_all // 2 if gated else n_all
    if fp8:
        out = torch.bfloat16 if out_dtype is None else out_dtype
        if out is not torch.bfloat16 and out is not torch.float16:
            raise ValueError(f"out_dtype must be float16 or bfloat16, not {out}.")
        if x_scale is None or w_scale is None:
            raise ValueError("float8_e4m3fn operands need x_scale and weight_scale.")
        _check(x_scale, "x_scale", torch.float32, shape[:-1], dev)
        _check(w_scale, "weight_scale", torch.float32, (n_all,), dev)
        x_scale, w_scale = x_scale.contiguous(), w_scale.contiguous()
    else:
        out = dtype
        if out_dtype is not None and out_dtype is not dtype:
            raise ValueError(f"out_dtype of {dtype} operands is {dtype}.")
        if x_scale is not None or w_scale is not None:
            raise ValueError("x_scale and weight_scale go with float8_e4m3fn operands.")
    if bias is not None:
        _check(bias, "bias", out, (n_all,), dev)
        bias = bias.contiguous()
    rows, wmat, res = _rows(x, "x"), _rows(weight, "weight"), None
    if residual is not None:
        _check(residual, "residual", out, (*shape[:-1], outputs), dev)
        res = _rows(residual, "residual")
    if torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad
            or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad)):
        if fp8:
            raise ValueError("float8_e4m3fn operands have no gradient; call under "
                             "torch.no_grad().")
        y = _Linear.apply(rows, wmat, bias, res, act, int(gated))
    else:
        y, _ = _linear_call(rows, wmat, bias, res, x_scale, w_scale, act, int(gated), out, False)
    return y if len(shape) == 2 else y.view(*shape[:-1], outputs)


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
