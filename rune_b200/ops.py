"""Network operators in mixed precision, with gradients: normalisation, linear and gated layers.

The layers of the Möbius networks (rune/mobius/layers.py:26-67) as differentiable operators on
CUDA tensors, for training, distilling or serving networks beside the engine's float32 inference:

* ``rms_norm`` / ``rms_norm_fp8``: root-mean-square norm with the residual's addition; the
  second leaves its rows in 8 bits (e4m3) with a scale per row.
* ``linear``: ``act(x W^T + b) + residual`` in one kernel; 16-bit operands, or e4m3 with scales.
* ``gated_linear``: ``act(x Wg^T + bg) * (x Wu^T + bu)`` in one kernel.
* ``padded``: a copy of a matrix whose rows start on 16 bytes each, for weights of odd widths.
* ``quantize_fp8``: rows to e4m3 with a scale per row (weights once, activations per call).
* ``check_waits``: whether a kernel of these gave up waiting, where no operator call follows.

Every function works on the last axis of its input, takes row-strided views, runs on the current
stream of the tensors' device without synchronising it, and returns new tensors. Wrong types,
shapes or devices raise ``ValueError``; failures of the GPU raise ``RuneError``. Gradients are
reverse-mode and of first order; forward-mode tangents, function transforms and traces are refused
(``RuntimeError``). Sums and statistics are float32. Results are rounded once, but dx and dweight of
the layers are products of a dz that is rounded to 16 bits first. Equal inputs give equal bits.
"""

from __future__ import annotations

import ctypes
from importlib.machinery import ExtensionFileLoader
from importlib.util import module_from_spec, spec_from_loader

import torch

from .runtime import library as L
from .runtime.build import BINDING

__all__ = ["check_waits", "gated_linear", "linear", "padded", "quantize_fp8", "rms_norm", "rms_norm_fp8"]

_ACTS = {None: L.RUNE_ACT_NONE, **L.RUNE_ACT}
_OUT = {None: -1, torch.float16: L.RUNE_F16, torch.bfloat16: L.RUNE_BF16}

# Largest input width at which the backward pass of an activated layer recomputes z = x W^T + b
# instead of reading a float32 copy that the forward saved. Per value of z the copy costs 8 bytes
# of traffic and its memory, the product 2 * inputs operations. B200, training step of 32768 rows
# and 1024 outputs, recomputed / saved: 512 inputs 177 / 191 us (gated 257 / 323), 1024 inputs
# 248 / 243 (424 / 432), 2048 inputs 428 / 379 (770 / 682).
RECOMPUTE_INPUTS = 1024

_BINDING = None


def _native():
    """The C++ binding (rune_b200/csrc/torch_ops.cpp), bound to the engine library."""
    global _BINDING
    if _BINDING is None:
        lib = L.load_library()
        if not BINDING.exists():
            raise ImportError(
                f"rune_b200 operator binding not found at {BINDING}; build it with "
                "`python -m rune_b200.runtime.build`. There is no other path.")
        loader = ExtensionFileLoader("rune_b200._ops", str(BINDING))
        module = module_from_spec(spec_from_loader("rune_b200._ops", loader))
        loader.exec_module(module)
        entries = (lib.rune_rms_norm, lib.rune_rms_norm_backward,
                   lib.rune_rms_norm_backward_workspace, lib.rune_linear,
                   lib.rune_linear_workspace, lib.rune_linear_backward,
                   lib.rune_linear_backward_workspace, lib.rune_pad_rows, lib.rune_last_error)
        module.bind(tuple(ctypes.cast(f, ctypes.c_void_p).value for f in entries), L.fail,
                    RECOMPUTE_INPUTS)
        _BINDING = module
    return _BINDING


def check_waits(device=None):
    """Raise ``RuneError`` if a linear kernel's bounded wait gave up on the CUDA device (default:
    the current one) since the last report; the results of that call are invalid.

    Every operator call reports it too. This is for results that no call follows and for replayed
    CUDA graphs, after a synchronisation.
    """
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    lib = L.load_library()
    L.check(lib, lib.rune_linear_check_waits(index))


def _activation(name):
    try:
        return _ACTS[name]
    except (KeyError, TypeError):
        key = str(name).strip().lower()
        if key in _ACTS:
            return _ACTS[key]
        raise ValueError(f"Unsupported activation {name!r}; choose one of "
                         f"{', '.join(sorted(L.RUNE_ACT))} or None.") from None


def _out_code(dtype):
    if dtype not in _OUT:
        raise ValueError(f"out_dtype must be float16 or bfloat16, not {dtype}.")
    return _OUT[dtype]


def rms_norm(x, weight, residual=None, eps=1.0e-8):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last axis, ``h = x + residual``.

    x and residual: float32, float16 or bfloat16 of one shape; weight [width]: their type or
    float32. Returns y, and with a residual ``(y, h)``: h is the residual stream for what
    follows. Differentiable in x, weight and residual.
    """
    return (_BINDING or _native()).rms_norm(x, weight, residual, eps)


def rms_norm_fp8(x, weight, residual=None, eps=1.0e-8):
    """``rms_norm`` with its rows in 8 bits: ``(q, scale)``, and with a residual
    ``(q, scale, h)``. q (float8_e4m3fn) stands for ``q * scale``; a row's scale maps its largest
    magnitude to 448, is 1 for a row of zeros and otherwise at least 2^-126 (float32's smallest
    normal number). Not differentiable.
    """
    if weight is None:
        raise ValueError("rms_norm_fp8 needs a weight.")
    return (_BINDING or _native()).to_fp8(x, weight, residual, eps)


def quantize_fp8(x):
    """Rows of x as float8_e4m3fn with a scale per row, ``(q, scale)``: x is about ``q * scale``.

    For the weights of an 8-bit ``linear`` or ``gated_linear`` (once) and for activations that no
    ``rms_norm_fp8`` precedes. Not differentiable.
    """
    return (_BINDING or _native()).to_fp8(x, None, None, 0.0)


def padded(t):
    """A copy of the matrix t as a view of a buffer whose rows start on 16 bytes each.

    ``linear`` and ``gated_linear`` read such operands in place; others they copy in every call,
    which with few rows of x takes longer than the product. For weights of widths that are no
    multiple of 8 (e4m3: 16), once. Not differentiable.
    """
    return (_BINDING or _native()).padded(t)


def linear(x, weight, bias=None, activation=None, residual=None, *, x_scale=None,
           weight_scale=None, out_dtype=None):
    """``act(x weight^T + bias) + residual`` over the last axis.

    x [..., inputs] and weight [outputs, inputs]: float16 or bfloat16, differentiable with bias
    [outputs] and residual [..., outputs] of the same type. Or both float8_e4m3fn with float32
    x_scale [...] and weight_scale [outputs] (forward only); out_dtype (bfloat16, or float16) is
    then the type of bias, residual and result. activation: "tanh", "silu", "gelu" (erf) or None.
    """
    return (_BINDING or _native()).layer(x, weight, bias, residual, x_scale, weight_scale,
                                         _activation(activation), 0, _out_code(out_dtype))


def gated_linear(x, weight, bias=None, activation="silu", *, x_scale=None, weight_scale=None,
                 out_dtype=None):
    """``act(x Wg^T + bg) * (x Wu^T + bu)`` over the last axis, weight = [Wg; Wu].

    weight [2 * outputs, inputs] and bias [2 * outputs] hold the gate's rows first. Types,
    gradients and e4m3 operands as in ``linear``.
    """
    act = _activation(activation)
    if act == L.RUNE_ACT_NONE:
        raise ValueError("gated_linear needs an activation.")
    return (_BINDING or _native()).layer(x, weight, bias, None, x_scale, weight_scale, act, 1,
                                         _out_code(out_dtype))
