"""Network operators in mixed precision, with gradients: normalisation, linear and gated layers,
the same by group of rows, and the orthogonalised update of an optimiser.

The layers of the Möbius networks (rune/mobius/layers.py:26-67) as differentiable operators on
CUDA tensors, for training, distilling or serving networks beside the engine's float32 inference:

* ``rms_norm`` / ``rms_norm_fp8``: root-mean-square norm with the residual's addition; the
  second leaves its rows in 8 bits (e4m3) with a scale per row.
* ``linear``: ``act(x W^T + b) + residual`` in one kernel; 16-bit operands, or e4m3 with scales.
* ``gated_linear``: ``act(x Wg^T + bg) * (x Wu^T + bu)`` in one kernel.
* ``padded``: a copy of a matrix whose rows start on 16 bytes each, for weights of odd widths.
* ``quantize_fp8``: rows to e4m3 with a scale per row (weights once, activations per call).
* ``route``, ``row_groups``, ``to_groups``, ``from_groups``: rows to the groups (experts, elements)
  whose weights they take, sorted by group, and back.
* ``grouped_linear``, ``grouped_gated_linear``: the layers with each group's own weights.
* ``orthogonalize``: a stack of updates, orthogonalised by Newton-Schulz products.
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
from collections import namedtuple
from importlib.machinery import ExtensionFileLoader
from importlib.util import module_from_spec, spec_from_loader

import torch

from .runtime import library as L
from .runtime.build import BINDING

__all__ = ["RowGroups", "check_waits", "from_groups", "gated_linear", "grouped_gated_linear",
           "grouped_linear", "linear", "orthogonalize", "padded", "quantize_fp8", "rms_norm",
           "rms_norm_fp8", "route", "row_groups", "to_groups"]

_ACTS = {None: L.RUNE_ACT_NONE, **L.RUNE_ACT}
_OUT = {None: -1, torch.float16: L.RUNE_F16, torch.bfloat16: L.RUNE_BF16}

# Largest input width at which the backward pass of an activated layer recomputes z = x W^T + b
# instead of reading a float32 copy that the forward saved. Per value of z the copy costs 8 bytes
# of traffic and its memory, the product 2 * inputs operations. B200, training step of 32768 rows
# and 1024 outputs, recomputed / saved: 512 inputs 177 / 191 us (gated 257 / 323), 1024 inputs
# 248 / 243 (424 / 432), 2048 inputs 428 / 379 (770 / 682).
RECOMPUTE_INPUTS = 1024

# A grouped layer also saves z where its groups are small: where ``rows * ROWS_TO_INPUTS`` is less than
# ``groups * inputs``, reading all groups' weights once more takes longer than z, written and read.
# B200, training step of gated layers, recomputed / saved, us, for groups of like sizes (and of sizes as
# the softmax of normal numbers):
#   61 groups of 1024 -> 2 x 1408    2000 rows  298 /  244 (299 / 272)   8001 rows  377 /  329 (373 / 341)
#                                   16000 rows  543 /  462 (532 / 522)  32000 rows  761 /  767 (821 / 832)
#                                   64000 rows 1475 / 1584 (1424 / 1516)
#   32 groups of 512 -> 2 x 512      4096 rows   92 /   88 (74 / 75)     8192 rows   81 /   82 (84 / 88)
#                                   16384 rows  111 /  123 (115 / 131)
ROWS_TO_INPUTS = 2

# Coefficients a, b, c of the quintic a x + b x^3 + c x^5 that ``orthogonalize`` iterates: steep at
# zero, so that five steps bring singular values from 0.01 and up to between 0.7 and 1.2.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)

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
                   lib.rune_linear_backward_workspace, lib.rune_pad_rows, lib.rune_route,
                   lib.rune_route_backward, lib.rune_row_groups, lib.rune_row_groups_workspace,
                   lib.rune_to_groups, lib.rune_from_groups, lib.rune_from_groups_backward,
                   lib.rune_grouped_linear, lib.rune_grouped_linear_workspace,
                   lib.rune_grouped_linear_backward, lib.rune_grouped_linear_backward_workspace,
                   lib.rune_orthogonalize, lib.rune_orthogonalize_workspace,
                   lib.rune_last_error)
        module.bind(tuple(ctypes.cast(f, ctypes.c_void_p).value for f in entries), L.fail,
                    RECOMPUTE_INPUTS, ROWS_TO_INPUTS)
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


RowGroups = namedtuple("RowGroups", ["offsets", "order", "place"])
RowGroups.__doc__ = """Rows sorted by group, as int32 tensors on the GPU; a slot is a row's choice.

offsets [groups + 1]: the groups' first places, and the end of the last. order [slots]: the slot
of each place, -1 behind the last group. place: the place of each slot, of the index's shape, -1
for slots in no group."""


def route(logits, k):
    """The k groups of each row with the largest logits, and the softmax over them:
    ``(index, weights)``, int32 and float32 [rows, k], largest first, ties to the lowest index.

    logits [rows, groups] (at most 1024 groups, k at most 32): float32, float16 or bfloat16. A logit
    of -inf is never chosen: index -1 and weight 0 in its place. NaN counts as the largest, and the
    row's weights are NaN. weights is differentiable in logits.
    """
    return (_BINDING or _native()).route(logits, k)


def row_groups(index, groups):
    """Sorts rows by group: ``RowGroups`` for ``to_groups``, ``grouped_linear`` and ``from_groups``.

    index [rows] or [rows, choices] (int32 or int64): the group of each slot; an index outside
    0 .. groups - 1 puts the slot in no group. Slots of a group keep their order. groups: at most
    1024.
    """
    return RowGroups(*(_BINDING or _native()).row_groups(index, groups))


def to_groups(x, groups):
    """The rows of x in the order of their groups: ``[slots, width]``, a row once for each of its
    choices, zeros behind the last group. x [rows, width]: float32, float16 or bfloat16,
    differentiable."""
    return (_BINDING or _native()).to_groups(x, *groups)


def from_groups(y, groups, weights=None):
    """Rows sorted by group back in their places: row r is ``sum_j weights[r, j] * y[place[r, j]]``.

    y [slots, width] (float32, float16 or bfloat16) and weights (float32, of the index's shape;
    None: all 1) are differentiable. Slots in no group add nothing, whatever their weight is.
    """
    return (_BINDING or _native()).from_groups(y, *groups, weights)


def grouped_linear(x, weight, groups, bias=None, activation=None):
    """``act(x weight[g]^T + bias[g])`` for the rows of each group g, as ``to_groups`` sorted them.

    x [slots, inputs], weight [groups, outputs, inputs] and bias [groups, outputs]: float16 or
    bfloat16, one type, differentiable. Rows behind the last group are zeros, and have no gradient.
    """
    return (_BINDING or _native()).grouped(x, weight, bias, *groups, _activation(activation), 0)


def grouped_gated_linear(x, weight, groups, bias=None, activation="silu"):
    """``act(x Wg[g]^T + bg[g]) * (x Wu[g]^T + bu[g])`` for the rows of each group g.

    weight [groups, 2 * outputs, inputs] and bias [groups, 2 * outputs] hold the gate's rows first.
    Types, order and gradients as in ``grouped_linear``.
    """
    act = _activation(activation)
    if act == L.RUNE_ACT_NONE:
        raise ValueError("grouped_gated_linear needs an activation.")
    return (_BINDING or _native()).grouped(x, weight, bias, *groups, act, 1)


def orthogonalize(x, steps=5, coefficients=NEWTON_SCHULZ, eps=1.0e-7):
    """x [..., rows, columns] with its singular values brought near 1, in bfloat16: ``steps`` times
    ``X <- a X + (b A + c A A) X`` with ``A = X X^T``, from ``x / (norm(x) + eps)``.

    For the update of a weight matrix, or of a stack of them (at most 65535). x: float32, float16 or
    bfloat16. The products take float16 operands and add in float32: a step rounds X, A and
    b A + c A A to 11 bits. Not differentiable.
    """
    a, b, c = coefficients
    return (_BINDING or _native()).orthogonalize(x, steps, a, b, c, eps)
