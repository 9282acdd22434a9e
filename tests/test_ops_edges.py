"""The network operators where their inputs, their environment or their waits are unusual: waits
that give up half way, values at the ends of the number range, transforms, several threads.
Bounds are derived from the roundings, as in test_ops.py."""

from __future__ import annotations

import ctypes
import math
import threading

import pytest
import torch

from rune_b200 import ops
from rune_b200.runtime import library as L
from tests.test_ops import (FUNC, U, act64, act_err, normal, products64, rounded, within,
                            z64)

gpu = pytest.mark.gpu


# -------------------------------------------------------------------------------- bounded waits
def give_up_after(polls, call):
    """call() with the in-kernel waits bounded by `polls`, to its end on the GPU"""
    lib = L.load_library()
    torch.cuda.synchronize()
    assert lib.rune_linear_set_wait_polls(polls) == L.RUNE_OK
    try:
        call()
        torch.cuda.synchronize()
    finally:
        lib.rune_linear_set_wait_polls(L.DEFAULT_WAIT_POLLS)


@gpu
@pytest.mark.parametrize("rows,inputs,outputs", [(3, 640, 512), (48, 8192, 256), (16, 96, 8)])
@pytest.mark.parametrize("gated", [False, True])
def test_few_rows_give_up_with_copies_and_products_in_flight(rows, inputs, outputs, gated):
    """A block whose waits run out part way lets its copies and products land and leaves its
    shared memory and TMEM in order: later launches on the same SMs give the same bits."""
    x, w = normal(1, rows, inputs), normal(2, 2 * outputs, inputs, scale=inputs ** -0.5)
    layer = ops.gated_linear if gated else ops.linear
    want = layer(x, w)
    for polls in (0, 1, 2, 3, 5, 8, 16):
        give_up_after(polls, lambda: layer(x, w))  # undefined, or whole if no wait was that long
        try:
            layer(x, w)
        except L.RuneError as e:
            assert "did not complete in time" in str(e)
        for _ in range(3):
            assert torch.equal(layer(x, w), want), polls


@gpu
@pytest.mark.parametrize("rows,inputs,outputs", [(300, 640, 512), (2000, 1024, 1024),
                                                 (130, 4096, 264), (9000, 256, 520)])
@pytest.mark.parametrize("gated", [False, True])
def test_tiles_give_up_with_copies_and_products_in_flight(rows, inputs, outputs, gated):
    """As above for the tiles, where the blocks of a pair may give up at different stages."""
    x, w = normal(1, rows, inputs), normal(2, 2 * outputs, inputs, scale=inputs ** -0.5)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    layer = ((lambda: ops.gated_linear(x, w, activation="tanh")) if gated
             else (lambda: ops.linear(x, w, activation="tanh")))
    y = layer()
    dy = normal(3, *y.shape)

    def backward():
        return torch.autograd.grad(y, leaves, dy, retain_graph=True)

    want = [y, *backward()]
    for polls in (0, 1, 2, 3, 5, 8, 16, 64):
        for call in (layer, backward):
            give_up_after(polls, call)
            try:
                layer()
            except L.RuneError as e:
                assert "did not complete in time" in str(e)
        for _ in range(3):
            for a, b in zip([layer(), *backward()], want):
                assert torch.equal(a, b), polls


@gpu
def test_every_operator_reports_a_wait_that_gave_up():
    x, w = normal(41, 300, 640), normal(42, 512, 640, scale=0.1)
    want = ops.linear(x, w)
    leaf = x.clone().requires_grad_(True)
    y, z = ops.rms_norm(leaf, w[0]), ops.linear(leaf, w)
    for call in (lambda: ops.rms_norm(x, w[0]), lambda: ops.rms_norm_fp8(x, w[0]),
                 lambda: ops.quantize_fp8(x), lambda: ops.padded(x), lambda: ops.linear(x, w),
                 lambda: ops.rms_norm(x[:0], w[0]), lambda: ops.linear(x[:0], w),
                 lambda: torch.autograd.grad(y.sum(), leaf, retain_graph=True),
                 lambda: torch.autograd.grad(z.sum(), leaf, retain_graph=True),
                 ops.check_waits, lambda: ops.check_waits("cuda"), lambda: ops.check_waits("cuda:0")):
        give_up_after(0, lambda: ops.linear(x, w))
        with pytest.raises(RuntimeError, match="did not complete in time"):
            call()
        call()  # reported once
        assert torch.equal(ops.linear(x, w), want)


@gpu
def test_a_replayed_graph_reports_a_wait_that_gave_up():
    x, w = normal(43, 300, 640), normal(44, 512, 640, scale=0.1)
    ops.linear(x, w)
    graph = torch.cuda.CUDAGraph()

    def capture():
        with torch.cuda.graph(graph):
            ops.linear(x, w)

    give_up_after(0, capture)  # the bound is the launch's
    ops.check_waits()
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(L.RuneError, match="did not complete in time"):
        ops.check_waits()
    ops.check_waits()


@gpu
@pytest.mark.parametrize("layer", ["norm", "linear", "gated"])
def test_a_failure_inside_a_backward_keeps_its_exception(layer):
    x, w = normal(45, 300, 640).requires_grad_(True), normal(46, 512, 640, scale=0.1)
    y = {"norm": lambda: ops.rms_norm(x, w[0]), "linear": lambda: ops.linear(x, w),
         "gated": lambda: ops.gated_linear(x, w)}[layer]()
    for run in (lambda: torch.autograd.grad(y.sum(), x, retain_graph=True),
                lambda: y.sum().backward(retain_graph=True)):
        give_up_after(0, lambda: ops.linear(x.detach(), w))
        with pytest.raises(L.RuneError, match="did not complete in time"):
            run()
        run()
    assert bool(x.grad.isfinite().all())


# ---------------------------------------------------------------------------------- tiny values
def check_rows_in_8_bits(q, scale, y, slack):
    """q * scale against y (float64): scale within `slack` of its definition, each value within
    e4m3's rounding (2^-4 of the value, 2^-10 below the smallest normal)"""
    amax = y.abs().amax(-1)
    want = torch.where(amax > 0, (amax / 448.0).clamp(min=2.0 ** -126), torch.ones_like(amax))
    assert bool(((scale.double() - want).abs() <= slack * want).all())
    v = y / scale.double()[:, None]
    off = (q.double() - v).abs()  # NaN where q is
    assert bool((off <= 2.0 ** -4 * (1 + 1e-3) * v.abs() + 2.0 ** -10 + 448 * slack).all())


def tiny_rows(width, tops, dtype):
    """rows of random values whose largest magnitudes are `tops`, every third value zero"""
    pattern = normal(11, len(tops), width, dtype=torch.float32).double()
    pattern[:, ::3] = 0.0
    pattern /= pattern.abs().amax(-1, keepdim=True)
    return (pattern * torch.tensor(tops, dtype=torch.float64, device="cuda")[:, None]).to(dtype)


TINY_TOPS = [1.0, 1e-28, 1e-30, 1e-32, 1e-34, 1e-35, 1e-36, 1e-37, 1e-38, 1e-40, 1e-42, 1e-44]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("width", [5, 64, 264, 1001, 5000, 20001])
def test_rows_of_tiny_values_to_8_bits(width, dtype):
    tops = TINY_TOPS if dtype is not torch.float16 else [1.0, 1e-4, 1e-6, 6e-8]
    x = tiny_rows(width, tops, dtype)
    check_rows_in_8_bits(*ops.quantize_fp8(x), x.double(), 4 * 2.0 ** -24)


@gpu
@pytest.mark.parametrize("width", [64, 1001, 20001])
@pytest.mark.parametrize("tiny_weight", [False, True])
def test_norm_of_tiny_values_to_8_bits(width, tiny_weight):
    """With h^2 below eps the norm multiplies by 1 / sqrt(eps); with a tiny weight only y is tiny.
    h w may be subnormal in float32: 2^-149 of it is 2^-149 / sqrt(eps) of y."""
    eps = 1e-8
    if tiny_weight:
        x = normal(12, 9, width, dtype=torch.float32)
        w = tiny_rows(width, [3e-38], torch.float32)[0]
    else:
        x = tiny_rows(width, [1e-22, 1e-28, 1e-32, 1e-34, 1e-36, 1e-37, 2e-38], torch.float32)
        w = normal(13, width, dtype=torch.float32, scale=0.2) + 1
    h = x.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()
    slack = (width + 16) * 2.0 ** -24
    if not tiny_weight:  # of a row's largest value
        slack += float((2.0 ** -149 * eps ** -0.5 / y.abs().amax(-1)).max())
    check_rows_in_8_bits(*ops.rms_norm_fp8(x, w, eps=eps), y, slack)


# --------------------------------------------------------------------------------- activations
def activation64(kind, z):
    """value, derivative and the sum of the derivative's terms' magnitudes, without cancellation"""
    if kind == "tanh":
        d = torch.cosh(z) ** -2
        return torch.tanh(z), d, d
    if kind == "silu":
        s = torch.sigmoid(z)
        rest = torch.sigmoid(-z)
        return z * s, s * (1 + z * rest), s * (1 + z.abs() * rest)
    cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    density = torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return z * cdf, cdf + z * density, cdf + z.abs() * density


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
@pytest.mark.parametrize("inputs", [8, 1032])  # z recomputed, z saved
@pytest.mark.parametrize("rows", [48, 4001])   # few rows, tiles
@pytest.mark.parametrize("gated", [False, True])
def test_activations_to_their_tails(act, dtype, inputs, rows, gated):
    """Each output is the activation of one exact z in -10 .. 10 (times 1 in the gated layer): off by
    its rounding and 4e-6, and z^2 2^-23 for the argument of an exponential, of itself; its
    derivative by as much of its terms."""
    z = torch.linspace(-10.0, 10.0, rows, device="cuda").to(dtype)
    x = torch.zeros(rows, inputs, dtype=dtype, device="cuda")
    x[:, 0] = z
    x.requires_grad_(True)
    w = torch.zeros(16, inputs, dtype=dtype, device="cuda")
    w[:8, 0] = 1.0
    if gated:
        b = torch.zeros(16, dtype=dtype, device="cuda")
        b[8:] = 1.0
        y = ops.gated_linear(x, w, bias=b, activation=act)
    else:
        y = ops.linear(x, w, activation=act)
    dy = torch.zeros_like(y)
    dy[:, 3] = 1.0
    (dx,) = torch.autograd.grad(y, x, dy)
    z = z.double()
    value, slope, terms = activation64(act, z)
    func = FUNC + 2.0 ** -23 * z * z
    within(y[:, 3].detach(), value, (U[dtype] + func) * value.abs(), "value")
    within(dx[:, 0], slope, U[dtype] * slope.abs() + (1 + U[dtype]) * func * terms, "derivative")


# ---------------------------------------------------------------------------------- transforms
def every_operator(x, w):
    """calls of square x and w, one an operator, with x and with w as the input"""
    for f in (lambda a, b: ops.linear(a, b), lambda a, b: ops.gated_linear(a, b),
              lambda a, b: ops.linear(b, b, bias=b[0], residual=a),
              lambda a, b: ops.rms_norm(a, b[0]), lambda a, b: ops.rms_norm_fp8(a, b[0])):
        yield lambda a, f=f: f(a, w)
        yield lambda a, f=f: f(x, a)
    yield lambda a: ops.quantize_fp8(a)
    yield lambda a: ops.padded(a)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_and_traces_are_refused(device):
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.ones(16, 16, dtype=torch.bfloat16, device=device)
    for f in every_operator(x, torch.ones_like(x)):
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError,
                                                                     match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(lambda a: f(a + 1), x, check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(lambda a: f(a + 1))(x)
        for transform in (lambda: torch.func.vmap(f)(x[None]), lambda: torch.func.jvp(f, (x,), (x,))):
            with pytest.raises((RuntimeError, ValueError)):
                transform()


@gpu
def test_transforms_of_a_backward_are_refused():
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    x = normal(21, 60, 64).requires_grad_(True)
    w = normal(22, 64, 64).requires_grad_(True)
    for y in (ops.linear(x, w, activation="tanh"), ops.rms_norm(x, w[0])):
        dy = torch.ones_like(y)

        def backward(g):
            return torch.autograd.grad(y, x, g, retain_graph=True)[0]

        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            backward(forward_ad.make_dual(dy, dy))
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(backward)(dy)
        assert bool(backward(dy).isfinite().all())


@gpu
def test_hooks_on_saved_tensors_keep_their_exceptions():
    """Activation checkpointing ends its recomputation by an exception in such a hook."""
    from torch.utils.checkpoint import checkpoint

    class Stop(Exception):
        pass

    def stop(_):
        raise Stop("here")

    w = normal(25, 64, 64)
    for f in (lambda t: ops.linear(t, w, activation="gelu"), lambda t: ops.gated_linear(t, w),
              lambda t: ops.rms_norm(t, w[0]),
              lambda t: ops.linear(ops.rms_norm(t, w[0], residual=t)[1], w, residual=t)):
        x = normal(24, 60, 64).requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(stop, lambda t: t), pytest.raises(
                Stop, match="here"):
            f(x)
        (want,) = torch.autograd.grad(f(x).sum(), x)
        (got,) = torch.autograd.grad(checkpoint(f, x, use_reentrant=False).sum(), x)
        assert torch.equal(got, want)
        checkpoint(f, x, use_reentrant=True).sum().backward()
        assert torch.equal(x.grad, want)


# ------------------------------------------------------------------------------------ refusals
def refused_at(name, args, fields, step):
    """rune_<name> refuses each field at an address `step` bytes off, and launches nothing"""
    call = getattr(L.load_library(), name)
    for field in fields:
        raw = type(args)()
        ctypes.pointer(raw)[0] = args
        setattr(raw, field, getattr(raw, field) + step)
        assert call(ctypes.byref(raw), None) == L.RUNE_ERR_INVALID, (name, field)


@gpu
def test_misaligned_arrays_are_refused():
    """An address inside a value, or a saved z off 16 bytes, would fault in the kernels."""
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    at = [buf.data_ptr() + 4096 * i for i in range(12)]
    size = dict(rows=4, width=16, x_stride=16, residual_stride=16, dtype=L.RUNE_F32,
                weight_dtype=L.RUNE_F32)
    norm = L.NormArgs(**size, out_dtype=L.RUNE_F32, x=at[0], residual=at[1], weight=at[2],
                      y=at[3], h=at[4], scale=at[5], rstd=at[6])
    refused_at("rune_rms_norm", norm, ("x", "residual", "weight", "y", "h", "scale", "rstd"), 2)
    grad = L.NormGradArgs(**size, dy_stride=16, dh_stride=16, x=at[0], residual=at[1],
                          weight=at[2], rstd=at[3], dy=at[4], dh=at[5], dx=at[6], dweight=at[7],
                          workspace=at[8], workspace_bytes=16384)
    refused_at("rune_rms_norm_backward", grad,
               ("x", "residual", "weight", "rstd", "dy", "dh", "dx", "dweight"), 2)
    size = dict(rows=4, inputs=16, outputs=8, x_stride=16, weight_stride=16, dtype=L.RUNE_BF16,
                activation=L.RUNE_ACT["silu"])
    linear = L.LinearArgs(**size, out_dtype=L.RUNE_BF16, residual_stride=8, x=at[0], weight=at[1],
                          bias=at[2], residual=at[3], y=at[4], saved=at[5])
    refused_at("rune_linear", linear, ("x", "weight", "bias", "residual", "y"), 1)
    refused_at("rune_linear", linear, ("saved",), 8)
    linear.dtype, linear.x_scale, linear.weight_scale = L.RUNE_E4M3, at[6], at[7]
    refused_at("rune_linear", linear, ("x_scale", "weight_scale"), 2)
    grad = L.LinearGradArgs(**size, dy_stride=8, x=at[0], weight=at[1], bias=at[2], dy=at[3],
                            saved=at[4], dx=at[5], dweight=at[6], dbias=at[7], workspace=at[8],
                            workspace_bytes=16384)
    refused_at("rune_linear_backward", grad,
               ("x", "weight", "bias", "dy", "dx", "dweight", "dbias"), 1)
    refused_at("rune_linear_backward", grad, ("saved",), 8)


@gpu
@pytest.mark.parametrize("layer", [ops.linear, ops.gated_linear])
def test_scales_that_require_a_gradient_are_refused(layer):
    """as the 8-bit operands and their bias are: the call has no gradient to give"""
    (x, xs), (w, ws) = ops.quantize_fp8(normal(31, 60, 64)), ops.quantize_fp8(normal(32, 48, 64))
    want = layer(x, w, x_scale=xs, weight_scale=ws)
    for scales in ((xs.clone().requires_grad_(True), ws), (xs, ws.clone().requires_grad_(True))):
        with pytest.raises(ValueError, match="no gradient"):
            layer(x, w, x_scale=scales[0], weight_scale=scales[1])
        with torch.no_grad():
            assert torch.equal(layer(x, w, x_scale=scales[0], weight_scale=scales[1]), want)


# ------------------------------------------------------------------------------------- threads
@gpu
@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, L.RUNE_BF16), (torch.float32, L.RUNE_F32)])
def test_two_threads_with_different_widths(dtype, code):
    """The norm's backward through the C entry, which holds no lock: each call's shared memory is
    allowed whatever the other thread's calls need."""
    lib = L.load_library()
    failures, results = [], {}

    def work(width, stream):
        x, dy = normal(51, 64, width, dtype=dtype), normal(52, 64, width, dtype=dtype)
        w, rstd = normal(53, width, dtype=dtype), torch.ones(64, device="cuda")
        dx, first = torch.empty_like(x), None
        args = L.NormGradArgs(rows=64, width=width, x_stride=width, dy_stride=width, dtype=code,
                              weight_dtype=code, x=x.data_ptr(), weight=w.data_ptr(),
                              rstd=rstd.data_ptr(), dy=dy.data_ptr(), dx=dx.data_ptr())
        torch.cuda.synchronize()
        for i in range(2000):
            status = lib.rune_rms_norm_backward(ctypes.byref(args), stream.cuda_stream)
            if status:
                failures.append((width, status, lib.rune_last_error()))
            if i == 0:
                stream.synchronize()
                first = dx.clone()
        stream.synchronize()
        results[width] = torch.equal(first, dx)

    threads = [threading.Thread(target=work, args=(width, torch.cuda.Stream()))
               for width in (4096, 8192)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures and results == {4096: True, 8192: True}, failures[:2]


# --------------------------------------------------------------------------------------- build
def test_the_binding_is_stale_under_another_torch(tmp_path, monkeypatch):
    """Its ABI is torch's and Python's; the sources' times alone do not show a new one."""
    from rune_b200.runtime import build

    binding, stamp = tmp_path / "_ops.so", tmp_path / "obj" / "_ops.txt"
    monkeypatch.setattr(build, "BINDING", binding)
    monkeypatch.setattr(build, "BINDING_STAMP", stamp)
    commands = []

    def compile_(cmd, **_):
        commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("Done", (), {"returncode": 0})

    monkeypatch.setattr(build.subprocess, "run", compile_)
    assert build.build_binding() == binding and len(commands) == 1
    assert build.build_binding() == binding and len(commands) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.binding_stale()
    assert build.build_binding() == binding and len(commands) == 2
    assert not build.binding_stale()


# ------------------------------------------------------------- sums that keep their digits
def cancelling(dy, first, second):
    """dy for even rows, and for odd ones the 16-bit values that cancel dy * first in a sum with
    second to a rounding of them: what is left is gone if a factor of a term is rounded again"""
    return torch.stack([dy, -(dy.double() * first / second).to(dy.dtype)])


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("width", [64, 264, 1001])
def test_norm_gradients_use_both_addends_unrounded(width, dtype):
    """h = x + residual has more digits than 16 bits. dweight: two kinds of rows whose terms cancel
    to a rounding's size; off by float32's errors of r, n and the sums, and its own rounding. dx:
    dy along n, which the projection cancels to a rounding's size likewise."""
    rows, eps = 512, 1e-6
    f = (width + 16) * 2.0 ** -23
    base = [normal(61 + i, 2, width, dtype=dtype, scale=s) for i, s in enumerate((1.0, 0.3))]
    base = [t + torch.sign(t) * (0.5 if i == 0 else 0.0) for i, t in enumerate(base)]
    pair = base[0].double() + base[1].double()
    n2 = pair / torch.sqrt((pair * pair).mean(-1, keepdim=True) + eps)
    x, res = (t.repeat(rows // 2, 1).requires_grad_(True) for t in base)
    w = torch.ones(width, dtype=dtype, device="cuda", requires_grad=True)
    dy = cancelling(normal(64, width, dtype=dtype), n2[0], n2[1]).repeat(rows // 2, 1)
    y, _ = ops.rms_norm(x, w, residual=res, eps=eps)
    (dw,) = torch.autograd.grad(y, w, dy, retain_graph=True)
    term = dy.double() * n2.repeat(rows // 2, 1)
    ok = term.abs().amax(0).isfinite()
    want, size = term.sum(0), term.abs().sum(0)
    within(dw[ok], want[ok], ((f + rows * 2.0 ** -24) * size + U[dtype] * want.abs())[ok], "dweight")
    n = n2.repeat(rows // 2, 1)
    dy = n.to(dtype)
    (dx,) = torch.autograd.grad(y, x, dy)
    r = 1.0 / torch.sqrt((pair * pair).mean(-1, keepdim=True) + eps).repeat(rows // 2, 1)
    dot = (dy.double() * n).mean(-1, keepdim=True)
    want = r * (dy.double() - n * dot)
    within(dx, want, U[dtype] * want.abs() + 4 * f * r * (dy.double().abs() + (n * dot).abs()), "dx")


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("inputs", [8, 1032])  # z recomputed, z saved
@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_dbias_sums_unrounded_dz(inputs, act, dtype, gated):
    """Two kinds of rows whose dz cancel to a rounding's size in every column; z is exact. Off by
    the activation's error of each term, float32 sums in a tree of fewer than 40 additions, and
    the sum's own rounding."""
    rows, outputs = 2000, 24
    x = torch.zeros(rows, inputs, dtype=dtype, device="cuda")
    x[0::2, 0], x[1::2, 0] = 0.75, 0.34375
    w = torch.zeros(2 * outputs if gated else outputs, inputs, dtype=dtype, device="cuda")
    w[:outputs, 0] = 0.5 + torch.rand(outputs, generator=torch.Generator().manual_seed(5)).cuda()
    b = torch.zeros(len(w), dtype=dtype, device="cuda", requires_grad=True)
    z = x[:2, :1].double() * w[:outputs, 0].double()
    value, slope, terms = activation64(act, z)
    up = 1.0
    if gated:
        w[outputs:, 0], up = 1.25, 1.25 * x[:2, :1].double()
    dy = cancelling(normal(65, outputs, dtype=dtype), (slope * up)[0], (slope * up)[1])
    y = (ops.gated_linear(x.requires_grad_(True), w, bias=b, activation=act) if gated
         else ops.linear(x.requires_grad_(True), w, bias=b, activation=act))
    (db,) = torch.autograd.grad(y, b, dy.repeat(rows // 2, 1))
    dz = (dy.double() * up * slope).sum(0) * (rows // 2)
    size = (dy.double().abs() * up * terms).sum(0) * (rows // 2)
    func = FUNC + 2.0 ** -23 * float(z.abs().max()) ** 2 + 42 * 2.0 ** -24
    within(db[:outputs], dz, U[dtype] * dz.abs() + func * size, "dbias")


# ------------------------------------------------------------------------------- many tiles
@gpu
@pytest.mark.parametrize("rows,inputs,outputs", [(10000, 264, 600), (300, 4200, 5000),
                                                 (6003, 1100, 1000)])
@pytest.mark.parametrize("gated", [False, True])
def test_more_tiles_than_blocks_and_more_than_one_group(rows, inputs, outputs, gated):
    """Every value of results and gradients whose products have more rows of tiles than a group and
    more tiles than blocks at once."""
    dtype, u = torch.bfloat16, U[torch.bfloat16]
    x = normal(71, rows, inputs, dtype=dtype).requires_grad_(True)
    w = normal(72, outputs, inputs, dtype=dtype, scale=inputs ** -0.5).requires_grad_(True)
    b = normal(73, outputs, dtype=dtype, scale=0.5).requires_grad_(True)
    half = outputs // 2 if gated else outputs
    dy = normal(74, rows, half, dtype=dtype)
    y = (ops.gated_linear(x, w, bias=b, activation="gelu") if gated
         else ops.linear(x, w, bias=b, activation="gelu"))
    grads = torch.autograd.grad(y, [x, w, b], dy)
    z, ez = z64(x.detach(), w.detach(), b.detach())
    g = dy.double()
    gate, eg = z[:, :half], ez[:, :half]
    a, da, _ = act64("gelu", gate)
    ea, eda = act_err("gelu", gate, eg)
    want, ey, dz, ddz = a, ea, g * da, g.abs() * eda
    if gated:
        up, eu = z[:, half:], ez[:, half:]
        want, ey = a * up, ea * (up.abs() + eu) + a.abs() * eu
        dz = torch.cat([g * up * da, g * a], 1)
        ddz = torch.cat([g.abs() * (eda * (up.abs() + eu) + da.abs() * eu), g.abs() * ea], 1)
    within(y.detach(), *rounded((want, ey + 2.0 ** -23 * want.abs()), u), "y")
    pairs = products64(dz, ddz + 2.0 ** -22 * dz.abs(), x.detach(), w.detach(), u, rows)
    for name, got, pair in zip(("dx", "dweight", "dbias"), grads, pairs):
        within(got, *rounded(pair, u), name)
