"""The network operators (rune_b200.ops) against their definitions in float64.

Tolerances are derived, elementwise, from the roundings that the kernels make. With unit
roundoffs u (2^-8 for bfloat16, 2^-11 for float16, 2^-24 for float32) and S the sum of the
absolute products of a result, a float32 sum of n products is off by at most n 2^-23 S (the tensor
core may truncate where it adds), the special functions by 4e-6 of their value and of their
argument's scale, dz by its one rounding to 16 bits, and every result by its own last rounding."""

from __future__ import annotations

import ctypes
import subprocess
import textwrap

import pytest
import torch

from rune_b200 import ops
from rune_b200.runtime import library as L
from tests.helpers import ROOT

gpu = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-38, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}
NARROW = [torch.float16, torch.bfloat16]
FUNC = 4.0e-6  # error of the special functions, of their value
EPS = 1.0e-6


def normal(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def within(got, want, bound, what):
    assert got.shape == want.shape, what
    bad = (got.double() - want).abs() > bound + TINY[got.dtype]
    bad |= got.double().isnan() != want.isnan()
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} off; worst "
        f"{float(((got.double() - want).abs() / (bound + TINY[got.dtype])).nan_to_num().max()):.3g}"
        " of the bound")


def act64(kind, z):
    """value, first and bound of the second derivative in float64"""
    if kind is None:
        return z, torch.ones_like(z), 0.0
    z = z.detach().requires_grad_(True)
    fn = {"tanh": torch.tanh, "silu": torch.nn.functional.silu,
          "gelu": torch.nn.functional.gelu}[kind]
    with torch.enable_grad():
        y = fn(z)
        (d,) = torch.autograd.grad(y.sum(), z)
    return y.detach(), d.detach(), {"tanh": 0.77, "silu": 0.5, "gelu": 0.8}[kind]


# ------------------------------------------------------------------------------------ CPU
def test_argument_structs_match_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text(textwrap.dedent(f"""
        #include <stddef.h>
        #include <stdio.h>
        #include "{ROOT / 'include' / 'rune_b200.h'}"
        int main(void) {{
            printf("%zu %zu %zu %zu %zu %zu %zu %zu\\n", sizeof(rune_norm_args),
                   sizeof(rune_norm_grad_args), sizeof(rune_linear_args),
                   sizeof(rune_linear_grad_args), offsetof(rune_norm_args, rstd),
                   offsetof(rune_norm_grad_args, workspace_bytes),
                   offsetof(rune_linear_args, workspace_bytes),
                   offsetof(rune_linear_grad_args, workspace_bytes));
            return 0;
        }}"""))
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    structs = (L.NormArgs, L.NormGradArgs, L.LinearArgs, L.LinearGradArgs)
    sizes = [ctypes.sizeof(s) for s in structs]
    assert got == sizes + [sizes[0] - 8, sizes[1] - 8, sizes[2] - 8, sizes[3] - 8]


def test_cpu_tensors_and_unknown_activations_are_refused():
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.rms_norm(x, w[0]), lambda: ops.linear(x, w),
                 lambda: ops.gated_linear(x, w), lambda: ops.quantize_fp8(x)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="Unsupported activation"):
        ops.linear(x, w, activation="relu6")
    with pytest.raises(ValueError, match="needs an activation"):
        ops.gated_linear(x, w, activation=None)


def test_null_arguments_are_refused_by_the_library():
    lib = L.load_library()
    need = ctypes.c_int64(0)
    assert lib.rune_rms_norm(None, None) == L.RUNE_ERR_INVALID
    assert lib.rune_rms_norm_backward(None, None) == L.RUNE_ERR_INVALID
    assert lib.rune_linear(None, None) == L.RUNE_ERR_INVALID
    assert lib.rune_linear_backward(None, None) == L.RUNE_ERR_INVALID
    assert lib.rune_linear_workspace(None, ctypes.byref(need)) == L.RUNE_ERR_INVALID


# ------------------------------------------------------------------------------------ norm
NORM_SIZES = [(1, 1), (1, 4096), (3, 7), (17, 256), (130, 128), (5, 264), (33, 1000), (9, 1001),
              (4, 1024), (3, 2049), (7, 5000), (2, 8192), (2, 8200), (3, 20001), (700, 96)]


def norm64(x, w, res, eps):
    h = x.double() if res is None else x.double() + res.double()
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * r * w.double(), h, r


def norm_bounds(h, y, width, dtype):
    """|y - y64| and |h - h64|: the mean's sum (width 2^-24 relative, halved by the root), four
    float32 operations, the output's rounding."""
    rel = width * 2.0 ** -24 + 8 * 2.0 ** -24
    return (rel + U[dtype]) * y.abs(), (U[dtype] + 2.0 ** -24) * h.abs()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, *NARROW], ids=str)
@pytest.mark.parametrize("rows,width", NORM_SIZES)
@pytest.mark.parametrize("with_res", [False, True])
def test_rms_norm_forward_and_backward(rows, width, dtype, with_res):
    x = normal(1, rows, width, dtype=dtype, scale=2.0).requires_grad_(True)
    w = (normal(2, width, dtype=dtype, scale=0.2) + 1).detach().requires_grad_(True)
    res = normal(3, rows, width, dtype=dtype).requires_grad_(True) if with_res else None
    dy, dh = normal(4, rows, width, dtype=dtype), normal(5, rows, width, dtype=dtype)
    y64, h64, r64 = norm64(x.detach(), w.detach(), None if res is None else res.detach(), EPS)
    by, bh = norm_bounds(h64, y64, width, dtype)
    got = ops.rms_norm(x, w, residual=res, eps=EPS)
    y, h = got if with_res else (got, None)
    within(y.detach(), y64, by, "y")
    if with_res:
        within(h.detach(), h64, bh, "h")
        dx, dw, dres = torch.autograd.grad([y, h], [x, w, res], [dy, dh])
        assert torch.equal(dx, dres)
    else:
        dx, dw = torch.autograd.grad(y, [x, w], dy)
    # the gradients as formulas; h reaches the backward rounded to the rows' type
    g, n = dy.double(), h64 * r64
    gw = g * w.detach().double()
    dot = (gw * n).mean(-1, keepdim=True)
    dx64 = r64 * (gw - n * dot) + (dh.double() if with_res else 0.0)
    dw64 = (g * n).sum(0)
    u = U[dtype] if with_res else 0.0  # of the saved h
    f = (width + 16) * 2.0 ** -23
    dn = (u + f) * n.abs()
    ddot = (gw.abs() * dn + f * (gw * n).abs()).mean(-1, keepdim=True)
    bx = r64 * (dn * dot.abs() + n.abs() * ddot) + f * r64 * (gw.abs() + (n * dot).abs())
    bx = bx + U[dtype] * dx64.abs() + f * (dx64.abs() + (dh.double().abs() if with_res else 0.0))
    bw = ((u + f + rows * 2.0 ** -24) * (g * n).abs()).sum(0) + U[dtype] * dw64.abs()
    within(dx, dx64, bx * (1 + U[dtype]), "dx")
    within(dw, dw64, bw * (1 + U[dtype]), "dweight")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, *NARROW], ids=str)
@pytest.mark.parametrize("rows,width", NORM_SIZES)
@pytest.mark.parametrize("with_res", [False, True])
def test_rms_norm_fp8(rows, width, dtype, with_res):
    x = normal(1, rows, width, dtype=dtype, scale=2.0)
    x[rows // 2] = 0.0
    w = normal(2, width, dtype=torch.float32, scale=0.2) + 1  # float32 weight beside any rows
    res = normal(3, rows, width, dtype=dtype) if with_res else None
    if with_res:
        res[rows // 2] = 0.0
    y64, h64, _ = norm64(x, w, res, EPS)
    got = ops.rms_norm_fp8(x, w, residual=res, eps=EPS)
    q, scale = got[:2]
    rel = (width + 16) * 2.0 ** -24
    amax = y64.abs().amax(-1)
    want = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    assert q.dtype is torch.float8_e4m3fn
    within(scale, want, rel * want, "scale")
    assert float(scale[rows // 2]) == 1.0 and not bool(q[rows // 2].float().any())
    # e4m3: 2^-4 of the value, 2^-10 below the smallest normal (2^-6)
    v = y64 / scale.double()[:, None]
    off = (q.double() - v).abs()
    assert bool((off <= 2.0 ** -4 * v.abs() * (1 + 1e-3) + 2.0 ** -10 + rel * 448).all())
    if with_res:
        within(got[2], h64, norm_bounds(h64, y64, width, dtype)[1], "h")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, *NARROW], ids=str)
def test_quantize_fp8_and_its_strides(dtype):
    base = normal(6, 40, 3, 200, dtype=dtype)
    x = base[:, 1, 8:135]  # rows 600 apart, odd width
    q, scale = ops.quantize_fp8(x)
    want = x.double().abs().amax(-1) / 448.0
    within(scale, want, 4 * 2.0 ** -24 * want, "scale")
    v = x.double() / scale.double()[:, None]
    assert bool(((q.double() - v).abs() <= 2.0 ** -4 * v.abs() * 1.001 + 2.0 ** -10).all())
    assert q.float().abs().amax() == 448.0


@gpu
def test_rms_norm_strided_and_leading_axes():
    base = normal(7, 6, 5, 300, dtype=torch.float16)
    w = normal(8, 256, dtype=torch.float16)
    for x in (base[:, 2, 7:263], base[:, :, 8:264], base[0, 0, :256], base[:0, 0, :256]):
        y = ops.rms_norm(x, w, eps=EPS)
        y64 = norm64(x, w, None, EPS)[0]
        within(y, y64, norm_bounds(y64, y64, 256, torch.float16)[0], "y")
    # a transposed view and a broadcast gradient
    t = normal(9, 256, 12, dtype=torch.float16).t().requires_grad_(True)
    y = ops.rms_norm(t, w, eps=EPS)
    (dx,) = torch.autograd.grad(y, t, torch.ones(1, 1, dtype=torch.float16,
                                                 device="cuda").expand(12, 256))
    (ref,) = torch.autograd.grad(ops.rms_norm(t.contiguous(), w, eps=EPS).sum(), t)
    assert torch.equal(dx, ref)


@gpu
def test_rms_norm_keeps_nan_and_inf_to_their_rows():
    x = normal(10, 8, 512, dtype=torch.bfloat16)
    x[2, 5], x[4, 7] = float("nan"), float("inf")
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    y = ops.rms_norm(x, w)
    assert bool(y[2].isnan().all()) and bool(y[4, 7].isnan())
    assert bool((y[4, :7] == 0).all())
    clean = [0, 1, 3, 5, 6, 7]
    assert torch.equal(y[clean], ops.rms_norm(x[clean].contiguous(), w))
    q, scale = ops.rms_norm_fp8(x, w)
    assert bool(scale[2].isnan()) and bool(q[2].float().isnan().all())
    assert bool(scale[clean].isfinite().all())


@gpu
def test_rms_norm_gradient_by_differences():
    """Directional derivative of the kernel's own float32 outputs. Central differences of step
    t have a remainder of t^2 / 6 times the third derivative (bounded by the measured curvature
    of the float64 form) and the outputs' rounding over t."""
    rows, width, t = 6, 320, 2.0 ** -6
    x = normal(11, rows, width, dtype=torch.float32).requires_grad_(True)
    w = (normal(12, width, dtype=torch.float32, scale=0.2) + 1).detach().requires_grad_(True)
    c = normal(13, rows, width, dtype=torch.float32)
    vx, vw = normal(14, rows, width, dtype=torch.float32), normal(15, width, dtype=torch.float32)
    dx, dw = torch.autograd.grad(ops.rms_norm(x, w, eps=EPS), [x, w], c)
    slope = float((dx.double() * vx.double()).sum() + (dw.double() * vw.double()).sum())

    def loss(s):
        return float((ops.rms_norm(x.detach() + s * vx, w.detach() + s * vw, eps=EPS).double()
                      * c.double()).sum())

    def loss64(s):
        y = norm64(x.detach().double() + s * vx.double(), w.detach().double() + s * vw.double(),
                   None, EPS)[0]
        return float((y * c.double()).sum())

    third = abs(loss64(2 * t) - 2 * loss64(t) + 2 * loss64(-t) - loss64(-2 * t)) / (2 * t ** 3)
    rounding = (width + 16) * 2.0 ** -24 * float((norm64(x.detach(), w.detach(), None, EPS)[0]
                                                 * c.double()).abs().sum())
    found = (loss(t) - loss(-t)) / (2 * t)
    assert abs(found - slope) <= t * t / 6 * third * 2 + 2 * rounding / t + 2 * rounding


# ---------------------------------------------------------------------------------- linear
LINEAR_SIZES = [(1, 8, 8), (2, 1, 1), (1, 100, 36), (3, 17, 5), (1, 4096, 256), (7, 513, 96),
                (16, 2048, 72), (33, 64, 128), (65, 136, 24), (130, 64, 128), (127, 129, 255),
                (300, 515, 1001), (257, 72, 8), (128, 1024, 128), (1000, 256, 512),
                (513, 520, 264)]


def z64(x, w, b, scaled=None):
    """pre-activation, and the bound of its float32 error"""
    x, w = x.double(), w.double()
    z, s = x @ w.t(), x.abs() @ w.abs().t()
    n = x.shape[1]
    err = (n + 2) * 2.0 ** -23 * s
    if scaled is not None:
        f = scaled[0].double()[:, None] * scaled[1].double()[None, :]
        z, err = z * f, err * f + 4 * 2.0 ** -24 * (s * f)
    if b is not None:
        z = z + b.double()
        err = err + 2.0 ** -23 * z.abs()
    return z, err


def act_err(kind, z, err):
    """error of act and of its derivative at z for an error err of z"""
    if kind is None:
        return err, torch.zeros_like(z)
    y, d, second = act64(kind, z)
    return 1.2 * err + FUNC * (y.abs() + z.abs() * 0.1), second * err + FUNC * (1 + z.abs())


def products64(dz, ddz, x, w, u, n_rows):
    """dx and dweight from dz (its error before the rounding to 16 bits: ddz), with bounds"""
    x, w = x.double(), w.double()
    e = ddz + u * dz.abs() * (1 + u)
    n_out = dz.shape[1]
    dx, dw = dz @ w, dz.t() @ x
    bx = e @ w.abs() + (n_out + 2) * 2.0 ** -23 * ((dz.abs() + e) @ w.abs())
    bw = e.t() @ x.abs() + (n_rows + 2) * 2.0 ** -23 * ((dz.abs() + e).t() @ x.abs())
    bb = e.sum(0) + n_rows * 2.0 ** -23 * (dz.abs() + e).sum(0)
    return (dx, bx), (dw, bw), (dz.sum(0), bb)


def rounded(pair, u):
    want, bound = pair
    return want, bound + u * (want.abs() + bound)


@gpu
@pytest.mark.parametrize("dtype", NARROW, ids=str)
@pytest.mark.parametrize("rows,inputs,outputs", LINEAR_SIZES)
@pytest.mark.parametrize("act", [None, "tanh", "silu", "gelu"])
@pytest.mark.parametrize("extras", [False, True])
def test_linear_forward_and_backward(rows, inputs, outputs, dtype, act, extras):
    x = normal(21, rows, inputs, dtype=dtype).requires_grad_(True)
    w = normal(22, outputs, inputs, dtype=dtype, scale=inputs ** -0.5).requires_grad_(True)
    b = normal(23, outputs, dtype=dtype, scale=0.5).requires_grad_(True) if extras else None
    res = normal(24, rows, outputs, dtype=dtype).requires_grad_(True) if extras else None
    dy = normal(25, rows, outputs, dtype=dtype)
    u = U[dtype]
    z, ez = z64(x.detach(), w.detach(), None if b is None else b.detach())
    a, da, _ = act64(act, z)
    ea, eda = act_err(act, z, ez)
    want = a + (res.detach().double() if extras else 0.0)
    y = ops.linear(x, w, bias=b, activation=act, residual=res)
    within(y.detach(), *rounded((want, ea + 2.0 ** -23 * want.abs()), u), "y")
    with torch.no_grad():
        assert torch.equal(y, ops.linear(x, w, bias=b, activation=act, residual=res))
    leaves = [x, w] + ([b, res] if extras else [])
    grads = torch.autograd.grad(y, leaves, dy)
    g = dy.double()
    dz, ddz = g * da, g.abs() * eda + 2.0 ** -22 * (g * da).abs()
    if act is None:
        ddz = torch.zeros_like(dz)
    pairs = products64(dz, ddz, x.detach(), w.detach(), 0.0 if act is None else u, rows)
    for name, got, pair in zip(("dx", "dweight", "dbias"), grads, pairs):
        within(got, *rounded(pair, u), name)
    if extras:
        assert torch.equal(grads[3], dy)


@gpu
@pytest.mark.parametrize("dtype", NARROW, ids=str)
@pytest.mark.parametrize("rows,inputs,outputs", LINEAR_SIZES)
@pytest.mark.parametrize("act,with_bias", [("tanh", True), ("silu", False), ("gelu", True)])
def test_gated_forward_and_backward(rows, inputs, outputs, dtype, act, with_bias):
    n = 2 * outputs
    x = normal(31, rows, inputs, dtype=dtype).requires_grad_(True)
    w = normal(32, n, inputs, dtype=dtype, scale=inputs ** -0.5).requires_grad_(True)
    b = normal(33, n, dtype=dtype, scale=0.5).requires_grad_(True) if with_bias else None
    dy = normal(34, rows, outputs, dtype=dtype)
    u16 = U[dtype]
    z, ez = z64(x.detach(), w.detach(), None if b is None else b.detach())
    gate, up, eg, eu = z[:, :outputs], z[:, outputs:], ez[:, :outputs], ez[:, outputs:]
    a, da, _ = act64(act, gate)
    ea, eda = act_err(act, gate, eg)
    want = a * up
    ey = ea * (up.abs() + eu) + a.abs() * eu + 2.0 ** -23 * want.abs()
    y = ops.gated_linear(x, w, bias=b, activation=act)
    within(y.detach(), *rounded((want, ey), u16), "y")
    with torch.no_grad():
        assert torch.equal(y, ops.gated_linear(x, w, bias=b, activation=act))
    grads = torch.autograd.grad(y, [x, w] + ([b] if with_bias else []), dy)
    g = dy.double()
    dz = torch.cat([g * up * da, g * a], 1)
    ddz = torch.cat([g.abs() * (eda * (up.abs() + eu) + da.abs() * eu), g.abs() * ea], 1)
    pairs = products64(dz, ddz + 2.0 ** -22 * dz.abs(), x.detach(), w.detach(), u16, rows)
    for name, got, pair in zip(("dx", "dweight", "dbias"), grads, pairs):
        within(got, *rounded(pair, u16), name)


@gpu
@pytest.mark.parametrize("out", [None, torch.float16])
@pytest.mark.parametrize("rows,inputs,outputs", LINEAR_SIZES)
@pytest.mark.parametrize("gated", [False, True])
def test_fp8_forward(rows, inputs, outputs, gated, out):
    n = 2 * outputs if gated else outputs
    x, xs = ops.quantize_fp8(normal(41, rows, inputs, dtype=torch.float32))
    w, ws = ops.quantize_fp8(normal(42, n, inputs, dtype=torch.float32, scale=inputs ** -0.5))
    dtype = out or torch.bfloat16
    b = normal(43, n, dtype=dtype, scale=0.5)
    z, ez = z64(x.float(), w.float(), b, (xs, ws))
    if gated:
        y = ops.gated_linear(x, w, bias=b, x_scale=xs, weight_scale=ws, out_dtype=out)
        a, e = act64("silu", z[:, :outputs])[0], act_err("silu", z[:, :outputs], ez[:, :outputs])[0]
        up, eu = z[:, outputs:], ez[:, outputs:]
        want, err = a * up, e * (up.abs() + eu) + a.abs() * eu
    else:
        res = normal(44, rows, outputs, dtype=dtype)
        y = ops.linear(x, w, bias=b, activation="gelu", residual=res, x_scale=xs,
                       weight_scale=ws, out_dtype=out)
        want, err = act64("gelu", z)[0] + res.double(), act_err("gelu", z, ez)[0]
    within(y, *rounded((want, err + 2.0 ** -23 * want.abs()), U[dtype]), "y")


@gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows", [1, 9, 200])
def test_layers_with_strides(rows, gated):
    """Row-strided views, odd offsets, transposed weights and expanded gradients give the bits of
    their contiguous copies."""
    dt = torch.bfloat16
    wide = normal(51, rows, 3, 400, dtype=dt)
    weights = normal(52, 130, 700, dtype=dt, scale=0.1)
    layer = (lambda *a: ops.gated_linear(*a)) if gated else (
        lambda *a: ops.linear(*a, activation="silu"))
    for x, w in ((wide[:, 1, 8:264], weights[:, 16:272]), (wide[:, 2, 7:263], weights[:, 1:257]),
                 (wide[:, 0, 1:256], weights[2:, :255]), (wide[:, 1, :130], weights[:, :256].t()[:130].t())):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = layer(x, w)
        dy = torch.full((), 0.5, dtype=dt, device="cuda").expand(y.shape)
        dx, dw = torch.autograd.grad(y, [x, w], dy)
        xc, wc = (t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
                  for t in (x, w))
        yc = layer(xc, wc)
        dxc, dwc = torch.autograd.grad(yc, [xc, wc], dy.contiguous())
        assert torch.equal(y, yc) and torch.equal(dx, dxc) and torch.equal(dw, dwc)


@gpu
def test_layers_keep_leading_axes_and_empty_rows():
    dt = torch.float16
    x = normal(53, 3, 5, 64, dtype=dt).requires_grad_(True)
    w = normal(54, 48, 64, dtype=dt, scale=0.1).requires_grad_(True)
    y = ops.linear(x, w, activation="tanh", residual=normal(55, 3, 5, 48, dtype=dt))
    assert y.shape == (3, 5, 48)
    flat = ops.linear(x.reshape(15, 64), w, activation="tanh",
                      residual=normal(55, 3, 5, 48, dtype=dt).reshape(15, 48))
    assert torch.equal(y.reshape(15, 48), flat)
    assert ops.gated_linear(x[0, 0], w).shape == (24,)
    none = x.detach()[:0].requires_grad_(True)
    y = ops.linear(none, w, bias=w.detach()[:, 0].contiguous().requires_grad_(True))
    assert y.shape == (0, 5, 48)
    dw, dx = torch.autograd.grad(y.sum(), [w, none])
    assert not bool(dw.any()) and dx.shape == none.shape
    g = ops.gated_linear(none, w)
    (dw,) = torch.autograd.grad(g.sum(), w)
    assert g.shape == (0, 5, 24) and not bool(dw.any())


@gpu
def test_layers_keep_nan_and_inf_to_their_rows():
    dt = torch.bfloat16
    x = normal(56, 200, 192, dtype=dt)
    w = normal(57, 64, 192, dtype=dt, scale=0.1)
    clean = ops.linear(x, w, activation="gelu")
    x[3, 4], x[150, 0] = float("nan"), float("inf")
    y = ops.linear(x, w, activation="gelu")
    keep = [i for i in range(200) if i not in (3, 150)]
    assert bool(y[3].isnan().all()) and torch.equal(y[keep], clean[keep])
    want = torch.nn.functional.gelu((x[150:151].double() @ w.double().t()))
    assert torch.equal(y[150:151].isnan(), want.isnan())


@gpu
@pytest.mark.parametrize("gated", [False, True])
def test_layer_gradient_by_differences(gated):
    """Slope of the float64 loss along a direction, by central differences, against the kernels'
    gradients: apart by at most the gradients' own elementwise bounds (one rounding of dz and one
    of the result: 2 u of the absolute sums) and the differences' remainder."""
    rows, inputs, outputs, dt, t = 40, 96, 56, torch.float16, 2.0 ** -10
    n = 2 * outputs if gated else outputs
    x = normal(61, rows, inputs, dtype=dt).requires_grad_(True)
    w = normal(62, n, inputs, dtype=dt, scale=0.1).requires_grad_(True)
    b = normal(63, n, dtype=dt, scale=0.5).requires_grad_(True)
    c = normal(64, rows, outputs, dtype=dt)
    y = (ops.gated_linear(x, w, bias=b, activation="gelu") if gated
         else ops.linear(x, w, bias=b, activation="tanh"))
    grads = torch.autograd.grad(y, [x, w, b], c)
    dirs = [normal(65, rows, inputs).double(), normal(66, n, inputs, scale=0.1).double(),
            normal(67, n).double()]

    def loss(s):
        xs, ws, bs = (p.detach().double() + s * v for p, v in zip((x, w, b), dirs))
        z = xs @ ws.t() + bs
        y = (torch.nn.functional.gelu(z[:, :outputs]) * z[:, outputs:] if gated
             else torch.tanh(z))
        return float((y * c.double()).sum())

    slope = sum(float((g.double() * v).sum()) for g, v in zip(grads, dirs))
    third = abs(loss(2 * t) - 2 * loss(t) + 2 * loss(-t) - loss(-2 * t)) / (2 * t ** 3)
    found = (loss(t) - loss(-t)) / (2 * t)
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    if gated:
        a, da, _ = act64("gelu", z[:, :outputs])
        dz = torch.cat([c.double() * z[:, outputs:] * da, c.double() * a], 1).abs()
    else:
        dz = (c.double() * act64("tanh", z)[1]).abs()
    u = U[dt]
    room = u * (((dz @ w.detach().double().abs()) * dirs[0].abs()).sum()
                + ((dz.t() @ x.detach().double().abs()) * dirs[1].abs()).sum()
                + (dz.sum(0) * dirs[2].abs()).sum())
    assert abs(found - slope) <= 2.1 * float(room) + t * t / 6 * third * 2


# ------------------------------------------------------------------------------- behaviour
@gpu
def test_operators_run_on_the_current_stream_and_repeat_their_bits():
    dt = torch.bfloat16
    x, w = normal(71, 300, 264, dtype=dt), normal(72, 520, 264, dtype=dt, scale=0.1)
    nw, b = normal(73, 264, dtype=dt), normal(74, 520, dtype=dt)

    def step():
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, nw, b)]
        n, h = ops.rms_norm(leaves[0], leaves[2], residual=leaves[0])
        y = ops.gated_linear(n, leaves[1], bias=leaves[3])
        z = ops.linear(h, leaves[1], activation="gelu")
        return [y, z, *torch.autograd.grad(y.float().sum() + z.float().sum(), leaves)]

    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)  # work queued before the operators on their stream
        again = step()
    side.synchronize()
    for p, q in zip(first, again):
        assert torch.equal(p, q)


@gpu
def test_operators_see_what_the_kernels_before_them_wrote():
    """Launches overlap the kernel before them; every result is that of one launch at a time."""
    dt = torch.bfloat16

    def chain(pause):
        x, w = normal(87, 40, 256, dtype=dt), normal(88, 264, 256, dtype=dt, scale=0.05)
        big, nw = normal(89, 3000, 256, dtype=dt), normal(90, 256, dtype=dt)
        w2 = normal(91, 256, 264, dtype=dt, scale=0.05)
        out = []
        for i in range(30):
            w.mul_(-1.01)
            pause()
            y = ops.linear(x, w, activation="gelu")  # few rows: reads the new w
            pause()
            x = ops.linear(y, w2, residual=x)
            pause()
            z = ops.linear(big, w)
            pause()
            big, _ = ops.rms_norm(ops.linear(z, w2), nw, residual=big)
            pause()
            nw.add_(0.01)
            pause()
            out.append(x.float().sum() + big.float().sum())
        return [x, big, torch.stack(out)]

    for got, want in zip(chain(lambda: None), chain(torch.cuda.synchronize)):
        assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("rows", [3, 300])
def test_a_wait_that_gives_up_is_reported_and_leaves_the_context_usable(rows):
    lib = L.load_library()
    x, w = normal(95, rows, 640), normal(96, 512, 640, scale=0.1)
    want = ops.linear(x, w)
    torch.cuda.synchronize()
    assert lib.rune_linear_set_wait_polls(0) == L.RUNE_OK
    try:
        ops.linear(x, w)  # undefined result
        torch.cuda.synchronize()
    finally:
        lib.rune_linear_set_wait_polls(L.DEFAULT_WAIT_POLLS)
    with pytest.raises(L.RuneError, match="did not complete in time"):
        ops.linear(x, w)
    assert torch.equal(ops.linear(x, w), want)


@gpu
def test_operators_in_a_cuda_graph():
    dt = torch.float16
    x, w = normal(75, 20, 200, dtype=dt), normal(76, 96, 200, dtype=dt, scale=0.1)
    nw = normal(77, 200, dtype=dt)

    def chain():
        return ops.linear(ops.rms_norm(x, nw), w, activation="silu")

    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = chain()
    x.copy_(normal(78, 20, 200, dtype=dt))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, chain())


@gpu
def test_offsets_beyond_32_bits():
    dt = torch.bfloat16
    rows, width = 4_200_003, 520  # 2.18e9 values
    x = torch.empty(rows, width, dtype=dt, device="cuda")
    x[-70:] = normal(81, 70, width, dtype=dt)
    w = normal(82, width, dtype=dt)
    y = ops.rms_norm(x, w)
    assert torch.equal(y[-70:], ops.rms_norm(x[-70:].clone(), w))
    del y
    m = normal(83, 8, width, dtype=dt, scale=0.1)
    assert torch.equal(ops.linear(x, m, activation="silu")[-70:],
                       ops.linear(x[-70:].clone(), m, activation="silu"))
    small, up = x[:, :8], normal(84, 2 * width, 8, dtype=dt, scale=0.3)
    got = ops.gated_linear(small, up)[-70:].clone()
    assert torch.equal(got, ops.gated_linear(small[-70:].clone(), up))


@gpu
@pytest.mark.parametrize("dtype", [*NARROW, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (65, 513), (70, 24), (2000, 130)])
def test_padded_rows_are_copies_on_16_bytes(rows, width, dtype):
    base = normal(85, rows, width + 5, dtype=torch.float32).to(dtype)
    for t in (base, base[:, 3:3 + width], base[:, 1:1 + width]):
        p = ops.padded(t)
        raw, want = p.view(torch.uint8), t.contiguous().view(torch.uint8)
        assert p.shape == t.shape and torch.equal(raw, want)
        assert p.data_ptr() % 16 == 0 and p.stride(0) * p.element_size() % 16 == 0
    if dtype is not torch.float8_e4m3fn:
        x = normal(86, 9, width, dtype=dtype)
        w = base[:, 3:3 + width]
        assert torch.equal(ops.linear(x, w), ops.linear(x, ops.padded(w)))


@gpu
def test_refusals():
    x, w = normal(91, 4, 16), normal(92, 8, 16)
    f32 = x.float()
    cases = [
        (lambda: ops.linear(f32, w.float()), "float16, bfloat16 or float8"),
        (lambda: ops.linear(x, w.half()), "weight must be"),
        (lambda: ops.linear(x, w[:, :8]), "weight must have shape"),
        (lambda: ops.linear(x, w[0]), "two axes"),
        (lambda: ops.linear(x[:, :0], w[:, :0]), "none of them empty"),
        (lambda: ops.linear(x, w, bias=x[0]), "bias must have shape"),
        (lambda: ops.linear(x, w, bias=f32[0, :8]), "bias must be"),
        (lambda: ops.linear(x, w, residual=x), "residual must have shape"),
        (lambda: ops.linear(x, w, residual=torch.zeros(4, 8, dtype=x.dtype)), "must be on"),
        (lambda: ops.linear(x, w, x_scale=f32[:, 0]), "go with float8"),
        (lambda: ops.linear(x, w, out_dtype=torch.float16), "out_dtype"),
        (lambda: ops.linear(x, w, activation="relu"), "Unsupported activation"),
        (lambda: ops.gated_linear(x, w[:7]), "odd"),
        (lambda: ops.gated_linear(x, w, activation=None), "needs an activation"),
        (lambda: ops.rms_norm(x, w), "weight must have shape"),
        (lambda: ops.rms_norm(x, w[0].half()), "weight must be"),
        (lambda: ops.rms_norm(x.to(torch.float64), w[0]), "rms_norm takes"),
        (lambda: ops.rms_norm(x, w[0], residual=x.half()), "residual must be"),
        (lambda: ops.rms_norm_fp8(x.requires_grad_(True), w[0]), "no gradient"),
        (lambda: ops.quantize_fp8(x[:, :0].detach()), "cannot be empty"),
        (lambda: ops.padded(w[0]), "two axes"),
    ]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()
    x = x.detach()
    q, s = ops.quantize_fp8(x)
    p, t = ops.quantize_fp8(w)
    with pytest.raises(ValueError, match="need x_scale"):
        ops.linear(q, p)
    with pytest.raises(ValueError, match="x_scale must have shape"):
        ops.linear(q, p, x_scale=t, weight_scale=t)
    with pytest.raises(ValueError, match="no gradient"):
        ops.linear(q, p, x_scale=s, weight_scale=t,
                   bias=w[:, 0].contiguous().requires_grad_(True))
    lib = L.load_library()
    raw = L.LinearArgs(rows=4, inputs=16, outputs=8, x_stride=16, weight_stride=16,
                       dtype=L.RUNE_F32, out_dtype=L.RUNE_F32, activation=L.RUNE_ACT_NONE,
                       x=x.data_ptr(), weight=w.data_ptr(), y=x.data_ptr())
    assert lib.rune_linear(ctypes.byref(raw), None) == L.RUNE_ERR_INVALID
    raw.dtype = raw.out_dtype = L.RUNE_BF16
    raw.device = 99
    assert lib.rune_linear(ctypes.byref(raw), None) == L.RUNE_ERR_CUDA
    assert torch.equal(ops.linear(x, w), ops.linear(x, w))  # the context is as before
