"""Rows by group (rune_b200.ops): the choice of groups, the sort, the moves and the groups' layers,
against their definitions in float64.

Tolerances as in test_ops: a float32 sum of n products is off by at most n 2^-23 of the sum of their
absolute values, a result by its own rounding; dz is rounded to 16 bits once. expf and the quotient of
the choice's weights are off by 2 units of 2^-24 and the sum of k of them by k 2^-24."""

from __future__ import annotations

import ctypes
import subprocess
import textwrap

import pytest
import torch

from rune_b200 import ops
from rune_b200.runtime import library as L
from tests.helpers import ROOT
from tests.test_ops import (FUNC, NARROW, U, act64, act_err, normal, products64, rounded, within,
                            z64)

gpu = pytest.mark.gpu
ALL = [torch.float32, *NARROW]


# ------------------------------------------------------------------------------------ CPU
def test_argument_structs_match_the_header(tmp_path):
    structs = {"rune_route_args": L.RouteArgs, "rune_row_groups_args": L.RowGroupsArgs,
               "rune_group_move_args": L.GroupMoveArgs,
               "rune_grouped_linear_args": L.GroupedLinearArgs,
               "rune_grouped_linear_grad_args": L.GroupedLinearGradArgs,
               "rune_orthogonalize_args": L.OrthogonalizeArgs}
    fields = [(c, f[0]) for c, s in structs.items() for f in s._fields_]
    lines = "".join(f'printf("%zu\\n", sizeof({c}));\n' for c in structs)
    lines += "".join(f'printf("%zu\\n", offsetof({c}, {"in" if f == "input" else f}));\n'
                     for c, f in fields)
    src = tmp_path / "sizes.c"
    src.write_text(textwrap.dedent(f"""
        #include <stddef.h>
        #include <stdio.h>
        #include "{ROOT / 'include' / 'rune_b200.h'}"
        int main(void) {{ {lines} return 0; }}"""))
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    want = [ctypes.sizeof(s) for s in structs.values()]
    want += [getattr(structs[c], f).offset for c, f in fields]
    assert got == want


def test_cpu_tensors_and_unknown_activations_are_refused():
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    index = torch.zeros(2, dtype=torch.int32)
    groups = ops.RowGroups(torch.zeros(2, dtype=torch.int32), index, index)
    w = torch.zeros(1, 4, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.route(x, 1), lambda: ops.row_groups(index, 1),
                 lambda: ops.to_groups(x, groups), lambda: ops.from_groups(x, groups),
                 lambda: ops.grouped_linear(x, w, groups),
                 lambda: ops.grouped_gated_linear(x, w, groups), lambda: ops.orthogonalize(x)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="Unsupported activation"):
        ops.grouped_linear(x, w, groups, activation="relu6")
    with pytest.raises(ValueError, match="needs an activation"):
        ops.grouped_gated_linear(x, w, groups, activation=None)


def test_null_arguments_are_refused_by_the_library():
    lib = L.load_library()
    need = ctypes.c_int64(0)
    for name in ("route", "route_backward", "row_groups", "to_groups", "from_groups",
                 "from_groups_backward", "grouped_linear", "grouped_linear_backward",
                 "orthogonalize"):
        assert getattr(lib, f"rune_{name}")(None, None) == L.RUNE_ERR_INVALID
    for name in ("row_groups", "grouped_linear", "grouped_linear_backward", "orthogonalize"):
        assert getattr(lib, f"rune_{name}_workspace")(None, ctypes.byref(need)) \
            == L.RUNE_ERR_INVALID


# ----------------------------------------------------------------------------------- route
def route64(logits, k):
    """index by repeated first maxima, NaN above all; -1 where the logit is -inf"""
    v = logits.double().cpu()
    v = torch.where(v.isnan(), torch.full_like(v, 1e300), v)
    v = torch.where(v == torch.inf, torch.full_like(v, 1e299), v)
    index = torch.empty(v.shape[0], k, dtype=torch.int64)
    taken = torch.zeros_like(v, dtype=torch.bool)
    for j in range(k):
        key = torch.where(taken, torch.full_like(v, -torch.inf), v)
        key = torch.where(~taken & (v == -torch.inf), torch.full_like(v, -1e301), key)
        at = (key == key.amax(1, keepdim=True)).double().argmax(1)
        index[:, j] = at
        taken[torch.arange(len(v)), at] = True
    masked = v.gather(1, index) == -torch.inf
    return torch.where(masked, -1, index).to(logits.device), masked.to(logits.device)


def weights64(logits, index, masked):
    chosen = logits.double().gather(1, index.clamp(min=0))
    chosen = torch.where(masked, torch.full_like(chosen, -torch.inf), chosen)
    w = torch.softmax(chosen, 1)
    return torch.where(masked, torch.zeros_like(w), w)


ROUTE_SIZES = [(1, 1, 1), (1, 64, 2), (3, 7, 7), (5, 33, 4), (130, 8, 2), (9, 256, 8),
               (17, 1024, 32), (4, 1000, 1), (2000, 100, 3), (2, 513, 5), (5000, 8, 2),
               (4097, 16, 16), (4500, 3, 3), (6000, 11, 1), (0, 5, 2)]


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("rows,groups,k", ROUTE_SIZES)
def test_route_forward_and_backward(rows, groups, k, dtype):
    logits = normal(1, rows, groups, dtype=dtype, scale=2.0).requires_grad_(True)
    index, w = ops.route(logits, k)
    want, masked = route64(logits.detach(), k)
    assert index.dtype is torch.int32 and torch.equal(index.long(), want)
    w64 = weights64(logits.detach(), want, masked)
    within(w.detach(), w64, (k + 8) * 2.0 ** -24 * w64, "weights")
    g = normal(2, rows, k, dtype=torch.float32)
    (d,) = torch.autograd.grad(w, logits, g)
    terms = w64 * g.double()
    d64 = torch.zeros(rows, groups, dtype=torch.float64, device="cuda").scatter(
        1, want, terms - w64 * terms.sum(1, keepdim=True))
    scale = torch.zeros_like(d64).scatter(
        1, want, terms.abs() + w64 * terms.abs().sum(1, keepdim=True))
    within(d, d64, 2 * (k + 12) * 2.0 ** -24 * scale + U[dtype] * d64.abs() * 1.01, "dlogits")


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("rows", [9, 5000])
def test_route_ties_masks_and_special_values(dtype, rows):
    inf, nan, low = torch.inf, torch.nan, torch.finfo(dtype).min
    table = torch.tensor([
        [1.0, 1.0, 1.0, 1.0, 1.0], [0.0, -0.0, 0.0, -0.0, 0.0], [-inf] * 5,
        [-inf, 2.0, -inf, 1.0, -inf], [low] * 5, [low, -inf, 3.0, low, -inf],
        [1.0, nan, 2.0, nan, 0.0], [inf, 0.0, 1.0, -inf, 2.0], [-1.0, -2.0, -1.0, -3.0, -2.0],
    ], dtype=dtype, device="cuda")
    logits = table[torch.arange(rows, device="cuda") % 9].requires_grad_(True)
    index, w = ops.route(logits, 3)
    repeat = torch.arange(rows, device="cuda") % 9
    assert torch.equal(index, index[:9][repeat])
    assert torch.equal(w.nan_to_num(-1.0), w[:9][repeat].nan_to_num(-1.0))
    assert index[:9].tolist() == [[0, 1, 2], [0, 1, 2], [-1] * 3, [1, 3, -1], [0, 1, 2], [2, 0, 3],
                              [1, 3, 2], [0, 4, 2], [0, 2, 1]]
    third = 3 * [pytest.approx(1 / 3, rel=1e-6)]
    got = w.tolist()
    assert got[0] == third and got[1] == third and got[4] == third
    assert got[2] == [0.0] * 3 and got[5] == [1.0, 0.0, 0.0]
    assert got[3] == [pytest.approx(0.7310585786, rel=1e-6),
                      pytest.approx(0.2689414214, rel=1e-6), 0.0]
    assert all(v != v for v in got[6]) and all(v != v for v in got[7])
    (d,) = torch.autograd.grad(w, logits, torch.ones_like(w))
    assert d[2].tolist() == [0.0] * 5 and bool(d[[0, 1, 3, 4, 5, 8]].isfinite().all())


@gpu
def test_route_strides_and_a_gradient_by_differences():
    base = normal(3, 12, 3, 50, dtype=torch.float32)
    x = base[:, 1, 3:43]
    a, b = ops.route(x, 4), ops.route(x.contiguous(), 4)
    t = x.t().contiguous().t()
    c = ops.route(t, 4)
    for other in (b, c):
        assert torch.equal(a[0], other[0]) and torch.equal(a[1], other[1])
    # central differences of the kernel's weights against its gradient, the choice unchanged: step
    # h leaves h^2 / 6 of a third derivative of at most 6 per unit of direction, and 2^-22 / h
    logits = x.clone().requires_grad_(True)
    index, w = ops.route(logits, 4)
    g, v = normal(4, 12, 4, dtype=torch.float32), normal(5, 12, 40, dtype=torch.float32)
    (d,) = torch.autograd.grad(w, logits, g)
    h = 2.0 ** -7
    up, down = ops.route(x + h * v, 4), ops.route(x - h * v, 4)
    same = ((up[0] == index) & (down[0] == index)).all(1)
    assert int(same.sum()) >= 4
    slope = (d.double() * v.double()).sum(1)
    found = ((up[1].double() - down[1].double()) * g.double()).sum(1) / (2 * h)
    size = v.double().abs().amax(1) ** 3 * g.double().abs().sum(1)
    assert bool(((found - slope).abs()[same] <= (h * h * size + 2.0 ** -22 / h
                                                 * g.double().abs().sum(1))[same]).all())


# ------------------------------------------------------------------------------------ sort
def groups64(index, groups):
    flat = index.reshape(-1).cpu().tolist()
    order = sorted((i for i, g in enumerate(flat) if 0 <= g < groups), key=lambda i: (flat[i], i))
    offsets = [sum(1 for i in order if flat[i] < g) for g in range(groups + 1)] \
        if groups < 100 else None
    place = [-1] * len(flat)
    for p, i in enumerate(order):
        place[i] = p
    if offsets is None:
        counts = [0] * (groups + 1)
        for i in order:
            counts[flat[i] + 1] += 1
        offsets = [sum(counts[:g + 1]) for g in range(groups + 1)]
    return offsets, order + [-1] * (len(flat) - len(order)), place


def choice(seed, rows, k, groups, wrong=0.0, dtype=torch.int32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (rows,) if k == 0 else (rows, k)
    u = torch.rand(shape, generator=gen, device="cuda")
    index = (groups * u * u).to(dtype).clamp(max=groups - 1)  # the first ones more often
    if wrong:
        bad = torch.rand(shape, generator=gen, device="cuda") < wrong
        other = torch.randint(0, 3, shape, generator=gen, device="cuda")
        values = torch.tensor([-1, groups, torch.iinfo(dtype).min], dtype=dtype, device="cuda")
        index = torch.where(bad, values[other], index)
    return index


SORT_SIZES = [(0, 0, 3), (1, 0, 1), (1, 2, 64), (5, 3, 4), (33, 1, 1024), (1000, 2, 7),
              (16384, 0, 89), (16385, 0, 3), (8193, 2, 1000), (70001, 3, 300), (300000, 0, 1024)]


@gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("rows,k,groups", SORT_SIZES)
@pytest.mark.parametrize("wrong", [0.0, 0.3, 1.1])
def test_row_groups(rows, k, groups, wrong, dtype):
    index = choice(11, rows, k, groups, wrong, dtype)
    got = ops.row_groups(index, groups)
    offsets, order, place = groups64(index, groups)
    assert [t.dtype for t in got] == [torch.int32] * 3
    assert got.place.shape == index.shape
    assert got.offsets.tolist() == offsets
    assert got.order.tolist() == order
    assert got.place.reshape(-1).tolist() == place


@gpu
def test_row_groups_takes_strided_indexes():
    base = choice(12, 40, 6, 9)
    for index in (base[:, ::2], base.t()[:3], base[::3, 1]):
        a, b = ops.row_groups(index, 9), ops.row_groups(index.contiguous(), 9)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ----------------------------------------------------------------------------------- moves
MOVE_SIZES = [(0, 2, 3, 8), (1, 0, 1, 1), (5, 2, 64, 4096), (7, 3, 4, 33), (130, 2, 8, 256),
              (65, 8, 16, 72), (40, 32, 64, 6), (999, 1, 89, 515), (33, 5, 7, 8200), (3000, 0, 3, 2)]


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("rows,k,groups,width", MOVE_SIZES)
@pytest.mark.parametrize("wrong", [0.0, 0.4])
def test_moves_forward_and_backward(rows, k, groups, width, wrong, dtype):
    index = choice(21, rows, k, groups, wrong)
    g = ops.row_groups(index, groups)
    slots = index.numel()
    x = normal(22, rows, width, dtype=dtype).requires_grad_(True)
    y = normal(23, slots, width, dtype=dtype).requires_grad_(True)
    w = normal(24, *index.shape, dtype=torch.float32).requires_grad_(True)
    dxs, dout = normal(25, slots, width, dtype=dtype), normal(26, rows, width, dtype=dtype)
    u, n = U[dtype], max(k, 1)
    place = g.place.long().reshape(rows, n)
    inside = place >= 0
    held = g.order >= 0
    row_of = torch.where(held, g.order.long() // n, 0)

    def zero_where(t, keep):
        return torch.where(keep, t, torch.zeros((), dtype=t.dtype, device="cuda"))

    def gathered(t):  # [rows, n, width]
        if slots == 0:
            return t.new_zeros(rows, n, width)
        return zero_where(t[place.clamp(min=0)], inside[..., None])

    xs = ops.to_groups(x, g)
    assert torch.equal(xs, zero_where(x.detach()[row_of], held[:, None]) if slots else xs)
    (dx,) = torch.autograd.grad(xs, x, dxs)
    parts = gathered(dxs.double())
    within(dx, parts.sum(1), n * 2.0 ** -24 * parts.abs().sum(1) + u * parts.sum(1).abs() * 1.01,
           "dx")
    # back, with and without weights
    for weights in (w, None):
        out = ops.from_groups(y, g, weights)
        w64 = (w.detach().double().reshape(rows, n) if weights is not None
               else torch.ones(rows, n, dtype=torch.float64, device="cuda"))
        parts = gathered(y.detach().double()) * w64[..., None]
        within(out.detach(), parts.sum(1),
               (n + 1) * 2.0 ** -24 * parts.abs().sum(1) + u * parts.sum(1).abs() * 1.01, "out")
        grads = torch.autograd.grad(out, [y] + ([w] if weights is not None else []), dout)
        slot_w = zero_where(w64.reshape(-1)[torch.where(held, g.order.long(), 0)], held) \
            if slots else w64.reshape(-1)
        dy64 = dout.double()[row_of] * slot_w[:, None] if slots else y.detach().double()
        within(grads[0], dy64, (u * 1.01 + 2.0 ** -24) * dy64.abs(), "dy")
        if weights is not None:
            terms = gathered(y.detach().double()) * dout.double()[:, None]
            within(grads[1].reshape(rows, n), terms.sum(-1),
                   (width + 2) * 2.0 ** -24 * terms.abs().sum(-1), "dweights")
    if slots and rows:
        # one gradient alone is the same
        out = ops.from_groups(y.detach(), g, w)
        (dw,) = torch.autograd.grad(out, w, dout)
        assert torch.equal(dw, torch.autograd.grad(ops.from_groups(y, g, w), [y, w], dout)[1])
        out = ops.from_groups(y, g, w.detach())
        (dy,) = torch.autograd.grad(out, y, dout)
        assert torch.equal(dy, torch.autograd.grad(ops.from_groups(y, g, w), [y, w], dout)[0])


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_moves_strides_and_what_lies_behind(dtype):
    """Views give the bits of their copies; rows in no group may hold anything."""
    index = choice(31, 50, 2, 5, 0.3)
    g = ops.row_groups(index, 5)
    w = normal(32, 50, 2, dtype=torch.float32)
    base, wide = normal(33, 50, 3, 90, dtype=dtype), normal(34, 100, 200, dtype=dtype)
    for x, y in ((base[:, 1, 8:72], wide[:, 16:80]), (base[:, 0, 1:65], wide[:, 3:67]),
                 (base[:, 2, :63], wide[:, :63]), (base[:, :, 4], wide.t()[:100, 5:8])):
        assert torch.equal(ops.to_groups(x, g), ops.to_groups(x.contiguous(), g))
        y = y.detach().clone().as_strided(y.shape, y.stride()) if y.is_contiguous() else y
        assert torch.equal(ops.from_groups(y, g, w), ops.from_groups(y.contiguous(), g, w))
    y = wide[:, :64].contiguous()
    total = int(g.offsets[-1])
    assert total < 100
    spoiled = y.clone()
    spoiled[total:] = float("nan")
    ws = w.clone()
    ws[g.place < 0] = float("nan")
    a = [t.requires_grad_(True) for t in (spoiled, ws)]
    b = [t.requires_grad_(True) for t in (y, w)]
    dout = normal(35, 50, 64, dtype=dtype)
    outs = [ops.from_groups(t[0], g, t[1]) for t in (a, b)]
    assert torch.equal(*outs)
    grads = [torch.autograd.grad(o, t, dout) for o, t in zip(outs, (a, b))]
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])
    assert not bool(grads[0][0][total:].any()) and not bool(grads[0][1][g.place < 0].any())
    # a broadcast gradient
    x = base[:, 1, :64].detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.to_groups(x, g).sum(), x)
    assert torch.equal(dx, (g.place >= 0).sum(1, keepdim=True).to(dtype).expand(50, 64))


# ---------------------------------------------------------------------------------- layers
def by_sizes(sizes, behind=0):
    """RowGroups of rows that are sorted already, `behind` of them in no group"""
    total = sum(sizes)
    index = torch.tensor([g for g, n in enumerate(sizes) for _ in range(n)] + [-1] * behind,
                         dtype=torch.int32, device="cuda")
    g = ops.row_groups(index, len(sizes))
    assert int(g.offsets[-1]) == total
    return g, index.long()


GROUP_SIZES = [([1], 0, 8, 8), ([0, 0], 3, 16, 8), ([3, 0, 5], 0, 1, 1), ([1] * 7, 2, 100, 36),
               ([40, 9, 0, 1], 6, 513, 96), ([127, 1, 128, 129, 0], 0, 64, 128),
               ([300, 77, 260], 31, 129, 255), ([64] * 5, 0, 256, 64), ([0, 700, 1, 0], 5, 72, 520),
               ([5] * 100, 0, 40, 24), ([513, 255, 1025], 0, 136, 264), ([0] * 30 + [200], 0, 35, 30),
               ([2100, 3], 1, 320, 200), ([97, 300, 255, 256, 1, 33, 600], 9, 520, 504),
               ([129, 0, 640, 225], 3, 1030, 235), ([3000, 1, 2500, 0, 4097], 7, 256, 512)]


def per_group(fn, index, groups, *tensors):
    """fn(tensors' rows of the group, g) for each group, put together; zeros in no group"""
    parts = []
    for g in range(groups):
        rows = index == g
        parts.append(fn(g, *(t[rows] for t in tensors)))
    return parts


@gpu
@pytest.mark.parametrize("dtype", NARROW, ids=str)
@pytest.mark.parametrize("sizes,behind,inputs,outputs", GROUP_SIZES)
@pytest.mark.parametrize("act,with_bias,gated", [
    (None, False, False), (None, True, False), ("tanh", True, False), ("gelu", False, False),
    ("silu", True, True), ("gelu", False, True)])
def test_grouped_layers(sizes, behind, inputs, outputs, dtype, act, with_bias, gated):
    n, u, count = outputs * (2 if gated else 1), U[dtype], len(sizes)
    g, index = by_sizes(sizes, behind)
    rows = len(index)
    x = normal(41, rows, inputs, dtype=dtype).requires_grad_(True)
    w = normal(42, count, n, inputs, dtype=dtype, scale=inputs ** -0.5).requires_grad_(True)
    b = normal(43, count, n, dtype=dtype, scale=0.5).requires_grad_(True) if with_bias else None
    dy = normal(44, rows, outputs, dtype=dtype)
    call = ops.grouped_gated_linear if gated else ops.grouped_linear
    y = call(x, w, g, bias=b, activation=act)
    with torch.no_grad():
        assert torch.equal(y, call(x, w, g, bias=b, activation=act))
    grads = torch.autograd.grad(y, [x, w] + ([b] if with_bias else []), dy)
    end = sum(sizes)
    assert not bool(y[end:].any()) and not bool(grads[0][end:].any())
    at = 0
    for i, size in enumerate(sizes):
        part = slice(at, at + size)
        at += size
        if size == 0:
            assert not bool(grads[1][i].any())
            assert not with_bias or not bool(grads[2][i].any())
            continue
        xg, wg, bg = x.detach()[part], w.detach()[i], None if b is None else b.detach()[i]
        z, ez = z64(xg, wg, bg)
        d = dy[part].double()
        if gated:
            gate, up = z[:, :outputs], z[:, outputs:]
            eg, eu = ez[:, :outputs], ez[:, outputs:]
            a, da, _ = act64(act, gate)
            ea, eda = act_err(act, gate, eg)
            want = a * up
            ey = ea * (up.abs() + eu) + a.abs() * eu
            dz = torch.cat([d * up * da, d * a], 1)
            ddz = torch.cat([d.abs() * (eda * (up.abs() + eu) + da.abs() * eu), d.abs() * ea], 1)
        else:
            want, da, _ = act64(act, z)
            ey, eda = act_err(act, z, ez)
            dz, ddz = d * da, d.abs() * eda
        within(y.detach()[part], *rounded((want, ey + 2.0 ** -23 * want.abs()), u), "y")
        plain = act is None
        ddz = torch.zeros_like(dz) if plain else ddz + 2.0 ** -22 * dz.abs()
        pairs = products64(dz, ddz, xg, wg, 0.0 if plain else u, size)
        within(grads[0][part], *rounded(pairs[0], u), "dx")
        within(grads[1][i], *rounded(pairs[1], u), "dweight")
        if with_bias:
            within(grads[2][i], *rounded(pairs[2], u), "dbias")


@gpu
@pytest.mark.parametrize("dtype", NARROW, ids=str)
@pytest.mark.parametrize("gated", [False, True])
def test_saved_z_in_long_and_short_groups(dtype, gated):
    """Long groups, an empty one and some of a row or two, with a saved z."""
    test_grouped_layers([5000, 1, 0, 15, 4001, 2, 2, 2], 3, 1040, 24, dtype, "silu", True, gated)


@gpu
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_layers_keep_groups_apart(gated):
    """A group's infinities and NaN, and whatever rows in no group hold, stay out of the others."""
    dt = torch.bfloat16
    g, index = by_sizes([70, 33, 129, 5], 40)
    n = 96 if gated else 48
    call = ops.grouped_gated_linear if gated else ops.grouped_linear
    x, w = normal(51, 277, 72, dtype=dt), normal(52, 4, n, 72, dtype=dt, scale=0.1)
    b, dy = normal(53, 4, n, dtype=dt), normal(54, 277, 48, dtype=dt)
    xs, ws, bs, ds = x.clone(), w.clone(), b.clone(), dy.clone()
    xs[index == 1], ds[index == 1] = float("nan"), float("inf")
    ws[1], bs[1] = float("inf"), float("nan")
    xs[index < 0], ds[index < 0] = float("nan"), float("nan")
    got = []
    for t in ((x, w, b, dy), (xs, ws, bs, ds)):
        leaves = [v.detach().clone().requires_grad_(True) for v in t[:3]]
        y = call(leaves[0], leaves[1], g, bias=leaves[2], activation="silu")
        got.append([y.detach(), *torch.autograd.grad(y, leaves, t[3])])
    rows, keep = (index >= 0) & (index != 1), [0, 2, 3]
    for a, c, rowwise in zip(*got, (True, True, False, False)):
        if rowwise:
            assert torch.equal(a[rows], c[rows]) and not bool(c[index < 0].any())
        else:
            assert torch.equal(a[keep], c[keep]) and bool(c[1].float().isnan().any())


@gpu
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_layers_with_strides(gated):
    dt = torch.float16
    g, index = by_sizes([30, 0, 170], 3)
    base, weights = normal(61, 203, 3, 400, dtype=dt), normal(62, 3, 140, 700, dtype=dt, scale=0.1)
    call = ops.grouped_gated_linear if gated else ops.grouped_linear
    for x, w in ((base[:, 1, 8:264], weights[:, :, 16:272]), (base[:, 2, 7:263], weights[:, :, 1:257]),
                 (base[:, 0, 1:256], weights[:, 2:132, :255]),
                 (base[:, 1, :130], weights[:, :, :130].transpose(1, 2)[:, :, :130])):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = call(x, w, g, activation="tanh")
        dy = torch.full((), 0.5, dtype=dt, device="cuda").expand(y.shape)
        got = torch.autograd.grad(y, [x, w], dy)
        xc, wc = (t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
                  for t in (x, w))
        yc = call(xc, wc, g, activation="tanh")
        want = torch.autograd.grad(yc, [xc, wc], dy.contiguous())
        assert torch.equal(y, yc) and all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_wrong_groups_reach_no_memory():
    """RowGroups that a caller made wrong select rows inside the tensors or none."""
    dt = torch.bfloat16
    x, w = normal(71, 20, 16, dtype=dt), normal(72, 2, 8, 16, dtype=dt)

    def i32(*v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    place = i32(*range(20))
    for offsets in (i32(-5, 7, 900), i32(10, 4, 20), i32(2 ** 31 - 1, -2 ** 31, 3)):
        y = ops.grouped_linear(x, w, ops.RowGroups(offsets, place, place))
        assert y.shape == (20, 8)
    wrong = i32(*(-7, 2 ** 31 - 1, 20, *range(17)))
    g = ops.RowGroups(i32(0, 20, 20), wrong, wrong)
    xs = ops.to_groups(x, g)
    assert not bool(xs[:3].any()) and torch.equal(xs[3:], x[:17])
    out = ops.from_groups(x, g)
    assert not bool(out[:3].any()) and torch.equal(out[3:], x[:17])
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("rows,groups,inputs,outputs", [(600, 64, 64, 96), (20000, 40, 72, 64),
                                                        (3000, 1024, 16, 8)])
@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("saved", [False, True])
def test_offsets_out_of_order_reach_no_memory(rows, groups, inputs, outputs, gated, saved):
    """Groups that overlap, each of all rows: more lines of tiles than offsets in order lead to. What
    lies behind the workspace and the results stays as it was."""
    lib = L.load_library()
    dt, guard = torch.bfloat16, 1 << 16
    n_all = (2 if gated else 1) * outputs
    x, w = normal(73, rows, inputs, dtype=dt), normal(74, groups, n_all, inputs, dtype=dt)
    bias, dy = normal(75, groups, n_all, dtype=dt), normal(76, rows, outputs, dtype=dt)
    offsets = torch.tensor([0, rows] * (groups // 2) + [0], dtype=torch.int32, device="cuda")
    line = (outputs + 3) // 4 * 4
    z = normal(77, rows, (2 if gated else 1) * line, dtype=torch.float32)

    def room(size):
        return torch.full((size + guard,), 0x5A, dtype=torch.uint8, device="cuda")

    def kept(t, size):
        return bool((t[size:] == 0x5A).all())

    sizes = [2 * rows * inputs, 2 * w.numel(), 2 * bias.numel(), 2 * rows * outputs]
    dx, dw, db, y = (room(n) for n in sizes)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    need = ctypes.c_int64(0)
    common = dict(rows=rows, inputs=inputs, outputs=outputs, groups=groups, x_stride=inputs,
                  weight_stride=inputs, device=0, dtype=L.RUNE_BF16,
                  activation=L.RUNE_ACT["silu"], gated=gated, x=x.data_ptr(), weight=w.data_ptr(),
                  bias=bias.data_ptr(), offsets=offsets.data_ptr())
    calls = [("grouped_linear", L.GroupedLinearArgs(**common, y=y.data_ptr()), [(y, sizes[3])]),
             ("grouped_linear_backward", L.GroupedLinearGradArgs(
                 **common, dy_stride=outputs, dy=dy.data_ptr(), dx=dx.data_ptr(),
                 dweight=dw.data_ptr(), dbias=db.data_ptr(), saved=z.data_ptr() if saved else None),
              list(zip((dx, dw, db), sizes)))]
    for name, args, results in calls:
        assert getattr(lib, f"rune_{name}_workspace")(ctypes.byref(args), ctypes.byref(need)) == 0
        ws = room(need.value)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need.value
        assert getattr(lib, f"rune_{name}")(ctypes.byref(args), stream) == 0
        torch.cuda.synchronize()
        assert kept(ws, need.value), name
        assert all(kept(t, n) for t, n in results), name


@gpu
def test_refusals():
    dt = torch.bfloat16
    x, w = normal(81, 6, 16, dtype=dt), normal(82, 3, 8, 16, dtype=dt)
    index = choice(83, 6, 0, 3)
    g = ops.row_groups(index, 3)
    pair = ops.row_groups(choice(84, 6, 2, 3), 3)
    cases = [
        (lambda: ops.route(x[0], 1), "two axes"), (lambda: ops.route(x, 0), "k must be"),
        (lambda: ops.route(x, 17), "k must be"), (lambda: ops.route(x.double(), 1), "float32"),
        (lambda: ops.row_groups(x, 3), "int32 or int64"),
        (lambda: ops.row_groups(index, 0), "1 to 1024"),
        (lambda: ops.row_groups(index, 1025), "1 to 1024"),
        (lambda: ops.row_groups(index[None, None], 3), "shape"),
        (lambda: ops.to_groups(x[:5], g), "rows"), (lambda: ops.to_groups(x[None], g), "two axes"),
        (lambda: ops.to_groups(x.double(), g), "float32"),
        (lambda: ops.to_groups(x, g._replace(order=g.order[:5])), "row_groups"),
        (lambda: ops.to_groups(x, g._replace(place=g.place.long())), "int32"),
        (lambda: ops.to_groups(x, g._replace(place=g.place.cpu())), "int32"),
        (lambda: ops.from_groups(x, pair), "slots"),
        (lambda: ops.from_groups(x, g, index.float()[:5]), "shape"),
        (lambda: ops.from_groups(x, g, index.to(dt)), "float32"),
        (lambda: ops.grouped_linear(x.float(), w.float(), g), "float16 or bfloat16"),
        (lambda: ops.grouped_linear(x, w.half(), g), "bfloat16"),
        (lambda: ops.grouped_linear(x, w[:2], g), "shape"),
        (lambda: ops.grouped_linear(x, w[0], g), "three"),
        (lambda: ops.grouped_linear(x[:5], w, g), "slots"),
        (lambda: ops.grouped_linear(x, w, g, bias=w[:, 0]), "shape"),
        (lambda: ops.grouped_gated_linear(x, w[:, :7], g), "odd"),
    ]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(TypeError):
        ops.to_groups([1], g)
    leaf = x.clone().requires_grad_(True)
    for call in (lambda: ops.to_groups(leaf, g), lambda: ops.grouped_linear(leaf, w, g),
                 lambda: ops.route(leaf, 2)[1], lambda: ops.from_groups(leaf, g)):
        y = call()
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)


# -------------------------------------------------------------------------------- together
def experts(x, router, w0, b0, w1, b1, k, act="silu"):
    """a mixture of gated experts as a network calls it"""
    count = w0.shape[0]
    index, weights = ops.route(ops.linear(x, router), k)
    g = ops.row_groups(index, count)
    h = ops.grouped_gated_linear(ops.to_groups(x, g), w0, g, bias=b0, activation=act)
    return ops.from_groups(ops.grouped_linear(h, w1, g, bias=b1), g, weights), index


@gpu
@pytest.mark.parametrize("rows,hidden,ffn,count,k", [(1, 64, 32, 4, 2), (37, 72, 40, 7, 3),
                                                     (700, 256, 128, 16, 2)])
def test_mixture_of_experts_forward_and_gradients(rows, hidden, ffn, count, k):
    """The run of all operators against float64 for the same choice. Each stage rounds to bfloat16
    once; the relative error of each result is compared in norm, where roundings of 2^-9 each (root
    mean square 2^-8 / sqrt(3) at most) of at most 12 stages of roundings add up below 12 * 2^-8."""
    dt = torch.bfloat16
    leaves = [normal(91, rows, hidden, dtype=dt), normal(92, count, hidden, dtype=dt, scale=0.2),
              normal(93, count, 2 * ffn, hidden, dtype=dt, scale=hidden ** -0.5),
              normal(94, count, 2 * ffn, dtype=dt, scale=0.3),
              normal(95, count, hidden, ffn, dtype=dt, scale=ffn ** -0.5),
              normal(96, count, hidden, dtype=dt, scale=0.3)]
    leaves = [t.requires_grad_(True) for t in leaves]
    out, index = experts(*leaves, k)
    dout = normal(97, rows, hidden, dtype=dt)
    grads = torch.autograd.grad(out, leaves, dout)
    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    x, router, w0, b0, w1, b1 = ref
    logits = x @ router.t()
    weights = torch.softmax(logits.gather(1, index.long()), 1)
    want = torch.zeros_like(x)
    for j in range(k):
        e = index[:, j].long()
        z = torch.einsum("rh,rfh->rf", x, w0[e]) + b0[e]
        h = torch.nn.functional.silu(z[:, :ffn]) * z[:, ffn:]
        want = want + weights[:, j:j + 1] * (torch.einsum("rf,rhf->rh", h, w1[e]) + b1[e])
    wanted = torch.autograd.grad(want, ref, dout.double())
    for name, a, b in zip(("out", "dx", "drouter", "dw0", "db0", "dw1", "db1"),
                          (out.detach(), *grads), (want.detach(), *wanted)):
        apart = float((a.double() - b).norm() / b.norm())
        assert apart <= 12 * 2.0 ** -8, (name, apart)


@gpu
def test_captured_graph_replays_with_other_sizes_of_groups():
    """The groups' sizes are the GPU's own: one captured run serves every choice."""
    dt = torch.bfloat16
    rows, hidden, ffn, count, k = 90, 64, 48, 6, 2
    args = [normal(101, rows, hidden, dtype=dt), normal(102, count, hidden, dtype=dt),
            normal(103, count, 2 * ffn, hidden, dtype=dt, scale=0.1),
            normal(104, count, 2 * ffn, dtype=dt), normal(105, count, hidden, ffn, dtype=dt),
            normal(106, count, hidden, dtype=dt)]
    params = [t.requires_grad_(True) for t in args]
    dout = normal(107, rows, hidden, dtype=dt)

    def step():
        out, index = experts(*params, k)
        return (out, index, *torch.autograd.grad(out, params, dout))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (108, 109, 110):
        with torch.no_grad():
            params[0].copy_(normal(seed, rows, hidden, dtype=dt))
            params[1].copy_(normal(seed + 50, count, hidden, dtype=dt, scale=0.1 * (seed - 107)))
        graph.replay()
        got = [t.detach().clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b.detach())
    torch.cuda.synchronize()
    ops.check_waits()


@gpu
def test_other_streams_at_once():
    dt = torch.bfloat16
    g, _ = by_sizes([200, 0, 313, 64], 7)
    x, w = normal(111, 584, 128, dtype=dt), normal(112, 4, 192, 128, dtype=dt, scale=0.1)
    want = ops.grouped_linear(x, w, g, activation="gelu")
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.grouped_linear(x, w, g, activation="gelu"))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


@gpu
@pytest.mark.parametrize("polls", [0, 1, 7])
def test_a_wait_that_gives_up_is_reported(polls):
    lib = L.load_library()
    dt = torch.bfloat16
    g, _ = by_sizes([300, 513, 1, 0, 700], 9)
    x = normal(121, 1523, 256, dtype=dt).requires_grad_(True)
    w = normal(122, 5, 384, 256, dtype=dt, scale=0.1).requires_grad_(True)
    y = ops.grouped_linear(x, w, g, activation="silu")
    want = [y.detach(), *torch.autograd.grad(y, [x, w], torch.ones_like(y))]
    torch.cuda.synchronize()
    try:
        lib.rune_linear_set_wait_polls(polls)
        ops.grouped_linear(x.detach(), w.detach(), g, activation="silu")
        torch.cuda.synchronize()
        reported = False
        try:
            ops.check_waits()
        except L.RuneError:
            reported = True
        assert reported or polls > 0
    finally:
        lib.rune_linear_set_wait_polls(L.DEFAULT_WAIT_POLLS)
    y = ops.grouped_linear(x, w, g, activation="silu")
    got = [y.detach(), *torch.autograd.grad(y, [x, w], torch.ones_like(y))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("sizes,inputs,outputs", [
    ([5000, 0, 1, 63, 64, 65, 9000], 35, 30), ([30000], 64, 24), ([0, 20011, 0], 136, 200),
    ([1, 2, 40000], 512, 520), ([700] * 40, 300, 264), ([2] * 900 + [3000], 24, 16)])
def test_weight_gradients_over_long_groups(sizes, inputs, outputs):
    """Groups whose rows many blocks share, and groups that end inside a block's range."""
    dt, u = torch.bfloat16, U[torch.bfloat16]
    g, index = by_sizes(sizes, 3)
    rows = len(index)
    x, dy = normal(131, rows, inputs, dtype=dt), normal(132, rows, outputs, dtype=dt)
    w = normal(133, len(sizes), outputs, inputs, dtype=dt, scale=inputs ** -0.5)
    b = normal(134, len(sizes), outputs, dtype=dt)
    w, b = w.requires_grad_(True), b.requires_grad_(True)
    dw, db = torch.autograd.grad(ops.grouped_linear(x, w, g, bias=b), [w, b], dy)
    at = 0
    for i, n in enumerate(sizes):
        d, part = dy[at:at + n].double(), x[at:at + n].double()
        at += n
        s = d.abs().t() @ part.abs()
        within(dw[i], d.t() @ part, *[(n + 2) * 2.0 ** -23 * s + u * (d.t() @ part).abs() * 1.01],
               "dweight")
        within(db[i], d.sum(0), (n + 2) * 2.0 ** -23 * d.abs().sum(0) + u * d.sum(0).abs() * 1.01,
               "dbias")
    again = torch.autograd.grad(ops.grouped_linear(x, w, g, bias=b), [w, b], dy)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


@gpu
def test_weight_gradients_keep_to_their_groups_wherever_the_operands_lie():
    """Operands at other addresses in each pass, and groups of other sizes."""
    gen = torch.Generator().manual_seed(7)
    for rows, inputs, outputs, count in ((2000, 64, 283, 31), (700, 72, 520, 5), (900, 1040, 24, 8)):
        held = []
        for turn in range(12):
            index = torch.randint(0, count, (rows,), generator=gen).sort().values.cuda()
            g = ops.row_groups(index, count)
            x, w = normal(161, rows, inputs, dtype=torch.float16).requires_grad_(True), \
                normal(162, count, outputs, inputs, dtype=torch.float16).requires_grad_(True)
            dy = normal(163, rows, outputs, dtype=torch.float16)
            dx, dw = torch.autograd.grad(ops.grouped_linear(x, w, g), [x, w], dy)
            held.append(torch.empty(100_000 + 4096 * turn, dtype=torch.uint8, device="cuda"))
            for i in range(count):
                part = index == i
                d, xs = dy[part].double(), x.detach()[part].double()
                pairs = products64(d, torch.zeros_like(d), xs, w.detach()[i], 0.0, rows)
                within(dw[i], *rounded(pairs[1], U[torch.float16]), "dweight")
        del held
        torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("count,size,inputs,outputs", [(40, 1650, 16, 128), (89, 1500, 35, 30),
                                                       (32, 2050, 64, 1024)])
def test_bias_gradients_of_many_long_groups(count, size, inputs, outputs):
    """More columns of all groups than the weights' tiles have blocks for."""
    test_weight_gradients_over_long_groups([size + 7 * i for i in range(count)], inputs, outputs)


@gpu
def test_offsets_beyond_32_bits():
    """Rows whose values start behind the 2^31st, spot-checked."""
    dt = torch.bfloat16
    rows, width = 70_000, 40_000
    x = torch.empty(rows, width, dtype=dt, device="cuda")
    for at in range(0, rows, 10_000):
        x[at:at + 10_000] = normal(at, 10_000, width, dtype=dt)
    g = ops.row_groups(torch.arange(rows, device="cuda", dtype=torch.int32) % 3, 3)
    xs = ops.to_groups(x, g)
    some = torch.tensor([0, 1, 2, 54_000, 69_997, 69_998, 69_999], device="cuda")
    assert torch.equal(xs[g.place.long()[some]], x[some])
    back = ops.from_groups(xs, g)
    assert torch.equal(back[some], x[some]) and torch.equal(back[53_680:53_700], x[53_680:53_700])
    w = torch.full((rows,), 2.0, device="cuda").requires_grad_(True)
    out = ops.from_groups(xs, g, w)
    (dw,) = torch.autograd.grad(out, w, back)
    want = (x[some].double() ** 2).sum(1)
    assert bool(((dw[some].double() - want).abs() <= (width + 2) * 2.0 ** -24 * want).all())
    del xs, back, out
    # and a layer's results
    rows, outputs = 280_000, 8_192
    sizes = [100_000, 0, 179_999]
    g, index = by_sizes(sizes, 1)
    x, w = normal(141, rows, 64, dtype=dt), normal(142, 3, outputs, 64, dtype=dt, scale=0.1)
    y = ops.grouped_linear(x, w, g)
    for r in (0, 99_999, 100_000, 262_144, 279_998):
        z, err = z64(x[r:r + 1], w[int(index[r])], None)
        within(y[r:r + 1], *rounded((z, err), U[dt]), "y")
    assert not bool(y[-1].any())


@gpu
def test_threads_at_once():
    """Calls from several threads, each on its own stream."""
    import threading

    dt = torch.bfloat16
    x = normal(151, 500, 96, dtype=dt)
    w = normal(152, 5, 160, 96, dtype=dt, scale=0.1)
    index = choice(153, 500, 2, 5)
    dy = normal(154, 500, 160, dtype=dt)

    def step():
        leaf, weight = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        g = ops.row_groups(index, 5)
        y = ops.from_groups(ops.grouped_linear(ops.to_groups(leaf, g), weight, g,
                                               activation="silu"), g)
        return (y, *torch.autograd.grad(y, [leaf, weight], dy))

    want = step()
    torch.cuda.synchronize()
    got, errors = [], []

    def run():
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got.append(step())
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(got) == 40
    for result in got:
        assert all(torch.equal(a, b) for a, b in zip(result, want))


@gpu
def test_two_graphs_with_one_workspace_each():
    """Two captured training steps, replayed in turn and on two streams at once."""
    dt = torch.bfloat16
    g, _ = by_sizes([130, 70, 0, 300], 5)
    dy = normal(161, 505, 72, dtype=dt)

    def make(seed):
        x = normal(seed, 505, 64, dtype=dt).requires_grad_(True)
        w = normal(seed + 1, 4, 72, 64, dtype=dt, scale=0.1).requires_grad_(True)
        b = normal(seed + 2, 4, 72, dtype=dt).requires_grad_(True)

        def step():
            y = ops.grouped_linear(x, w, g, bias=b, activation="gelu")
            return (y, *torch.autograd.grad(y, [x, w, b], dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return graph, out, [t.detach().clone() for t in step()]

    graphs = [make(seed) for seed in (162, 172)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for (graph, _, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want in graphs:
            assert all(torch.equal(a.detach(), b) for a, b in zip(out, want))
    ops.check_waits()


@gpu
@pytest.mark.parametrize("polls", [0, 1, 3, 9, 40])
def test_waits_that_give_up_in_training_steps(polls):
    """Every kind of product of a step, among them ones turned round and over ranges of rows: whatever
    gives up, the next step with the usual bound has the usual bits."""
    lib = L.load_library()
    dt = torch.bfloat16
    g, _ = by_sizes([300, 97, 0, 1200, 513], 4)
    x = normal(181, 2114, 576, dtype=dt).requires_grad_(True)
    w0 = normal(182, 5, 512, 576, dtype=dt, scale=0.05).requires_grad_(True)
    w1 = normal(183, 5, 512, 256, dtype=dt, scale=0.05).requires_grad_(True)
    dy = normal(184, 2114, 512, dtype=dt)

    def step():
        h = ops.grouped_gated_linear(x, w0, g)
        y = ops.grouped_linear(h, w1, g, activation="tanh")
        z = ops.grouped_linear(y, w0.transpose(1, 2).contiguous(), g)
        return (z, *torch.autograd.grad([y, z], [x, w0, w1], [dy, torch.ones_like(z)]))

    want = step()
    torch.cuda.synchronize()
    try:
        lib.rune_linear_set_wait_polls(polls)
        for _ in range(3):
            try:
                step()
            except L.RuneError:
                pass
        torch.cuda.synchronize()
        try:
            ops.check_waits()
        except L.RuneError:
            pass
    finally:
        lib.rune_linear_set_wait_polls(L.DEFAULT_WAIT_POLLS)
    assert all(torch.equal(a, b) for a, b in zip(step(), want))


def every_operator(x, w, g, index):
    return [lambda a: ops.route(a, 2)[1], lambda a: ops.to_groups(a, g),
            lambda a: ops.from_groups(a, g), lambda a: ops.grouped_linear(a, w, g),
            lambda a: ops.grouped_linear(x, a[None], g),
            lambda a: ops.grouped_gated_linear(a, w, g), lambda a: ops.orthogonalize(a)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_and_traces_are_refused(device):
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.ones(16, 16, dtype=torch.bfloat16, device=device)
    index = torch.zeros(16, dtype=torch.int32, device=device)
    place = torch.arange(16, dtype=torch.int32, device=device)
    g = ops.RowGroups(torch.tensor([0, 16], dtype=torch.int32, device=device), place, place)
    for f in every_operator(x, x[None], g, index):
        with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError,
                                                                     match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(lambda a: f(a + 1), x, check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(lambda a: f(a + 1))(x)
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.vmap(f)(x[None])
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda i: ops.row_groups(i + 0, 1)[0])(index)


@gpu
def test_transforms_of_a_backward_are_refused_and_checkpoints_work():
    from torch.autograd import forward_ad
    from torch.utils.checkpoint import checkpoint

    dt = torch.bfloat16
    g, _ = by_sizes([20, 0, 41], 3)
    x = normal(191, 64, 48, dtype=dt).requires_grad_(True)
    w = normal(192, 3, 48, 48, dtype=dt, scale=0.1).requires_grad_(True)
    for y in (ops.to_groups(x, g), ops.from_groups(x, g), ops.route(x, 2)[1],
              ops.grouped_linear(x, w, g, activation="silu")):
        dy = torch.ones_like(y)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, forward_ad.make_dual(dy, dy), retain_graph=True)
        assert bool(torch.autograd.grad(y, x, dy)[0].isfinite().all())

    def block(a):
        return ops.from_groups(ops.grouped_linear(ops.to_groups(a, g), w, g, activation="gelu"), g)

    want = torch.autograd.grad(block(x).float().sum(), [x, w])
    got = torch.autograd.grad(checkpoint(block, x, use_reentrant=False).float().sum(), [x, w])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_weights_changed_between_the_passes_are_noticed():
    dt = torch.bfloat16
    g, _ = by_sizes([20, 44])
    x = normal(193, 64, 48, dtype=dt).requires_grad_(True)
    w = normal(194, 2, 48, 48, dtype=dt).requires_grad_(True)
    y = ops.grouped_linear(x, w, g, activation="silu")
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


# (rows of each group, rows in none): far fewer lines of rows in groups than blocks share among them
MOSTLY_NONE = [([1000, 700, 0], 30000, 35, 30), ([64, 65, 200], 30000, 128, 128),
               ([1124, 61, 802, 937], 26334, 128, 128), ([3000], 27000, 64, 64),
               ([3327, 4611], 71454, 64, 128), ([0, 0, 130], 40000, 35, 30), ([0, 1], 30000, 64, 64),
               ([0, 0], 30000, 128, 128)]


@gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sizes,behind,inputs,outputs", MOSTLY_NONE)
def test_gradients_where_most_rows_are_in_no_group(sizes, behind, inputs, outputs, gated):
    """A padded batch, or one rank's experts: no gradient depends on what the workspace and the results
    held before the call, or on what the rows in no group hold."""
    lib = L.load_library()
    dt, rows, groups = torch.bfloat16, sum(sizes) + behind, len(sizes)
    n_all = (2 if gated else 1) * outputs
    g, _ = by_sizes(sizes, behind)
    pad = (inputs + 7) // 8 * 8
    x = normal(201, rows, pad, dtype=dt)
    w = normal(202, groups, n_all, pad, dtype=dt, scale=inputs ** -0.5)
    dy = normal(203, rows, outputs, dtype=dt)
    x[sum(sizes):], dy[sum(sizes):] = float("nan"), float("inf")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    need = ctypes.c_int64(0)
    results = []
    for stale in (0xFF, 0x3C, 0):  # NaN, values near 0.01, zeros
        dx, dw, db = (torch.full((n,), stale, dtype=torch.uint8, device="cuda").view(dt)
                      for n in (2 * rows * inputs, 2 * groups * n_all * inputs, 2 * groups * n_all))
        args = L.GroupedLinearGradArgs(
            rows=rows, inputs=inputs, outputs=outputs, groups=groups, x_stride=pad,
            weight_stride=pad, dy_stride=outputs, device=0, dtype=L.RUNE_BF16,
            activation=L.RUNE_ACT["silu"] if gated else L.RUNE_ACT_NONE, gated=int(gated),
            x=x.data_ptr(), weight=w.data_ptr(), offsets=g.offsets.data_ptr(), dy=dy.data_ptr(),
            dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr())
        assert lib.rune_grouped_linear_backward_workspace(ctypes.byref(args), ctypes.byref(need)) == 0
        ws = torch.full((need.value,), stale, dtype=torch.uint8, device="cuda")
        args.workspace, args.workspace_bytes = ws.data_ptr(), need.value
        assert lib.rune_grouped_linear_backward(ctypes.byref(args), stream) == 0
        results.append([t.clone() for t in (dx, dw, db)])
    for t in results[0]:
        assert bool(t.isfinite().all())
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@gpu
@pytest.mark.parametrize("act,gated", [(None, False), ("tanh", False), ("silu", True)])
@pytest.mark.parametrize("sizes,behind,inputs,outputs", MOSTLY_NONE)
def test_layers_where_most_rows_are_in_no_group(sizes, behind, inputs, outputs, act, gated):
    test_grouped_layers(sizes, behind, inputs, outputs, torch.bfloat16, act, True, gated)


@gpu
@pytest.mark.parametrize("sizes", [[0] * 200 + [3, 0, 70, 1] + [0] * 90 + [65],
                                   [1] * 3 + [0] * 500 + [2, 1] + [0] * 7 + [64, 63]])
@pytest.mark.parametrize("act,gated", [(None, False), ("silu", True)])
def test_few_rows_among_many_groups(sizes, act, gated):
    test_grouped_layers(sizes, 2, 136, 72, torch.bfloat16, act, True, gated)


@gpu
def test_scratch_of_few_rows_does_not_grow_with_the_groups():
    """10 rows among 1024 groups of 4096 -> 4096: 64 lines of both operands for each of the ten groups
    that may have rows, a float32 sum of each bias, and less than a MB beside."""
    lib, need = L.load_library(), ctypes.c_int64(0)
    rows, groups, width = 10, 1024, 4096
    some = 1 << 20  # any aligned address: sizes alone are asked
    args = L.GroupedLinearGradArgs(
        rows=rows, inputs=width, outputs=width, groups=groups, x_stride=width, weight_stride=width,
        dy_stride=width, device=0, dtype=L.RUNE_BF16, activation=L.RUNE_ACT_NONE, x=some, weight=some,
        offsets=some, dy=some, dx=some, dweight=some, dbias=some)
    assert lib.rune_grouped_linear_backward_workspace(ctypes.byref(args), ctypes.byref(need)) == 0
    assert need.value <= 2 * rows * 64 * width * 2 + groups * width * 4 + (1 << 20)


@gpu
@pytest.mark.parametrize("inputs,outputs,gated", [(1 << 29, 1, 0), (64, 1 << 29, 0), (64, 1 << 28, 1),
                                                  ((1 << 28) + 1, 8, 0)])
def test_weight_gradients_refuse_lines_that_their_counters_cannot_hold(inputs, outputs, gated):
    """By the workspace's size, that is before anything is launched; dx alone has no such limit."""
    lib, need, some = L.load_library(), ctypes.c_int64(0), 1 << 20
    width = inputs
    args = L.GroupedLinearGradArgs(
        rows=1, inputs=inputs, outputs=outputs, groups=1, x_stride=width, weight_stride=width,
        dy_stride=outputs, device=0, dtype=L.RUNE_BF16, activation=L.RUNE_ACT["silu"], gated=gated,
        x=some, weight=some, offsets=some, dy=some, dx=some, dweight=some)
    assert lib.rune_grouped_linear_backward_workspace(ctypes.byref(args), ctypes.byref(need)) \
        == L.RUNE_ERR_INVALID
    assert b"weight gradients" in lib.rune_last_error()
    args.dweight = None
    assert lib.rune_grouped_linear_backward_workspace(ctypes.byref(args), ctypes.byref(need)) == 0


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("width", [1, 33, 64, 520])
def test_weighted_rows_to_groups_by_the_c_entry(dtype, width):
    """rune_to_groups with weights, which no operator of ops passes: one product a value, rounded as
    torch does, whatever lies in rows that have no place."""
    lib = L.load_library()
    rows, k = 70, 3
    g = ops.row_groups(choice(211, rows, k, 9, wrong=0.3), 9)
    x, w = normal(212, rows, width, dtype=dtype), normal(213, rows, k, dtype=torch.float32)
    w[g.place < 0] = float("nan")
    out = torch.full((rows * k, width), float("nan"), dtype=dtype, device="cuda")
    code = {torch.float32: L.RUNE_F32, torch.float16: L.RUNE_F16, torch.bfloat16: L.RUNE_BF16}
    args = L.GroupMoveArgs(rows=rows, k=k, width=width, in_stride=width, device=0, dtype=code[dtype],
                           input=x.data_ptr(), order=g.order.data_ptr(), place=g.place.data_ptr(),
                           weights=w.data_ptr(), out=out.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.rune_to_groups(ctypes.byref(args), stream) == 0
    slot = g.order.long()
    want = x.float()[slot.clamp(min=0) // k] * w.flatten()[slot.clamp(min=0)][:, None]
    want = torch.where(slot[:, None] >= 0, want, torch.zeros_like(want)).to(dtype)
    assert torch.equal(out, want)


@gpu
def test_a_replayed_step_whose_rows_leave_their_groups():
    """A captured training step of 30000 rows, replayed as all but a few of them lose their group and
    come back: the bits of the same step run at once, weights' gradients over ranges among them."""
    dt, rows, count = torch.bfloat16, 30000, 4
    x = normal(221, rows, 64, dtype=dt).requires_grad_(True)
    w = normal(222, count, 96, 64, dtype=dt, scale=0.1).requires_grad_(True)
    b = normal(223, count, 96, dtype=dt).requires_grad_(True)
    dy = normal(224, rows, 96, dtype=dt)
    index = choice(225, rows, 0, count)
    whole = index.clone()

    def step():
        g = ops.row_groups(index, count)
        y = ops.from_groups(ops.grouped_linear(ops.to_groups(x, g), w, g, bias=b,
                                               activation="silu"), g)
        return (y, *torch.autograd.grad(y, [x, w, b], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for left in (rows, 1000, 130, 1, 0, 20000):
        index.copy_(torch.where(torch.arange(rows, device="cuda") < left, whole, -1))
        graph.replay()
        got = [t.detach().clone() for t in out]
        assert all(torch.equal(a, c) for a, c in zip(got, step()))
        assert left > 0 or not any(bool(t.any()) for t in got)
    ops.check_waits()
