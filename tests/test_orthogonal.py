"""ops.orthogonalize against its definition in float64.

A step takes X, A and B rounded to float16 (2^-11 of each value, 2^-24 / 1024 below its smallest
normal numbers), with float32 sums, and its last result to bfloat16. One step's error is bounded value
by value. Over several steps the errors E of X in the Frobenius norm grow by at most the largest
slope s of the odd polynomial a t + b t^3 + c t^5 on [0, 1.3], where the singular values stay: the
derivative of such a matrix function in any direction is a Hadamard product with divided
differences of the polynomial, which that slope bounds."""

from __future__ import annotations

import pytest
import torch

from rune_b200 import ops
from rune_b200.runtime import library as L
from tests.test_ops import normal

gpu = pytest.mark.gpu
H, TINY = 2.0 ** -11, 2.0 ** -25 / 1024  # of float16, and half its smallest number, scaled back
BF = 2.0 ** -8
A, B, C = ops.NEWTON_SCHULZ
SHAPES = [(1, 1, 1), (2, 1, 9), (1, 9, 1), (3, 8, 8), (1, 64, 200), (2, 200, 64), (2, 129, 127),
          (1, 127, 300), (1, 300, 515), (1, 515, 300), (4, 256, 512), (1, 777, 260), (1, 640, 640)]


def start(x, eps=1.0e-7):
    x = x.double()
    return x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)


def step64(x, a=A, b=B, c=C):
    g = x @ x.mT if x.shape[-2] <= x.shape[-1] else x.mT @ x
    p = b * g + c * g @ g
    return a * x + (p @ x if x.shape[-2] <= x.shape[-1] else x @ p)


def one_step_bound(x, a=A, b=B, c=C):
    """|error| of each value after one step from the exact normalised x: products of operands that
    are off by e_x, e_g, e_p, their float32 sums, and the rounding of each result"""
    wide = x.shape[-2] <= x.shape[-1]
    small, large = sorted(x.shape[-2:])
    y = x.abs()
    ex = H * y * 1.01 + TINY
    gram = (lambda u, v: u @ v.mT) if wide else (lambda u, v: u.mT @ v)
    g = gram(y, y)
    eg = gram(ex, y) + gram(y, ex) + gram(ex, ex) + (large + 4) * 2.0 ** -23 * gram(y, y)
    eg = eg + H * (gram(x, x).abs() + eg) + TINY
    p = abs(b) * g + abs(c) * g @ g
    ep = abs(b) * eg + abs(c) * (eg @ g + g @ eg + eg @ eg) + (small + 8) * 2.0 ** -23 * p
    ep = ep + H * (p + ep) + TINY
    times = (lambda u, v: u @ v) if wide else (lambda u, v: v @ u)
    out = abs(a) * y + times(p, y)
    return abs(a) * ex + times(ep, y) + times(p, ex) + times(ep, ex) \
        + (small + 8) * 2.0 ** -23 * out


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("count,m,n", SHAPES)
def test_one_step(count, m, n, dtype):
    x = normal(1, count, m, n, dtype=dtype, scale=0.02)
    got = ops.orthogonalize(x, steps=1)
    s = start(x)
    want, err = step64(s), one_step_bound(s)
    assert got.dtype is torch.bfloat16 and got.shape == x.shape
    off = (got.double() - want).abs()
    assert bool((off <= err + BF * (want.abs() + err)).all()), float((off / (err + BF * want.abs())).max())


@gpu
@pytest.mark.parametrize("steps", [0, 2, 5, 6])
@pytest.mark.parametrize("count,m,n", SHAPES)
def test_steps(count, m, n, steps):
    x = normal(2, count, m, n, dtype=torch.float32, scale=3.0)
    got = ops.orthogonalize(x, steps=steps).double()
    s = start(x)
    t = torch.linspace(0, 1.3, 2000, dtype=torch.float64)
    slope = float((A + 3 * B * t ** 2 + 5 * C * t ** 4).abs().max())
    small, large = sorted((m, n))
    err = torch.zeros(count, dtype=torch.float64, device="cuda")
    norm = torch.linalg.matrix_norm
    for _ in range(steps):
        # of this step alone, in the norm: operands X, G and P with their roundings (at most
        # |P| <= |b| + |c| times what X has, and G at most X's largest singular value squared)
        nx, sx = norm(s), norm(s, ord=2) if min(m, n) else None
        g = sx ** 2
        p = abs(B) * g + abs(C) * g * g
        eg = 2 * H * nx * sx + H * nx * sx + (large + 4) * 2.0 ** -23 * nx * nx
        ep = (abs(B) + 2 * abs(C) * g) * eg + H * p * small ** 0.5 \
            + (small + 8) * 2.0 ** -23 * (abs(B) * nx * nx + abs(C) * nx ** 4)
        own = (A + p) * H * nx + ep * sx + (small + 8) * 2.0 ** -23 * (A * nx + p * nx)
        pads = TINY * (m * n) ** 0.5 * 8
        err = slope * err * 1.02 + 1.02 * own + pads
        s = step64(s)
    apart = norm(got - s)
    assert bool((apart <= err + BF * (norm(s) + err)).all()), (apart, err)


@gpu
def test_singular_values_come_near_one():
    x = normal(3, 3, 200, 320, dtype=torch.float32)
    sv = torch.linalg.svdvals(ops.orthogonalize(x).double())
    assert float(sv.max()) < 1.3 and float(sv.min()) > 0.6
    # and the singular vectors stay: for exact ones u v^T has the inner product of nearly all of it
    u, _, vh = torch.linalg.svd(x.double(), full_matrices=False)
    inner = ((u @ vh) * ops.orthogonalize(x).double()).sum((1, 2)) / sv.norm(dim=1) / 200 ** 0.5
    assert float(inner.min()) > 0.95


@gpu
def test_zeros_infinities_and_other_scales():
    x = normal(4, 4, 40, 64, dtype=torch.float32)
    x[1] = 0.0
    x[2, 3, 4] = float("nan")
    got = ops.orthogonalize(x)
    assert not bool(got[1].any()) and bool(got[2].isnan().all())
    keep = [0, 3]
    assert torch.equal(got[keep], ops.orthogonalize(x[keep]))
    # a power of two changes nothing but eps's share, here 2^-30 at most of the norm
    for scale in (2.0 ** 100, 2.0 ** -12):
        assert torch.equal(ops.orthogonalize(x[:1] * scale, eps=0.0), ops.orthogonalize(x[:1], eps=0.0))
    x[3, 0, 0] = float("inf")
    assert bool(ops.orthogonalize(x)[3].isnan().any())


@gpu
def test_strides_axes_and_equal_bits():
    base = normal(5, 4, 90, 3, 130, dtype=torch.bfloat16)
    for x in (base[:, :, 1, 7:107], base[:, :, 1, 7:107].transpose(1, 2), base[0, :, 0], base[:, 0],
              base[:, :, 2].transpose(0, 1)[3:5], base):
        a = ops.orthogonalize(x)
        assert a.shape == x.shape and a.is_contiguous()
        assert torch.equal(a, ops.orthogonalize(x.contiguous()))
    assert ops.orthogonalize(base[:0, :, 0]).shape == (0, 90, 130)
    assert ops.orthogonalize(base[:, :0, 0]).shape == (4, 0, 130)
    # the batch does not change a matrix's bits, as long as the tiles are the same
    x = normal(6, 3, 128, 128, dtype=torch.float32)
    whole = ops.orthogonalize(x)
    assert all(torch.equal(whole[i], ops.orthogonalize(x[i])) for i in range(3))


@gpu
def test_refusals():
    x = normal(7, 8, 8, dtype=torch.float32)
    for call, message in ((lambda: ops.orthogonalize(x[0]), "two axes"),
                          (lambda: ops.orthogonalize(x, steps=-1), "steps"),
                          (lambda: ops.orthogonalize(x, steps=65), "steps"),
                          (lambda: ops.orthogonalize(x, eps=-1.0), "eps"),
                          (lambda: ops.orthogonalize(x.double()), "float32"),
                          (lambda: ops.orthogonalize(x.clone().requires_grad_(True)), "no gradient")):
        with pytest.raises(ValueError, match=message):
            call()


@gpu
def test_a_wait_that_gives_up_is_reported():
    lib = L.load_library()
    x = normal(8, 2, 300, 520, dtype=torch.float32)
    want = ops.orthogonalize(x)
    torch.cuda.synchronize()
    try:
        lib.rune_linear_set_wait_polls(0)
        try:
            ops.orthogonalize(x)
        except L.RuneError:
            pass
        torch.cuda.synchronize()
        with pytest.raises(L.RuneError, match="did not complete"):
            ops.check_waits()
    finally:
        lib.rune_linear_set_wait_polls(L.DEFAULT_WAIT_POLLS)
    assert torch.equal(want, ops.orthogonalize(x))


@gpu
def test_offsets_beyond_32_bits():
    """A stack of more than 2^31 values. The last matrix alone may take other tiles: both results are
    off by a few float16 roundings of values that five steps amplify, and one to bfloat16."""
    x = torch.empty(530, 2048, 2048, dtype=torch.bfloat16, device="cuda")
    for at in range(0, 530, 53):
        x[at:at + 53] = normal(at, 53, 2048, 2048, dtype=torch.bfloat16)
    got = ops.orthogonalize(x)[-1].double()
    alone = ops.orthogonalize(x[-1]).double()
    assert float((got - alone).norm() / alone.norm()) <= 2.0 ** -6


@gpu
def test_captured_and_replayed():
    x = normal(9, 6, 96, 160, dtype=torch.float32)
    ops.orthogonalize(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.orthogonalize(x)
    for seed in (10, 11):
        x.copy_(normal(seed, 6, 96, 160, dtype=torch.float32))
        graph.replay()
        assert torch.equal(y, ops.orthogonalize(x))


@gpu
def test_the_largest_stack_and_one_more():
    test_one_step(65535, 2, 3, torch.float32)
    with pytest.raises(ValueError, match="65535"):
        ops.orthogonalize(torch.zeros(65536, 2, 3, device="cuda"))
