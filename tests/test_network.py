"""ScalarNetwork (rune_b200.network): the Möbius Local network on the mixed-precision operators."""

from __future__ import annotations

import importlib.util

import numpy as np
import pytest
import torch

from rune_b200.network import ScalarNetwork
from tests.helpers import GOLDEN, ROOT, load_params, load_state


def tiny_local():
    from rune_b200.mobius.plugin import build_model

    g = np.load(GOLDEN / "tiny_local.npz")
    model = build_model(load_params(g))
    model.load_state_dict({k: torch.as_tensor(v, dtype=torch.float32)
                           for k, v in load_state(g).items()}, strict=True)
    return model


def reference(net, q, types):
    """Energies in float64 and the sum of the magnitudes of their terms, per atom."""
    p = {k: v.detach().double() for k, v in net.state_dict().items()}
    act = {"tanh": torch.tanh, "silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu}[net.activation]

    def norm(h, w):
        return h / torch.sqrt((h * h).mean(-1, keepdim=True) + net.norm_eps) * w

    h = (q.double() * p["q_scaler"]) @ p["input_projection.weight"].t()
    h = h + p["input_projection.bias"] + p["element_embedding.weight"][types]
    for i in range(len(net.residual_blocks)):
        b = f"residual_blocks.{i}."
        z = norm(h, p[b + "norm.weight"]) @ p[b + "ffn.0.weight"].t() + p[b + "ffn.0.bias"]
        if net.gated:
            gate, up = z.chunk(2, -1)
            z = act(gate) * up
        else:
            z = act(z)
        h = h + z @ p[b + "ffn.2.weight"].t() + p[b + "ffn.2.bias"]
    terms = norm(h, p["output_norm.weight"]) * p["energy_heads.weight"][types]
    return terms.sum(-1) + p["energy_heads.bias"][types], terms.abs().sum(-1)


def test_from_mobius_copies_every_parameter_and_refuses_messages():
    model = tiny_local()
    net = ScalarNetwork.from_mobius(model)
    theirs = model.state_dict()
    for key, value in net.state_dict().items():
        assert torch.equal(value, theirs[key]), key
    model.message_layers = 1
    with pytest.raises(ValueError, match="no messages"):
        ScalarNetwork.from_mobius(model)
    with pytest.raises(ValueError, match="dtype"):
        ScalarNetwork(2, 4, 8, 16, 1, dtype=torch.float32)
    with pytest.raises(ValueError, match="positive"):
        ScalarNetwork(2, 0, 8, 16, 1)
    with pytest.raises(ValueError, match="CUDA tensor"):
        net(torch.zeros(2, model.input_dim), torch.zeros(2, dtype=torch.long))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,unit", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_network_matches_the_mobius_local_network(dtype, unit):
    """Each block rounds the stream, the normalised rows, the activations and its output once, the
    weights are rounded once: some ten roundings of relative size `unit` per block, independent,
    of values whose contributions the last normalisation keeps at the scale of the terms."""
    model = tiny_local().cuda()
    net = ScalarNetwork.from_mobius(model, dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(203, model.input_dim, generator=gen, device="cuda")
    types = torch.randint(0, model.n_elements, (203,), generator=gen, device="cuda")
    want, scale = reference(net, q, types)
    bound = 10 * unit * (len(net.residual_blocks) + 2)
    with torch.no_grad():
        assert float(((net(q, types).double() - want).abs() / scale).max()) <= bound
    # 8 bits: e4m3 rounds weights and activations to 2^-4, the products average over their terms
    apart = (net.quantized()(q, types).double() - want).abs() / scale
    assert float(apart.max()) <= 10 * 2.0 ** -4 * (len(net.residual_blocks) + 2)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_gradients_reach_every_parameter(gated):
    """Gradients of the mixed-precision network against automatic differentiation in float64:
    the angle between them is that of relative errors of some units of bfloat16."""
    torch.manual_seed(5)
    net = ScalarNetwork(3, 40, 64, 96, 2, activation="gelu", gated=gated).cuda()
    q = torch.randn(500, 40, device="cuda")
    types = torch.randint(0, 3, (500,), device="cuda")
    net(q, types).pow(2).sum().backward()
    double = ScalarNetwork(3, 40, 64, 96, 2, activation="gelu", gated=gated).cuda().double()
    double.load_state_dict(net.state_dict())
    leaves = dict(double.named_parameters())

    class Leaves:  # reference() on parameters that record gradients
        residual_blocks, activation, gated = net.residual_blocks, net.activation, net.gated
        norm_eps = net.norm_eps

        @staticmethod
        def state_dict():
            return {k: _Live(v) for k, v in {**leaves, "q_scaler": double.q_scaler}.items()}

    reference(Leaves, q, types)[0].pow(2).sum().backward()
    for name, p in net.named_parameters():
        g, w = p.grad.double(), leaves[name].grad
        assert float((g - w).norm()) <= 20 * 2.0 ** -8 * float(w.norm()), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,unit", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_embedding_gradient_of_many_atoms(dtype, unit):
    """33333 atoms an element whose gradients have one sign. The network is projection, norm and
    head: an atom's gradient is the norm's, with 16-bit operands h, w and dy and a result of 16
    bits, each off by one rounding of its two terms; then float32 sums of all atoms (n 2^-24)."""
    torch.manual_seed(0)
    net = ScalarNetwork(3, 8, 64, 96, 0, dtype=dtype).cuda()
    with torch.no_grad():
        net.energy_heads.weight.copy_(torch.randn(3, 64, device="cuda"))
        net.output_norm.weight.copy_(1 + 0.2 * torch.randn(64, device="cuda"))
    n = 99999
    q = 0.05 * torch.randn(n, 8, device="cuda")
    types = torch.arange(n, device="cuda") % 3
    (100.0 * net(q, types)).sum().backward()
    p = {k: v.detach().double() for k, v in net.state_dict().items()}
    # h as the projection rounds it: one rounding of the operands' products and of the sum
    h = (q.double() * p["q_scaler"]) @ p["input_projection.weight"].t()
    h = h + p["input_projection.bias"] + p["element_embedding.weight"][types]
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + net.norm_eps)
    gw = 100.0 * p["energy_heads.weight"][types] * p["output_norm.weight"]
    normed = h * r
    dot = (gw * normed).mean(-1, keepdim=True)
    dh = r * (gw - normed * dot)
    # roundings: dy, dx and h (q, weights, bias, embedding and the sum, of the terms' magnitudes)
    terms = (q.double().abs() @ p["input_projection.weight"].abs().t()
             + p["input_projection.bias"].abs() + p["element_embedding.weight"][types].abs())
    eh = 4 * unit * terms
    en = r * (eh + normed.abs() * (normed.abs() * eh * r).mean(-1, keepdim=True))
    edot = (gw.abs() * (2 * unit * normed.abs() + en)).mean(-1, keepdim=True)
    er = (normed.abs() * eh * r).mean(-1, keepdim=True)  # of r, relative
    bound = r * (2 * unit * gw.abs() + en * dot.abs() + normed.abs() * edot)
    bound = bound + (unit + er + n * 2.0 ** -24) * r * (gw.abs() + (normed * dot).abs())
    want, room = (torch.zeros(3, 64, dtype=torch.float64, device="cuda").index_add_(0, types, t)
                  for t in (dh, bound))
    got = net.element_embedding.weight.grad.double()
    assert bool(((got - want).abs() <= 1.01 * room).all())
    # and 5 roundings of bfloat16 of the largest sum: the gradients of an element are alike
    assert float((got - want).abs().max()) <= 0.02 * float(want.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("stored", [torch.float32, torch.bfloat16])
def test_the_8_bit_network_is_a_copy(gated, stored):
    """of every parameter and buffer, also where their type is the states' already"""
    torch.manual_seed(6)
    net = ScalarNetwork(3, 40, 64, 96, 2, activation="gelu", gated=gated).cuda().to(stored)
    q = torch.randn(100, 40, device="cuda")
    types = torch.randint(0, 3, (100,), device="cuda")
    serve = net.quantized()
    before = serve(q, types)
    with torch.no_grad():
        for t in (*net.parameters(), *net.buffers()):
            t.mul_(1.5).add_(0.25)
    assert torch.equal(serve(q, types), before)
    assert not torch.equal(net.quantized()(q, types), before)


class _Live:
    """detach().double() of a float64 leaf that is to keep its gradient."""

    def __init__(self, t):
        self.t = t

    def detach(self):
        return self

    def double(self):
        return self.t


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_distillation_example_learns(gated):
    spec = importlib.util.spec_from_file_location("distil", ROOT / "examples/distil_network.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    first, last, apart = module.train(steps=60, cells=4, gated=gated, log=None)
    assert last < 0.5 * first and apart < 0.2
