"""Networks with experts, networks per element, and Muon, on the grouped operators."""

from __future__ import annotations

import importlib.util

import pytest
import torch

from rune_b200.network import ElementNetwork, ScalarNetwork
from rune_b200.optim import Muon
from tests.helpers import ROOT

gpu = pytest.mark.gpu


def nep_model():
    from rune_b200.nep.plugin import build_model, resolve_params

    torch.manual_seed(3)
    return build_model(resolve_params(dict(
        elements=["Cu", "Ag", "Au"], rcut_radial=6.0, rcut_angular=4.0, l_max=4, l_max_4body=2,
        l_max_5body=1, hidden_dims=[30], max_neighbors_radial=200, max_neighbors_angular=100)))


# ------------------------------------------------------------------------------------ CPU
def test_dimensions_are_checked():
    for bad in ({"experts": -1}, {"experts": 4, "top_k": 5}, {"experts": 4, "top_k": 0}):
        with pytest.raises(ValueError):
            ScalarNetwork(2, 4, 8, 16, 1, **bad)
    with pytest.raises(ValueError, match="8-bit"):
        ScalarNetwork(2, 4, 8, 16, 1, experts=4).quantized()
    with pytest.raises(ValueError, match="positive"):
        ElementNetwork(0, 4, 8)
    with pytest.raises(ValueError, match="dtype"):
        ElementNetwork(2, 4, 8, dtype=torch.float32)


@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 2), (7, 2)])
def test_the_number_of_choices_follows_the_experts(experts, top_k):
    assert ScalarNetwork(2, 4, 8, 16, 1, experts=experts).residual_blocks[0].top_k == top_k
    with pytest.raises(ValueError, match="top_k"):
        ScalarNetwork(2, 4, 8, 16, 1, experts=experts, top_k=experts + 1)


def test_from_nep_copies_every_parameter():
    model = nep_model()
    net = ElementNetwork.from_nep(model)
    for i, e in enumerate(model.elements):
        mlp = model.element_mlps[e]
        assert torch.equal(net.weight[i], mlp[0].weight) and torch.equal(net.bias[i], mlp[0].bias)
        assert torch.equal(net.head.weight[i], mlp[2].weight[0])
    assert not bool(net.head.weight[len(model.elements)].any())
    assert torch.equal(net.q_scaler, model.q_scaler)


def test_muon_takes_matrices_alone():
    with pytest.raises(ValueError, match="matrices"):
        Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError, match="lr"):
        Muon([torch.nn.Parameter(torch.zeros(4, 4))], lr=-1.0)


def test_muon_refuses_vectors_added_later_and_keeps_float32_momentum_when_loaded():
    p = torch.nn.Parameter(torch.zeros(4, 6, dtype=torch.bfloat16))
    opt = Muon([p])
    with pytest.raises(ValueError, match="matrices"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))]})
    assert len(opt.param_groups) == 1
    torch.manual_seed(4)
    opt.state[p]["momentum"] = torch.randn(4, 6)
    other = torch.nn.Parameter(p.detach().clone())
    loaded = Muon([other])
    loaded.load_state_dict(opt.state_dict())
    assert loaded.state[other]["momentum"].dtype == torch.float32
    assert torch.equal(loaded.state[other]["momentum"], opt.state[p]["momentum"])
    assert loaded.state[other]["momentum"] is not opt.state[p]["momentum"]


def test_muon_skips_empty_matrices():
    p = torch.nn.Parameter(torch.zeros(4, 0))
    p.grad = torch.zeros(4, 0)
    Muon([p]).step()


# ------------------------------------------------------------------------------------ GPU
def experts64(net, q, types, choices):
    """Energies in float64 with the given choice of experts in each block."""
    p = {k: v.detach().double() for k, v in net.state_dict().items()}
    act = {"silu": torch.nn.functional.silu, "tanh": torch.tanh,
           "gelu": torch.nn.functional.gelu}[net.activation]

    def norm(h, w):
        return h / torch.sqrt((h * h).mean(-1, keepdim=True) + net.norm_eps) * w

    h = (q.double() * p["q_scaler"]) @ p["input_projection.weight"].t()
    h = h + p["input_projection.bias"] + p["element_embedding.weight"][types]
    for i, index in enumerate(choices):
        b = f"residual_blocks.{i}."
        x = norm(h, p[b + "norm.weight"])
        w = torch.softmax((x @ p[b + "router.weight"].t()).gather(1, index), 1)
        for j in range(index.shape[1]):
            e = index[:, j]
            z = torch.einsum("nh,nfh->nf", x, p[b + "weight_in"][e]) + p[b + "bias_in"][e]
            if net.gated:
                gate, up = z.chunk(2, -1)
                z = act(gate) * up
            else:
                z = act(z)
            z = torch.einsum("nf,nhf->nh", z, p[b + "weight_out"][e]) + p[b + "bias_out"][e]
            h = h + w[:, j:j + 1] * z
    terms = norm(h, p["output_norm.weight"]) * p["energy_heads.weight"][types]
    return terms.sum(-1) + p["energy_heads.bias"][types], terms.abs().sum(-1)


@gpu
@pytest.mark.parametrize("gated,activation", [(False, "silu"), (True, "gelu")])
def test_scalar_network_with_experts(gated, activation, monkeypatch):
    """Against float64 with the network's own choice of experts. A state goes through at most ten
    roundings to bfloat16 in each of three blocks and four more, 2^-8 of its size each at most, and
    the energy is a sum of terms of the state."""
    from rune_b200 import ops

    torch.manual_seed(1)
    net = ScalarNetwork(3, 20, 64, 96, 3, activation=activation, gated=gated, experts=6,
                        top_k=2).cuda()
    q, types = torch.randn(157, 20, device="cuda"), torch.arange(157, device="cuda") % 3
    choices, route = [], ops.route

    def recorded(logits, k):
        index, weights = route(logits, k)
        choices.append(index.long())
        return index, weights

    monkeypatch.setattr(ops, "route", recorded)
    energies = net(q, types)
    want, size = experts64(net, q, types, choices)
    assert energies.shape == (157,) and energies.dtype is torch.float32
    assert bool(((energies.double() - want).abs() <= 34 * 2.0 ** -8 * size).all())
    energies.sum().backward()
    for name, p in net.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()), name
        assert bool(p.grad.any()), name


@gpu
def test_element_network_is_the_models():
    """The hidden layer's operands and results are rounded to bfloat16: of z by 2^-7 of the products'
    sizes at most (two operands), of the result by 2^-8, and the head sums in float32."""
    model = nep_model().cuda()
    net = ElementNetwork.from_nep(model)
    torch.manual_seed(5)
    q = 0.3 * torch.randn(1000, model.input_dim, device="cuda")
    types = torch.randint(0, 3, (1000,), device="cuda")
    types[7] = -1
    energies = net(q, types)
    x = q.double() * net.q_scaler.double()
    w, b, head = net.weight.double(), net.bias.double(), net.head.weight.double()
    t = types.clamp(min=0)
    z = torch.einsum("nd,nhd->nh", x, w[t]) + b[t]
    size = torch.einsum("nd,nhd->nh", x.abs(), w[t].abs()) + b[t].abs()
    want = (torch.tanh(z) * head[t]).sum(-1) - net.shared_bias.double()
    err = ((2.0 ** -7 * size + 2.0 ** -8) * head[t].abs()).sum(-1) * 1.05 + 1e-6
    held = types >= 0
    assert bool(((energies.double() - want).abs() <= err)[held].all())
    assert float(energies[7].detach()) == -float(net.shared_bias.detach())
    energies.sum().backward()
    for name, p in net.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()), name
    assert not bool(net.head.weight.grad[3].any())


@gpu
@pytest.mark.parametrize("atoms", [0, 1])
def test_no_atoms_and_one(atoms):
    torch.manual_seed(4)
    q, types = torch.randn(atoms, 20, device="cuda"), torch.zeros(atoms, dtype=torch.int32,
                                                                 device="cuda")
    for net in (ScalarNetwork(3, 20, 64, 96, 2, experts=6, top_k=3).cuda(),
                ElementNetwork(3, 20, 30).cuda()):
        energies = net(q, types)
        assert energies.shape == (atoms,) and bool(energies.isfinite().all())
        energies.sum().backward()
        for name, p in net.named_parameters():
            assert p.grad is None or bool(p.grad.isfinite().all()), name


@gpu
def test_muon_step_is_its_formula():
    torch.manual_seed(2)
    shapes = [(64, 32), (3, 40, 96), (64, 32), (1, 40, 96)]
    params = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in shapes]
    before = [p.detach().clone() for p in params]
    opt = Muon(params, lr=0.1, momentum=0.9, weight_decay=0.01)
    from rune_b200 import ops

    moments = [torch.zeros_like(p) for p in params]
    for _ in range(2):
        for p in params:
            p.grad = torch.randn_like(p)
        for p, m, w in zip(params, moments, before):
            m.mul_(0.9).add_(p.grad)
            u = ops.orthogonalize(p.grad + 0.9 * m).float()
            scale = max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
            w.mul_(1 - 0.1 * 0.01).add_(u, alpha=-0.1 * scale)
        opt.step()
    for p, w in zip(params, before):
        # the stack's tiles may be others than a single matrix's: the update's rounding, twice
        assert bool(((p - w).abs() <= 2 * 0.1 * 1.5 * 2.0 ** -7 * 1.3).all())
    params[0].grad = None
    kept = params[0].detach().clone()
    opt.step()
    assert torch.equal(kept, params[0])


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_muon_holds_the_momentum_of_16_bit_parameters_in_float32(dtype):
    torch.manual_seed(5)
    p = torch.nn.Parameter(torch.randn(48, 40, device="cuda").to(dtype))
    opt = Muon([p], lr=0.1, momentum=0.9, nesterov=False)
    moment = torch.zeros(48, 40, dtype=torch.float64, device="cuda")
    for _ in range(8):
        p.grad = torch.randn_like(p)
        moment = 0.9 * moment + p.grad.double()
        opt.step()
    # three float32 roundings a step (0.9 itself among them) of values below sum |g| < 8 * 6 in size
    kept = opt.state[p]["momentum"]
    assert kept.dtype == torch.float32 and bool(p.isfinite().all())
    assert float((kept.double() - moment).abs().max()) <= 8 * 3 * 2.0 ** -24 * 48


@gpu
@pytest.mark.parametrize("experts,muon", [(4, False), (0, True), (4, True)])
def test_example_runs(experts, muon):
    spec = importlib.util.spec_from_file_location("distil_network",
                                                  ROOT / "examples" / "distil_network.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    first, last, apart = module.train(steps=6, cells=3, hidden=32, blocks=2, log=None,
                                      experts=experts, muon=muon)
    assert first == first and last == last and (apart is None) == bool(experts)
