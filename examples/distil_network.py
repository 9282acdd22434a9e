"""Distil a model's per-atom energies into a ScalarNetwork, in bfloat16 on one GPU.

The teacher is a NEP4 engine model (random initialisation from a seed); the student sees, for each
atom of a periodic alloy, a histogram of its neighbours' distances by species, and learns the
teacher's per-atom energies. The training step runs the operators of ``rune_b200.ops`` forward and
backward; at the end the 8-bit copy serves the same energies.

    python examples/distil_network.py [--steps 300] [--cells 8] [--gated] [--experts 8] [--muon]

``--experts`` gives the blocks as many feed-forward networks, two for each atom (and no 8-bit copy);
``--muon`` updates the blocks' matrices by their orthogonalised momentum.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import numpy as np
import torch

from rune_b200.nep.plugin import build_model, resolve_params
from rune_b200.network import ScalarNetwork
from rune_b200.optim import Muon


def alloy(cells, seed, a=3.6, jitter=0.1, species=3):
    """Positions [N, 3], edge length and species of a jittered FCC alloy box."""
    rng = np.random.default_rng(seed)
    basis = np.array([[0, 0, 0], [0, .5, .5], [.5, 0, .5], [.5, .5, 0]])
    grid = np.stack(np.meshgrid(*(np.arange(cells),) * 3, indexing="ij"), -1).reshape(-1, 3)
    pos = (grid[:, None] + basis[None]).reshape(-1, 3) * a + rng.normal(0, jitter, (4 * cells ** 3, 3))
    return pos, cells * a, rng.integers(0, species, len(pos))


def features(pos, edge, types, species=3, bins=24, cutoff=6.0):
    """[N, species * bins] smooth histogram of neighbour distances (minimum image)."""
    d = pos[:, None] - pos[None]
    r = (d - edge * torch.round(d / edge)).norm(dim=-1)
    r.fill_diagonal_(2 * cutoff)
    out = []
    fade = 0.5 * (1 + torch.cos(np.pi * (r / cutoff).clamp(max=1.0)))
    for s in range(species):
        seen = fade * (types[None] == s)
        out += [(seen * torch.exp(-0.5 * ((r - c) / 0.15) ** 2)).sum(1)
                for c in torch.linspace(1.8, cutoff, bins).tolist()]
    return torch.stack(out, 1)


def train(steps=300, cells=8, gated=False, hidden=128, blocks=3, seed=7, log=print, experts=0,
          muon=False):
    """(first and last loss, the 8-bit copy's root-mean-square deviation from the network, or None)."""
    dev = torch.device("cuda")
    torch.manual_seed(seed)
    teacher = build_model(resolve_params(dict(
        elements=["Cu", "Ag", "Au"], rcut_radial=6.0, rcut_angular=4.0, l_max=4, l_max_4body=2,
        l_max_5body=1, hidden_dims=[30], max_neighbors_radial=200,
        max_neighbors_angular=100))).to(dev).eval()
    data = []
    for k in range(4):
        pos, edge, types = alloy(cells, seed + k)
        pos, types = torch.as_tensor(pos, device=dev), torch.as_tensor(types, device=dev)
        out = teacher.evaluate(pos, np.eye(3).reshape(1, 9) * edge, np.ones((1, 3), bool),
                               types.to(torch.int32), compute_forces=False,
                               compute_virial=False)
        data.append((features(pos.float(), edge, types), types, out["energies"].float()))
    mean = torch.cat([e for _, _, e in data]).mean()
    spread = torch.cat([e for _, _, e in data]).std()
    net = ScalarNetwork(3, data[0][0].shape[1], hidden, 2 * hidden, blocks, gated=gated,
                        experts=experts).to(dev)
    net.q_scaler.copy_(1.0 / torch.cat([q for q, _, _ in data]).std(0).clamp(min=1e-3))
    matrices = [p for p in net.residual_blocks.parameters()
                if muon and (p.dim() == 3 or not experts and p.dim() == 2)]
    inside = {id(p) for p in matrices}
    opts = [torch.optim.AdamW([p for p in net.parameters() if id(p) not in inside], lr=2e-3)]
    if matrices:
        opts.append(Muon(matrices, lr=5e-3))
    losses = []
    for step in range(steps):
        q, types, energies = data[step % len(data)]
        loss = ((net(q, types) - (energies - mean) / spread) ** 2).mean()
        net.zero_grad(set_to_none=True)
        loss.backward()
        for opt in opts:
            opt.step()
        losses.append(loss.detach())
        if log and step % max(1, steps // 10) == 0:
            log(f"step {step}: mean squared error {float(losses[-1]):.4f} of the variance")
    q, types, _ = data[0]
    apart = None
    if not experts:
        with torch.no_grad():
            apart = float((net.quantized()(q, types) - net(q, types)).pow(2).mean().sqrt())
    first, last = float(losses[0]), float(torch.stack(losses[-4:]).mean())
    if log:
        log(f"mean squared error {first:.4f} -> {last:.4f}"
            + ("" if experts else f"; 8-bit copy {apart:.4f} apart"))
    return first, last, apart


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--steps", type=int, default=300)
    parser.add_argument("--cells", type=int, default=8)
    parser.add_argument("--gated", action="store_true")
    parser.add_argument("--experts", type=int, default=0)
    parser.add_argument("--muon", action="store_true")
    args = parser.parse_args()
    train(args.steps, args.cells, args.gated, experts=args.experts, muon=args.muon)
