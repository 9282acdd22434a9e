"""An optimiser for the networks' matrices: momentum, orthogonalised (Muon).

The update of a weight matrix is its momentum with all singular values brought near 1
(``rune_b200.ops.orthogonalize``). For the hidden matrices of ``rune_b200.network``, a plain matrix
each or a stack of them (the experts' weights); embeddings, heads, norms and biases go to another
optimiser.
"""

from __future__ import annotations

import math

import torch

from . import ops


class Muon(torch.optim.Optimizer):
    """``p <- (1 - lr weight_decay) p - lr sqrt(max(1, rows / columns)) U``, U the orthogonalised
    momentum ``m <- momentum m + g`` (nesterov: of ``g + momentum m``).

    params: CUDA parameters of two axes, or more for stacks of matrices (float32, float16 or
    bfloat16). Those of one shape are orthogonalised in one call. The momentum is float32 whatever
    the parameters are.
    """

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=ops.NEWTON_SCHULZ, eps=1.0e-7):
        if lr < 0.0 or not 0.0 <= momentum < 1.0 or weight_decay < 0.0:
            raise ValueError("lr and weight_decay cannot be negative, momentum is 0 to 1.")
        super().__init__(params, {"lr": lr, "momentum": momentum, "nesterov": nesterov,
                                  "weight_decay": weight_decay, "steps": steps,
                                  "coefficients": tuple(coefficients), "eps": eps})

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                self.param_groups.pop()
                raise ValueError("Muon takes matrices and stacks of them; give vectors to "
                                 "another optimiser.")

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class brings states to their parameters' type, which may have fewer bits
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                moment = state_dict["state"][i]["momentum"]
                self.state[p]["momentum"] = moment.detach().to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    alike.setdefault((p.shape[-2:], p.dtype, p.device), []).append(p)
            for params in alike.values():
                self._update(params, group)
        return loss

    def _update(self, params, group):
        for p in params:
            if "momentum" not in self.state[p]:
                self.state[p]["momentum"] = torch.zeros_like(p.grad, dtype=torch.float32)
        moments = [self.state[p]["momentum"] for p in params]
        grads = [p.grad.float() for p in params]
        torch._foreach_mul_(moments, group["momentum"])
        torch._foreach_add_(moments, grads)
        if group["nesterov"]:
            moments = torch._foreach_add(grads, moments, alpha=group["momentum"])
        rows, cols = params[0].shape[-2:]
        parts = [m.reshape(-1, rows, cols) for m in moments]
        stack = parts[0] if len(parts) == 1 else torch.cat(parts)
        update = ops.orthogonalize(stack, steps=group["steps"], coefficients=group["coefficients"],
                                   eps=group["eps"])
        updates = [u.view_as(p).to(p.dtype)
                   for u, p in zip(update.split([len(m) for m in parts]), params)]
        if group["weight_decay"]:
            torch._foreach_mul_(params, 1.0 - group["lr"] * group["weight_decay"])
        torch._foreach_add_(params, updates,
                            alpha=-group["lr"] * math.sqrt(max(1.0, rows / cols)))
