"""The Möbius scalar network in mixed precision, trainable: projection, residual blocks, head; with
experts in its blocks on request; and NEP's networks, one per element.

The engine evaluates Möbius models in float32 without parameter gradients. ``ScalarNetwork`` is
the same per-atom network (rune/mobius/model.py:256-305 without messages, layers.py:26-89) on the
operators of ``rune_b200.ops``: float32 parameters under the reference's names, 16-bit products
with float32 accumulation, gradients for all of them. For distilling a model into it, or for
adapting a checkpoint's network and serving many atoms' energies where the caller has their
descriptors (the engine computes its own inside the kernels and returns none); no forces.
``quantized`` gives an 8-bit copy for serving.

A block adds its output to the residual stream in the next block's normalisation, so the stream
is read and written once per block.

``ElementNetwork`` is the network of NEP models (rune/nep/model.py:157-170 loops over the elements):
atoms sorted by element, one product for all of them.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import ops
from .mobius.model import ElementwiseLinearHead, ResidualBlock, RMSNorm


def _stack(groups, outputs, inputs):
    """Weights and biases of ``groups`` linear layers, each initialised as nn.Linear's."""
    bound = 1.0 / math.sqrt(inputs)
    return (nn.Parameter(torch.empty(groups, outputs, inputs).uniform_(-bound, bound)),
            nn.Parameter(torch.empty(groups, outputs).uniform_(-bound, bound)))


class ExpertBlock(nn.Module):
    """The residual block with ``experts`` feed-forward networks, ``top_k`` of them for each row,
    weighted by the softmax of their router logits."""

    def __init__(self, hidden, ffn, experts, top_k, activation, gated, norm_eps):
        super().__init__()
        self.activation, self.gated, self.top_k = activation, gated, top_k
        self.norm = RMSNorm(hidden, eps=norm_eps)
        self.router = nn.Linear(hidden, experts, bias=False)
        self.weight_in, self.bias_in = _stack(experts, (2 if gated else 1) * ffn, hidden)
        self.weight_out, self.bias_out = _stack(experts, hidden, ffn)

    def forward(self, x):
        """What the block adds to the stream, of its normalised rows."""
        dtype, experts = x.dtype, self.weight_in.shape[0]
        # The logits have 16 bits, as every layer's results here: half a step (2^-8 or 2^-11 of a
        # logit) is within what the rounded rows and weights leave open, experts nearer than that
        # tie and the first one wins. The softmax over the choices and its gradient are float32.
        index, weights = ops.route(ops.linear(x, self.router.weight.to(dtype)), self.top_k)
        groups = ops.row_groups(index, experts)
        layer = ops.grouped_gated_linear if self.gated else ops.grouped_linear
        x = layer(ops.to_groups(x, groups), self.weight_in.to(dtype), groups,
                  bias=self.bias_in.to(dtype), activation=self.activation)
        x = ops.grouped_linear(x, self.weight_out.to(dtype), groups, bias=self.bias_out.to(dtype))
        return ops.from_groups(x, groups, weights)


class ScalarNetwork(nn.Module):
    """Per-atom energies [N] (float32) of descriptors [N, inputs] and element indices [N].

    gated: the blocks' first layer is ``act(x Wg^T + bg) * (x Wu^T + bu)``; ``ffn.0`` then holds
    2 * ffn rows, the gate's first. experts: the blocks are ``ExpertBlock``s of as many networks,
    ``top_k`` of which each atom takes (default: two, or the one that there is); 0: none. dtype:
    torch.bfloat16 or torch.float16, of the states.
    """

    def __init__(self, n_elements, inputs, hidden, ffn, blocks, activation="silu", gated=False,
                 norm_eps=1.0e-8, dtype=torch.bfloat16, experts=0, top_k=None):
        super().__init__()
        if min(n_elements, inputs, hidden, ffn) <= 0 or blocks < 0 or experts < 0:
            raise ValueError("ScalarNetwork dimensions must be positive.")
        if top_k is None:
            top_k = min(2, experts)
        if experts and not 1 <= top_k <= min(experts, 32):
            raise ValueError(f"top_k must be 1 to 32 and at most the {experts} experts.")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be float16 or bfloat16, not {dtype}.")
        self.activation, self.gated, self.dtype = str(activation).strip().lower(), bool(gated), dtype
        self.norm_eps, self.experts = float(norm_eps), int(experts)
        self.register_buffer("q_scaler", torch.ones(inputs))
        self.input_projection = nn.Linear(inputs, hidden)
        self.element_embedding = nn.Embedding(n_elements, hidden)
        if experts:
            self.residual_blocks = nn.ModuleList(
                ExpertBlock(hidden, ffn, experts, top_k, self.activation, self.gated, norm_eps)
                for _ in range(blocks))
        else:
            self.residual_blocks = nn.ModuleList(
                ResidualBlock(hidden, ffn, activation, norm_eps=norm_eps) for _ in range(blocks))
        if gated and not experts:
            for block in self.residual_blocks:
                block.ffn[0] = nn.Linear(hidden, 2 * ffn)
        self.output_norm = RMSNorm(hidden, eps=norm_eps)
        self.energy_heads = ElementwiseLinearHead(n_elements, hidden)

    @classmethod
    def from_mobius(cls, model, dtype=torch.bfloat16):
        """The network of a Möbius Local model (``rune_b200.mobius.plugin``), its weights copied."""
        if model.message_layers:
            raise ValueError("ScalarNetwork has no messages: a Mobius model with "
                             "message_layers = 0 is needed.")
        net = cls(model.n_elements, model.input_dim, model.hidden_dim, model.ffn_dim,
                  model.blocks, model.activation, norm_eps=model.norm_eps, dtype=dtype)
        own = net.state_dict()
        net.load_state_dict({k: v for k, v in model.state_dict().items() if k in own})
        return net.to(model.q_scaler.device)

    def _cast(self, module):
        return module.weight.to(self.dtype), module.bias.to(self.dtype)

    def _start(self, descriptors, types):
        q = (descriptors * self.q_scaler).to(self.dtype)
        weight, bias = self._cast(self.input_projection)
        # rows first, then 16 bits: a table's gradient sums over all atoms of an element, in float32
        embedding = self.element_embedding(types).to(self.dtype)
        return ops.linear(q, weight, bias=bias, residual=embedding)

    def _finish(self, stream, delta, types):
        head = self.energy_heads
        return _energies(stream, delta, types, self.norm_eps, self.output_norm.weight,
                         head.weight, head.bias)

    def forward(self, descriptors, types):
        stream, delta = self._start(descriptors, types), None
        for block in self.residual_blocks:
            if delta is None:
                x = ops.rms_norm(stream, block.norm.weight, eps=self.norm_eps)
            else:
                x, stream = ops.rms_norm(delta, block.norm.weight, residual=stream,
                                         eps=self.norm_eps)
            if self.experts:
                delta = block(x)
                continue
            weight, bias = self._cast(block.ffn[0])
            if self.gated:
                x = ops.gated_linear(x, weight, bias=bias, activation=self.activation)
            else:
                x = ops.linear(x, weight, bias=bias, activation=self.activation)
            weight, bias = self._cast(block.ffn[2])
            delta = ops.linear(x, weight, bias=bias)
        return self._finish(stream, delta, types)

    def quantized(self):
        """A function like ``forward`` with the blocks' products in 8 bits: a copy of the network
        as it is now, its weights laid out; later changes of the network do not reach it. Not of
        networks with experts."""
        if self.experts:
            raise ValueError("The experts' products have no 8-bit form.")
        return _Quantized(self)


def _energies(stream, delta, types, eps, norm_weight, head_weight, head_bias):
    """Output normalisation of stream (+ delta) and the elements' head."""
    h = (ops.rms_norm(stream, norm_weight, eps=eps) if delta is None
         else ops.rms_norm(delta, norm_weight, residual=stream, eps=eps)[0])
    return (h.float() * head_weight[types]).sum(-1) + head_bias[types]


class _Quantized:
    """Forward of a ``ScalarNetwork`` whose blocks read e4m3 weights and activations."""

    @torch.no_grad()
    def __init__(self, net):
        def copy(t, dtype=None):
            return t.detach().to(dtype or t.dtype, copy=True)

        self.activation, self.gated, self.dtype = net.activation, net.gated, net.dtype
        self.norm_eps = net.norm_eps
        self.q_scaler = copy(net.q_scaler)
        self.projection = [copy(t, net.dtype) for t in (net.input_projection.weight,
                                                        net.input_projection.bias)]
        self.embedding = copy(net.element_embedding.weight, net.dtype)
        self.ends = [copy(t) for t in (net.output_norm.weight, net.energy_heads.weight,
                                       net.energy_heads.bias)]
        self.layers = [(copy(block.norm.weight),
                        *((*ops.quantize_fp8(layer.weight), copy(layer.bias, net.dtype))
                          for layer in (block.ffn[0], block.ffn[2])))
                       for block in net.residual_blocks]

    @torch.no_grad()
    def __call__(self, descriptors, types):
        delta = None
        first = ops.gated_linear if self.gated else ops.linear
        more = {"out_dtype": self.dtype}
        weight, bias = self.projection
        stream = ops.linear((descriptors * self.q_scaler).to(self.dtype), weight, bias=bias,
                            residual=self.embedding[types])
        for norm, (w0, s0, b0), (w1, s1, b1) in self.layers:
            if delta is None:
                x, sx = ops.rms_norm_fp8(stream, norm, eps=self.norm_eps)
            else:
                x, sx, stream = ops.rms_norm_fp8(delta, norm, residual=stream, eps=self.norm_eps)
            x = first(x, w0, bias=b0, activation=self.activation, x_scale=sx, weight_scale=s0,
                      **more)
            x, sx = ops.quantize_fp8(x)
            delta = ops.linear(x, w1, bias=b1, x_scale=sx, weight_scale=s1, **more)
        return _energies(stream, delta, types, self.norm_eps, *self.ends)


class ElementNetwork(nn.Module):
    """Per-atom energies [N] (float32) of descriptors [N, inputs] and element indices [N], by a
    network of its own for each element: ``head . act(W q + b) - shared_bias``, as NEP's.

    An atom whose index is no element's gets ``-shared_bias``. dtype: torch.bfloat16 or
    torch.float16, of the hidden layer.
    """

    def __init__(self, n_elements, inputs, hidden, activation="tanh", dtype=torch.bfloat16):
        super().__init__()
        if min(n_elements, inputs, hidden) <= 0:
            raise ValueError("ElementNetwork dimensions must be positive.")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be float16 or bfloat16, not {dtype}.")
        self.activation, self.dtype = str(activation).strip().lower(), dtype
        self.register_buffer("q_scaler", torch.ones(inputs))
        self.weight, self.bias = _stack(n_elements, hidden, inputs)
        # a table's rows with float32 gradients; the last one for atoms of no element
        self.head = nn.Embedding(n_elements + 1, hidden, padding_idx=n_elements)
        bound = 1.0 / math.sqrt(hidden)
        with torch.no_grad():
            self.head.weight[:n_elements].uniform_(-bound, bound)
        self.shared_bias = nn.Parameter(torch.zeros(1))

    @classmethod
    def from_nep(cls, model, dtype=torch.bfloat16):
        """The networks of a NEP model (``rune_b200.nep.plugin``), their weights copied."""
        mlps = [model.element_mlps[e] for e in model.elements]
        net = cls(len(mlps), model.input_dim, mlps[0][0].out_features, dtype=dtype)
        with torch.no_grad():
            net.q_scaler.copy_(model.q_scaler)
            net.shared_bias.copy_(model.shared_bias)
            for i, mlp in enumerate(mlps):
                net.weight[i].copy_(mlp[0].weight)
                net.bias[i].copy_(mlp[0].bias)
                net.head.weight[i].copy_(mlp[2].weight[0])
        return net.to(model.q_scaler.device)

    def forward(self, descriptors, types):
        elements = self.weight.shape[0]
        groups = ops.row_groups(types, elements)
        x = ops.to_groups((descriptors * self.q_scaler).to(self.dtype), groups)
        h = ops.grouped_linear(x, self.weight.to(self.dtype), groups,
                               bias=self.bias.to(self.dtype), activation=self.activation)
        rows = torch.where((types >= 0) & (types < elements), types, elements)
        return (ops.from_groups(h, groups).float() * self.head(rows)).sum(-1) - self.shared_bias
