"""The Möbius scalar network in mixed precision, trainable: projection, residual blocks, head.

The engine evaluates Möbius models in float32 without parameter gradients. ``ScalarNetwork`` is
the same per-atom network (rune/mobius/model.py:256-305 without messages, layers.py:26-89) on the
operators of ``rune_b200.ops``: float32 parameters under the reference's names, 16-bit products
with float32 accumulation, gradients for all of them. For distilling a model into it, or for
adapting a checkpoint's network and serving many atoms' energies where the caller has their
descriptors (the engine computes its own inside the kernels and returns none); no forces.
``quantized`` gives an 8-bit copy for serving.

A block adds its output to the residual stream in the next block's normalisation, so the stream
is read and written once per block.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import ops
from .mobius.model import ElementwiseLinearHead, ResidualBlock, RMSNorm


class ScalarNetwork(nn.Module):
    """Per-atom energies [N] (float32) of descriptors [N, inputs] and element indices [N].

    gated: the blocks' first layer is ``act(x Wg^T + bg) * (x Wu^T + bu)``; ``ffn.0`` then holds
    2 * ffn rows, the gate's first. dtype: torch.bfloat16 or torch.float16, of the states.
    """

    def __init__(self, n_elements, inputs, hidden, ffn, blocks, activation="silu", gated=False,
                 norm_eps=1.0e-8, dtype=torch.bfloat16):
        super().__init__()
        if min(n_elements, inputs, hidden, ffn) <= 0 or blocks < 0:
            raise ValueError("ScalarNetwork dimensions must be positive.")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be float16 or bfloat16, not {dtype}.")
        self.activation, self.gated, self.dtype = str(activation).strip().lower(), bool(gated), dtype
        self.norm_eps = float(norm_eps)
        self.register_buffer("q_scaler", torch.ones(inputs))
        self.input_projection = nn.Linear(inputs, hidden)
        self.element_embedding = nn.Embedding(n_elements, hidden)
        self.residual_blocks = nn.ModuleList(
            ResidualBlock(hidden, ffn, activation, norm_eps=norm_eps) for _ in range(blocks))
        if gated:
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
        as it is now, its weights laid out; later changes of the network do not reach it."""
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
