"""``PredictionNet``: a prediction network with a selective state space in place of the LSTM.

Same place and interface as the reference's ``BaseDecoder`` (src/decoder/decoder.py:5-44): ``forward(inputs, length=None,
hidden=None) -> (outputs, hidden)``, embedding first, a projection to the joint's width last; ``rnnt_amd.greedy_decode``
and ``greedy_search_batch`` take it as their ``decoder``, ``rnnt_amd.JointNet.transducer_loss`` its outputs.  The state
that decoding carries has a fixed size, and a label sequence is one scan instead of one LSTM step after the other.

Per layer: ``LayerNorm -> Linear to (x, z) -> causal_conv(x) -> Linear to (dt, B, C) -> selective_scan -> Linear``, added
to the layer's input.  Embedding, convolution and scan are this package's kernels, the Linear layers library products.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn as nn

from .embedding import TokenEmbedding
from .state_space import causal_conv, causal_conv_step, selective_scan, selective_scan_step


class _StateLayer(nn.Module):
    def __init__(self, dim: int, inner: int, state: int, width: int):
        super().__init__()
        self.inner, self.state, self.rank = inner, state, max(1, math.ceil(dim / 16))
        self.norm = nn.LayerNorm(dim)
        self.in_proj = nn.Linear(dim, 2 * inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(inner, width).uniform_(-1, 1) / math.sqrt(width))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.x_proj = nn.Linear(inner, self.rank + 2 * state, bias=False)
        self.dt_proj = nn.Linear(self.rank, inner, bias=False)
        # steps between 1e-3 and 1e-1 to begin with, rates -1 .. -state
        step = torch.exp(torch.rand(inner) * (math.log(1e-1) - math.log(1e-3)) + math.log(1e-3))
        self.dt_bias = nn.Parameter(torch.log(torch.expm1(step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, state + 1, dtype=torch.float32)).repeat(inner, 1))
        self.D = nn.Parameter(torch.ones(inner))
        self.out_proj = nn.Linear(inner, dim, bias=False)

    def forward(self, u, lengths, conv_state, scan_state):
        x, z = self.in_proj(self.norm(u)).split(self.inner, dim=-1)
        # (the kernels take these parameters in fp32 whatever type the module was cast to)
        conv_weight, conv_bias, dt_bias, D = (p.float() for p in (self.conv_weight, self.conv_bias, self.dt_bias, self.D))
        A = -torch.exp(self.A_log.float())
        single = u.size(1) == 1 and lengths is None and conv_state is not None and not torch.is_grad_enabled()
        if single:
            x, conv_state = causal_conv_step(x[:, 0], conv_state, conv_weight, conv_bias)
            z = z[:, 0]
        else:
            x, conv_state = causal_conv(x, conv_weight, conv_bias, conv_state, lengths)
        rate, B, C = self.x_proj(x).split((self.rank, self.state, self.state), dim=-1)
        dt = self.dt_proj(rate)
        if single:
            y, scan_state = selective_scan_step(x, dt, A, B, C, scan_state, D=D, z=z, dt_bias=dt_bias)
            y = y[:, None]
        else:
            y, scan_state = selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=dt_bias, initial_state=scan_state, lengths=lengths)
        return u + self.out_proj(y), conv_state, scan_state


class PredictionNet(nn.Module):
    """Prediction network over state-space layers; see the module docstring.

    Args:
        vocab_size, embed_dim, output_size: tokens, width of the embedding and of the layers, width the joint takes.
        layers: number of layers.
        inner_dim: channels of convolution and scan (default ``2 * embed_dim``).
        state_size: states per channel, 8, 16 or 32.
        conv_width: taps of the convolution, 2, 3 or 4.
        padding_idx: token whose embedding row is zero and stays so (the reference: 0, the blank, which also starts every
            sequence); None: none.
        embed_scale: factor of the embedding, or ``"sqrt"``.
    """

    def __init__(self, vocab_size: int, embed_dim: int, output_size: int, layers: int = 1, inner_dim: Optional[int] = None,
                 state_size: int = 16, conv_width: int = 4, padding_idx: Optional[int] = 0, embed_scale=1.0):
        super().__init__()
        if state_size not in (8, 16, 32):
            raise ValueError("state_size must be 8, 16 or 32")
        if conv_width not in (2, 3, 4):
            raise ValueError("conv_width must be 2, 3 or 4")
        if layers < 1:
            raise ValueError("layers must be positive")
        inner_dim = 2 * embed_dim if inner_dim is None else inner_dim
        self.embedding = TokenEmbedding(vocab_size, embed_dim, padding_idx, embed_scale)
        self.layers = nn.ModuleList(_StateLayer(embed_dim, inner_dim, state_size, conv_width) for _ in range(layers))
        self.norm = nn.LayerNorm(embed_dim)
        self.output_proj = nn.Linear(embed_dim, output_size)

    def forward(self, inputs: torch.Tensor, length: Optional[torch.Tensor] = None,
                hidden: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
        """``inputs [B, U]`` tokens, ``length`` int32 or int64 ``[B]`` (None: all) -> ``(outputs [B, U, output_size], hidden)``.
        Rows from ``length`` on hold any token of the vocabulary (one outside it gives NaN, in the Linear layers' gradients too).
        ``hidden`` is ``(conv [layers, B, width - 1, inner], scan [layers, B, inner, state])``, None: zeros; it is not changed."""
        if inputs.dim() != 2:
            raise ValueError("inputs must be [B, U]")
        if length is not None:
            length = length.to(device=inputs.device, dtype=torch.int32)
        u = self.embedding(inputs)
        conv, scan = [], []
        for i, layer in enumerate(self.layers):
            c, s = (None, None) if hidden is None else (hidden[0][i], hidden[1][i])
            u, c, s = layer(u, length, c, s)
            conv.append(c)
            scan.append(s)
        return self.output_proj(self.norm(u)), (torch.stack(conv), torch.stack(scan))
