"""Pixel mixer in front of the optimisation layers: blocks of linear attention and a pixel-wise MLP between fused norms.

    h = pre_norm(x)
    per block:  x, h = residual_norm(x, attention(h), gate = W h)        gate, scale, residual sum and next norm in one pass
                x, h = residual_norm(x, MLP(h))

Runs [N, H, W, C] images (pixels in raster order) or [N, T, C] sequences at once, or one token at a time with the state of
every block kept by the caller.  `checkpoint` ("int8", "e4m3") keeps what the norms and the MLP's activation save for the
backward pass in 8 bits.  The projections are plain library products; under torch.autocast they, the attention and the
activation run in 16 bits, the norms and the stream in the type of x."""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .blocknorm import PreNorm, ResidualNorm
from .ckpt8 import Activation8
from .dist import allreduce_scalar_grads
from .linattn import LinearAttention


class PixelMixer(nn.Module):
    def __init__(self, channels: int, heads: int, depth: int = 2, hidden: Optional[int] = None, kind: str = "rms",
                 checkpoint: Optional[str] = None):
        super().__init__()
        if depth < 1:
            raise ValueError("a mixer has at least one block")
        hidden = 2 * channels if hidden is None else hidden
        self.pre = PreNorm(channels, kind, checkpoint=checkpoint)
        self.attention = nn.ModuleList(LinearAttention(channels, heads) for _ in range(depth))
        self.gate = nn.ModuleList(nn.Linear(channels, channels) for _ in range(depth))
        self.after_attention = nn.ModuleList(ResidualNorm(channels, kind, scale=0.5, checkpoint=checkpoint) for _ in range(depth))
        self.up = nn.ModuleList(nn.Linear(channels, hidden) for _ in range(depth))
        self.act = nn.GELU() if checkpoint is None else Activation8("gelu", checkpoint)
        self.down = nn.ModuleList(nn.Linear(hidden, channels) for _ in range(depth))
        self.after_mlp = nn.ModuleList(ResidualNorm(channels, kind, scale=0.5, following=i + 1 < depth, checkpoint=checkpoint)
                                       for i in range(depth))

    def _blocks(self, x, mix):
        h = self.pre(x)
        for i, gate in enumerate(self.gate):
            # (under autocast the projections leave 16 bits, the stream stays as it is)
            x, h = self.after_attention[i](x, mix(i, h).to(x.dtype), gate(h).to(x.dtype))
            out = self.after_mlp[i](x, self.down[i](self.act(self.up[i](h))).to(x.dtype))
            x, h = out if i + 1 < len(self.gate) else (out, None)
        return x

    def forward(self, x, states=None, lengths=None):
        """x [N, H, W, C] or [N, T, C] -> (x, states): one end state per block; states and lengths as in linear_attention."""
        ends = []

        def mix(i, h):
            u, end = self.attention[i](h, None if states is None else states[i], lengths)
            ends.append(end)
            return u

        return self._blocks(x, mix), ends

    def new_states(self, n: int):
        return [a.new_state(n) for a in self.attention]

    @torch.no_grad()
    def step(self, x, states):
        """x [N, C]: one token; states (from new_states or forward) are updated in place."""
        return self._blocks(x, lambda i, h: self.attention[i].step(h, states[i]))

    def allreduce_parameter_grads(self) -> None:
        """Data-parallel step: sum the parameter gradients, the projections' among them, over all ranks."""
        for p in self.parameters():
            if p.grad is not None:
                allreduce_scalar_grads(p.grad)
