"""Norms before and after a network block, fused with the block's gate, residual scale and residual sum.

    h = N(x; w, b)                                        pre_norm
    y = x + scale * a(gate) * N(u; w, b)                  residual_norm: u is the block's output
    h = N(y; next_weight, next_bias)                      ... and the norm in front of the next block, in the same pass

N is the rms norm (kind "rms") or the layer norm ("layer") over the last dimension, a the sigmoid or the identity.  The
gate has the stream's shape, or one row for a whole image (size 1 in the dimensions it is shared over).  With
checkpoint="int8" / "e4m3" the backward pass reads 8-bit checkpoints (see `ckpt8`) of x, u and a full gate, written by the
forward pass, instead of keeping the tensors alive."""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn
from torch.autograd import Function

from . import _lib
from ._tensor import DTYPES, check_tensor, first_order, launch, on_device, ptr, wants_grad
from .ckpt8 import BLOCK, format_code
from .dist import allreduce_scalar_grads

KINDS = {"rms": 0, "layer": 1}
GATES = {"identity": 0, "sigmoid": 1}
MAX_CHANNELS = 8192


def _gate_mode(x, gate):
    """(mode, groups): 0 no gate (or none to read), 1 of x's shape, 2 shared by the rows of each of `groups` groups."""
    if gate is None:
        return 0, 1
    if gate.dim() > x.dim() or gate.dim() < 1 or gate.shape[-1] != x.shape[-1]:
        raise RuntimeError(f"gate {list(gate.shape)} does not go with x {list(x.shape)}")
    if gate.shape == x.shape:
        return 1, 1
    lead = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape[:-1])
    groups, i = 1, 0
    while i < len(lead) and lead[i] == x.shape[i]:
        groups *= lead[i]
        i += 1
    if any(n != 1 for n in lead[i:]):
        raise RuntimeError(f"gate {list(gate.shape)} must have x's shape {list(x.shape)}, or size 1 in all dimensions between "
                           "some leading ones and the last")
    return (2, groups) if groups else (0, 1)     # the gates of no images: there is no row either


def _check(x, u, gate, scale, weight, bias, next_weight, next_bias):
    check_tensor(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise RuntimeError(f"x must have 1 to {MAX_CHANNELS} channels in its last dimension")
    d = x.shape[-1]
    device = x.device
    if u is not None:
        check_tensor(u, "u", x.dtype, device, x.shape)
    if gate is not None:
        check_tensor(gate, "gate", x.dtype, device)
    first = weight if u is not None else next_weight
    if first is None:
        raise RuntimeError("a norm needs its weight")
    wdtype = first.dtype
    if wdtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"parameters must be {x.dtype} or float32, not {wdtype}")
    for t, name in ((scale, "scale"), (weight, "weight"), (bias, "bias"), (next_weight, "next_weight"), (next_bias, "next_bias")):
        if t is not None:
            check_tensor(t, name, wdtype, device, (d,))
    if next_bias is not None and next_weight is None:
        raise RuntimeError("next_bias needs next_weight")
    return wdtype


def forward(x, u, gate, scale, weight, bias, next_weight, next_bias, kind="rms", eps=1e-6, gate_kind="sigmoid", fmt=None,
            keep=False):
    """(y, h, stats, codes, scales).  u None: the norm alone (next_weight, next_bias), y is None.  keep: also what the backward
    pass needs (stats, and the codes and scales of `fmt`)."""
    if kind not in KINDS:
        raise RuntimeError(f"kind must be 'rms' or 'layer', not {kind!r}")
    if gate_kind not in GATES:
        raise RuntimeError(f"gate_kind must be 'sigmoid' or 'identity', not {gate_kind!r}")
    code = format_code(fmt) if keep else _lib.CKPT_NONE
    wdtype = _check(x, u, gate, scale, weight, bias, next_weight, next_bias)
    mode, groups = _gate_mode(x, gate)
    d = x.shape[-1]
    rows = x.numel() // d
    y = None if u is None else torch.empty_like(x)
    h = None if next_weight is None else torch.empty_like(x)
    stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if keep else None
    codes = scales = None
    if code:
        planes = 1 if u is None else 3 if mode == 1 else 2
        codes = torch.empty((planes, rows, d), dtype=torch.uint8, device=x.device)
        scales = torch.empty((planes, rows, -(-d // BLOCK)), dtype=torch.uint8, device=x.device)
    launch("block norm forward", _lib.load().cnl_blocknorm_forward, x.device, x.data_ptr(), ptr(u), ptr(gate), ptr(scale),
           ptr(weight), ptr(bias), ptr(next_weight), ptr(next_bias), ptr(y), ptr(h), ptr(stats), ptr(codes), ptr(scales), rows, d,
           groups, mode, GATES[gate_kind], KINDS[kind], eps, DTYPES[x.dtype], DTYPES[wdtype], code)
    return y, h, stats, codes, scales


def _contiguous(*tensors):
    return [None if t is None else t.contiguous() for t in tensors]


class BlockNormFunction(Function):
    """forward(x, u, gate, scale, weight, bias, next_weight, next_bias, kind, eps, gate_kind, fmt) -> y, h or (y, h)."""

    @staticmethod
    def forward(ctx, x, u, gate, scale, weight, bias, next_weight, next_bias, kind, eps, gate_kind, fmt):
        x, u, gate, scale, weight, bias, next_weight, next_bias = _contiguous(x, u, gate, scale, weight, bias, next_weight, next_bias)
        y, h, stats, codes, scales = forward(x, u, gate, scale, weight, bias, next_weight, next_bias, kind, eps, gate_kind, fmt, True)
        mode, groups = _gate_mode(x, gate)
        packed = fmt is not None
        ctx.save_for_backward(None if packed or next_weight is None else x, None if packed else u,
                              None if packed and mode == 1 else gate, codes, scales, stats, scale, weight, bias, next_weight,
                              next_bias)
        ctx.set_materialize_grads(False)
        ctx.meta = (x.shape, x.dtype, x.device, mode, groups, None if gate is None else gate.shape, GATES[gate_kind], KINDS[kind],
                    format_code(fmt))
        if u is None:
            return h
        return y if h is None else (y, h)

    @staticmethod
    @first_order
    def backward(ctx, *grads):
        x, u, gate, codes, scales, stats, scale, weight, bias, next_weight, next_bias = ctx.saved_tensors
        shape, dtype, device, mode, groups, gate_shape, sigmoid, layer, code = ctx.meta
        if weight is None:
            g_y, g_h = None, grads[0]
        else:
            g_y, g_h = grads[0], grads[1] if next_weight is not None else None
        if g_y is None and g_h is None:
            return (None,) * 12
        g_y, g_h = (None if g is None else g.contiguous() for g in (g_y, g_h))
        for g, name in ((g_y, "gradient of y"), (g_h, "gradient of h")):
            if g is not None:
                check_tensor(g, name, dtype, device, shape)
        need = ctx.needs_input_grad
        d = shape[-1]
        rows = shape.numel() // d
        wdtype = (weight if weight is not None else next_weight).dtype
        like = g_y if g_y is not None else g_h
        g_x = torch.empty_like(like) if need[0] else None
        g_u = torch.empty_like(like) if need[1] else None
        g_gate = torch.empty(gate_shape, dtype=dtype, device=device) if need[2] else None
        g_params = [None] * 5
        wanted = [i for i in range(5) if need[3 + i]]
        if wanted:
            for i, g in zip(wanted, torch.empty((len(wanted), d), dtype=wdtype, device=device).unbind(0)):
                g_params[i] = g
        lib = _lib.load()
        scratch = torch.empty(on_device(device, lib.cnl_blocknorm_scratch_bytes, rows, d, groups), dtype=torch.uint8, device=device)
        launch("block norm backward", lib.cnl_blocknorm_backward, device, ptr(x), ptr(u), ptr(gate), ptr(codes), ptr(scales),
               stats.data_ptr(), ptr(scale), ptr(weight), ptr(bias), ptr(next_weight), ptr(next_bias), ptr(g_y), ptr(g_h), ptr(g_x),
               ptr(g_u), ptr(g_gate), *(ptr(g) for g in g_params), scratch.data_ptr(), rows, d, groups, mode, sigmoid, layer,
               DTYPES[dtype], DTYPES[wdtype], code)
        return (g_x, g_u, g_gate, *g_params, None, None, None, None)


def pre_norm(x, weight, bias=None, *, kind: str = "rms", eps: float = 1e-6, checkpoint: Optional[str] = None):
    """N(x; weight, bias) over the last dimension."""
    if wants_grad(x, weight, bias):
        return BlockNormFunction.apply(x, None, None, None, None, None, weight, bias, kind, eps, "sigmoid", checkpoint)
    format_code(checkpoint)
    return forward(*_contiguous(x, None, None, None, None, None, weight, bias), kind, eps)[1]


def residual_norm(x, u, weight, bias=None, *, gate=None, gate_kind: str = "sigmoid", scale=None, next_weight=None, next_bias=None,
                  kind: str = "rms", eps: float = 1e-6, checkpoint: Optional[str] = None):
    """y = x + scale * a(gate) * N(u; weight, bias); with next_weight (y, N(y; next_weight, next_bias))."""
    if wants_grad(x, u, weight, bias, gate, scale, next_weight, next_bias):
        return BlockNormFunction.apply(x, u, gate, scale, weight, bias, next_weight, next_bias, kind, eps, gate_kind, checkpoint)
    format_code(checkpoint)
    y, h = forward(*_contiguous(x, u, gate, scale, weight, bias, next_weight, next_bias), kind, eps, gate_kind)[:2]
    return y if h is None else (y, h)


class PreNorm(nn.Module):
    """forward(x [..., channels]) -> N(x)."""

    def __init__(self, channels: int, kind: str = "rms", bias: bool = False, eps: float = 1e-6, checkpoint: Optional[str] = None):
        super().__init__()
        self.kind, self.eps, self.checkpoint = kind, eps, checkpoint
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels)) if bias else None

    def forward(self, x):
        return pre_norm(x, self.weight, self.bias, kind=self.kind, eps=self.eps, checkpoint=self.checkpoint)


class ResidualNorm(nn.Module):
    """forward(x, u, gate=None) -> y, or with following=True (y, h): the norm after a block, its gate, learned residual scale
    and residual sum, and the norm in front of the next block."""

    def __init__(self, channels: int, kind: str = "rms", bias: bool = False, eps: float = 1e-6, scale: Optional[float] = 1.0,
                 gate_kind: str = "sigmoid", following: bool = True, checkpoint: Optional[str] = None):
        super().__init__()
        self.kind, self.eps, self.gate_kind, self.checkpoint = kind, eps, gate_kind, checkpoint
        vector = lambda v: nn.Parameter(torch.full((channels,), float(v)))  # noqa: E731
        self.weight = vector(1)
        self.bias = vector(0) if bias else None
        self.scale = None if scale is None else vector(scale)
        self.next_weight = vector(1) if following else None
        self.next_bias = vector(0) if following and bias else None

    def forward(self, x, u, gate=None):
        return residual_norm(x, u, self.weight, self.bias, gate=gate, gate_kind=self.gate_kind, scale=self.scale,
                             next_weight=self.next_weight, next_bias=self.next_bias, kind=self.kind, eps=self.eps,
                             checkpoint=self.checkpoint)

    def allreduce_parameter_grads(self) -> None:
        """Data-parallel step: sum the parameter gradients over all ranks."""
        for p in self.parameters():
            if p.grad is not None:
                allreduce_scalar_grads(p.grad)
