"""Linear attention with a decay for each head: a recurrence whose cost grows with the number of pixels, not its square.

    S_t = exp(log_decay_h) S_{t-1} + k_t v_t^T,    o_t = scale q_t^T S_t

`linear_attention` runs whole sequences (training, or an image at once) in chunks, `step` advances one token with the
state kept between calls.  Both use the same state [B, H, Dk, Dv] in fp32, so a prompt can be run at once and continued token
by token.  Sequences are [B, T, H, D] (channel last, like the optimisation layers' public layout), fp32, fp16 or bf16."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.graph import increment_version

from . import _lib
from ._tensor import DTYPES, check_tensor, first_order, has_tangent, launch, on_device, ptr, wants_grad

MAX_HEAD = 128
_ARRAYS = {n: ctypes.c_longlong * n for n in (6, 9, 12)}


def _strides(*tensors):
    """HOST array of the strides, in elements, of every dimension but the last."""
    flat = [s for t in tensors for s in t.stride()[:-1]]
    return _ARRAYS[len(flat)](*flat)


def _check(q, k, v, log_decay, state, lengths, dims: int):
    check_tensor(q, "q", contiguous=False)
    if q.dim() != dims or v.dim() != dims:
        raise RuntimeError(f"q, k, v must have {dims} dimensions")
    check_tensor(k, "k", q.dtype, q.device, q.shape, contiguous=False)
    check_tensor(v, "v", q.dtype, q.device, (*q.shape[:-1], v.shape[-1]), contiguous=False)
    h, dk, dv = q.shape[-2], q.shape[-1], v.shape[-1]
    if h < 1 or not (1 <= dk <= MAX_HEAD and 1 <= dv <= MAX_HEAD):
        raise RuntimeError(f"there must be a head, and head sizes must be within 1..{MAX_HEAD}")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            raise RuntimeError(f"the last dimension of {name} must be contiguous")
    check_tensor(log_decay, "log_decay", torch.float32, q.device, (h,))
    if state is not None:
        check_tensor(state, "state", torch.float32, q.device, (q.shape[0], h, dk, dv))
    if lengths is not None:
        check_tensor(lengths, "lengths", torch.int32, q.device, (q.shape[0],))


def forward(q, k, v, log_decay, state=None, lengths=None, scale: Optional[float] = None):
    """(out [B, T, H, Dv], end state [B, H, Dk, Dv], starts): starts is what the backward pass needs of the forward pass."""
    _check(q, k, v, log_decay, state, lengths, 4)
    b, t, h, dk = q.shape
    dv = v.shape[-1]
    scale = dk ** -0.5 if scale is None else float(scale)
    lib = _lib.load()
    out = torch.empty((b, t, h, dv), dtype=q.dtype, device=q.device)
    end = torch.empty((b, h, dk, dv), dtype=torch.float32, device=q.device)
    segments = on_device(q.device, lib.cnl_linattn_segments, b, t, h, dk, dv, DTYPES[q.dtype])
    if segments < 1:
        raise RuntimeError("linear attention: " + _lib.last_error())
    starts = torch.empty((b, h, segments, dk, dv), dtype=torch.float32, device=q.device) if segments > 1 else None
    launch("linear attention forward", lib.cnl_linattn_forward, q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(),
           _strides(q, k, v), log_decay.data_ptr(), ptr(lengths), ptr(state), out.data_ptr(), end.data_ptr(), ptr(starts), b, t, h,
           dk, dv, scale, DTYPES[q.dtype])
    return out, end, starts


def backward(grad_out, grad_state, q, k, v, log_decay, state, lengths, starts, scale: Optional[float] = None, want_state: bool = True):
    """(g_q, g_k, g_v, g_state) from the gradients of the output and of the end state (the latter may be None); g_state, the
    gradient of the carried state, is None unless wanted."""
    _check(q, k, v, log_decay, state, lengths, 4)
    b, t, h, dk = q.shape
    dv = v.shape[-1]
    scale = dk ** -0.5 if scale is None else float(scale)
    check_tensor(grad_out, "grad_out", q.dtype, q.device, (b, t, h, dv), contiguous=False)
    if grad_out.stride(-1) != 1 and dv > 1:
        raise RuntimeError("the last dimension of grad_out must be contiguous")
    if grad_state is not None:
        check_tensor(grad_state, "grad_state", torch.float32, q.device, (b, h, dk, dv))
    new = lambda *s, dtype=q.dtype: torch.empty(s, dtype=dtype, device=q.device)  # noqa: E731
    g_q, g_k, g_v = new(b, t, h, dk), new(b, t, h, dk), new(b, t, h, dv)
    g_state = new(b, h, dk, dv, dtype=torch.float32) if want_state else None
    scratch = None if starts is None else torch.empty_like(starts)
    launch("linear attention backward", _lib.load().cnl_linattn_backward, q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(),
           grad_out.data_ptr(), _strides(q, k, v, grad_out), log_decay.data_ptr(), ptr(lengths), ptr(state), ptr(starts),
           ptr(grad_state), g_q.data_ptr(), g_k.data_ptr(), g_v.data_ptr(), ptr(g_state), ptr(scratch), b, t, h, dk, dv, scale,
           DTYPES[q.dtype])
    return g_q, g_k, g_v, g_state


def _rows(t):
    """t with a contiguous last dimension (a slice of a wider projection stays where it is)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class LinearAttentionFunction(Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale):
        q, k, v = _rows(q), _rows(k), _rows(v)
        state = None if state is None else state.contiguous()
        out, end, starts = forward(q, k, v, log_decay, state, lengths, scale)
        ctx.save_for_backward(q, k, v, log_decay, state, lengths, starts)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, end

    @staticmethod
    @first_order
    def backward(ctx, grad_out, grad_state):
        q, k, v, log_decay, state, lengths, starts = ctx.saved_tensors
        if grad_out is None and grad_state is None:
            return (None,) * 7
        if grad_out is None:
            grad_out = torch.zeros((*q.shape[:-1], v.shape[-1]), dtype=q.dtype, device=q.device)
        grad_state = None if grad_state is None else grad_state.contiguous()
        g_q, g_k, g_v, g_state = backward(_rows(grad_out), grad_state, q, k, v, log_decay, state, lengths, starts, ctx.scale,
                                          ctx.needs_input_grad[4])
        return g_q, g_k, g_v, None, g_state, None, None


def linear_attention(q, k, v, log_decay, *, state=None, lengths=None, scale: Optional[float] = None):
    """q, k [B, T, H, Dk], v [B, T, H, Dv] -> (out [B, T, H, Dv], end state [B, H, Dk, Dv] fp32).

    log_decay [H] fp32, at most 0, is a constant; state (optional) is what came before; lengths [B] int32 (optional): tokens
    at or behind a sequence's length are not read and give zeros (values are held to 0..T).  scale defaults to Dk ** -0.5.
    A token that is not finite makes all later outputs of its head not finite, and may make those of up to 127 earlier ones
    (a chunk meets as one product); sequences of the batch do not touch one another."""
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("log_decay is a constant of the layer: there is no gradient for it")
    if wants_grad(q, k, v, state) or has_tangent(log_decay):
        return LinearAttentionFunction.apply(q, k, v, log_decay, state, lengths, scale)
    return forward(_rows(q), _rows(k), _rows(v), log_decay, None if state is None else state.contiguous(), lengths, scale)[:2]


def step(q, k, v, log_decay, state, *, scale: Optional[float] = None):
    """One token: q, k [B, H, Dk], v [B, H, Dv] -> out [B, H, Dv]; state [B, H, Dk, Dv] is updated in place.  No gradient."""
    if wants_grad(q, k, v, state) or has_tangent(log_decay):
        raise RuntimeError("step keeps no gradient: call it under torch.no_grad()")
    q, k, v = _rows(q), _rows(k), _rows(v)
    if state is None:
        raise RuntimeError("step needs a state (zeros for a new sequence)")
    _check(q, k, v, log_decay, state, None, 3)
    b, h, dk = q.shape
    dv = v.shape[-1]
    out = torch.empty((b, h, dv), dtype=q.dtype, device=q.device)
    launch("linear attention step", _lib.load().cnl_linattn_step, q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(),
           _strides(q, k, v), log_decay.data_ptr(), state.data_ptr(), out.data_ptr(), b, h, dk, dv,
           dk ** -0.5 if scale is None else float(scale), DTYPES[q.dtype])
    if not state.is_inference():
        increment_version(state)                 # a graph that has kept this state refuses to use it, as after any in-place call
    return out


class LinearAttention(nn.Module):
    """Token mixer over [N, T, C] or [N, H, W, C] (pixels in raster order): projections, linear attention, projection.

    forward(x, state=None, lengths=None) -> (out, state); step(x [N, C], state) -> out.  Memories of the heads run from
    2^first to 2^last tokens; the decays stay fp32 whatever type the module is brought to."""

    def __init__(self, channels: int, heads: int, first: float = 2.0, last: float = 11.0):
        super().__init__()
        if channels % heads or channels // heads > MAX_HEAD:
            raise ValueError(f"{heads} heads must divide {channels} channels into at most {MAX_HEAD} each")
        self.heads = heads
        self.qkv = nn.Linear(channels, 3 * channels, bias=False)
        self.out = nn.Linear(channels, channels, bias=False)
        self.register_buffer("log_decay", -torch.exp2(-torch.linspace(first, last, heads, dtype=torch.float32)))

    def _apply(self, fn, recurse=True):
        decay = self.log_decay
        super()._apply(fn, recurse)
        if self.log_decay.dtype != torch.float32:        # the weights' type is not the memories': bf16 would change their lengths
            self.log_decay = decay.to(self.log_decay.device)
        return self

    def forward(self, x, state=None, lengths=None):
        n, c = x.shape[0], x.shape[-1]
        q, k, v = self.qkv(x).view(n, x.shape[1:-1].numel(), 3, self.heads, c // self.heads).unbind(2)
        o, state = linear_attention(q, k, v, self.log_decay.float(), state=state, lengths=lengths)
        return self.out(o.reshape(x.shape)), state

    def new_state(self, n: int):
        d = self.out.weight.shape[0] // self.heads
        return torch.zeros(n, self.heads, d, d, dtype=torch.float32, device=self.log_decay.device)

    def step(self, x, state):
        q, k, v = self.qkv(x).view(x.shape[0], 3, self.heads, x.shape[-1] // self.heads).unbind(1)
        return self.out(step(q, k, v, self.log_decay.float(), state).reshape(x.shape))
