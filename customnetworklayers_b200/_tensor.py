"""Argument checks and launch plumbing shared by the network operators (`ckpt8`, `blocknorm`, `linattn`)."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def check_tensor(t, name: str, dtype=None, device=None, shape=None, contiguous: bool = True) -> None:
    if (t.dtype is dtype and t.device == device and (shape is None or t.shape == shape) and (not contiguous or t.is_contiguous())
            and t.is_cuda):
        return                                   # the usual case, in as few calls as it takes
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if contiguous and not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if dtype is None:
        if t.dtype not in DTYPES:
            raise RuntimeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    elif t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, not {t.dtype}")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} must be on {device}, not on {t.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name} must have shape {list(shape)}, not {list(t.shape)}")


def ptr(t):
    return None if t is None else t.data_ptr()


def on_device(device, fn, *args):
    """fn(*args) with `device` current."""
    if device.index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(device):
        return fn(*args)


def launch(what: str, fn, device, *args) -> None:
    """fn(*args, stream) on the current stream of `device`, with that device current."""
    index = device.index
    # the raw handle of the current stream; building a Stream object for it costs as much as half a launch
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch.cuda.current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc != 0:
        _lib.check(rc, what)


def has_tangent(*tensors) -> bool:
    """Whether a forward-mode derivative enters with one of the tensors."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def wants_grad(*tensors) -> bool:
    """Whether a derivative is asked for: a gradient, or a forward-mode one, which the autograd functions refuse."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or has_tangent(*tensors)


def first_order(backward):
    """once_differentiable whose bookkeeping is paid only by a caller that asked for a graph of the backward pass."""
    graphed = once_differentiable(backward)

    def run(ctx, *grads):
        return graphed(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run
