"""Activations kept in 8 bits for the backward pass.

At the layers' own resolution (8 x 32 x 384 x 1280 feature maps are half a gigabyte in fp32) what a network saves for its
backward pass is what fills the memory.  `store` / `restore` put a tensor away in 8.25 bits an element; `activation`
(GELU, SiLU) leaves the codes of its input in the same pass that computes its output and reads only them in the backward
pass; `blocknorm` and `QuadFittingFromFlow` take the same formats through their `checkpoint` argument.

Formats: thirty-two neighbouring elements of the flattened tensor share a power-of-two scale.  "int8": whole numbers
-127..127, error at most max|block| / 128; "e4m3": 8-bit floats, error at most 1/16 of the element.  Elements that are not
finite come back as NaN."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch import nn
from torch.autograd import Function

from . import _lib
from ._tensor import DTYPES, check_tensor, first_order, launch, wants_grad

FORMATS = {"int8": _lib.CKPT_INT8, "e4m3": _lib.CKPT_E4M3}
KINDS = {"gelu": _lib.ACT_GELU, "silu": _lib.ACT_SILU}
BLOCK = 32


def format_code(fmt: Optional[str]) -> int:
    if fmt is None:
        return _lib.CKPT_NONE
    if fmt not in FORMATS:
        raise RuntimeError(f"checkpoint format must be 'int8' or 'e4m3', not {fmt!r}")
    return FORMATS[fmt]


def _kind_code(kind: str) -> int:
    if kind not in KINDS:
        raise RuntimeError(f"activation must be 'gelu' or 'silu', not {kind!r}")
    return KINDS[kind]


@dataclass
class Stored8:
    """A tensor put away in 8 bits: codes [n] and scales [ceil(n / 32)] (uint8), and what it was."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype
    fmt: str

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def empty_codes(x: torch.Tensor):
    n = x.numel()
    return (torch.empty(n, dtype=torch.uint8, device=x.device),
            torch.empty(-(-n // BLOCK), dtype=torch.uint8, device=x.device))


def store(x: torch.Tensor, fmt: str = "int8") -> Stored8:
    """x (contiguous, fp32, fp16 or bf16) in 8 bits."""
    check_tensor(x, "x")
    code = format_code(fmt)
    if code == _lib.CKPT_NONE:
        raise RuntimeError("store needs a format")
    codes, scales = empty_codes(x)
    launch("ckpt8 store", _lib.load().cnl_ckpt8_store, x.device, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), x.numel(),
           DTYPES[x.dtype], code)
    return Stored8(codes, scales, x.shape, x.dtype, fmt)


def restore(stored: Stored8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The tensor a Stored8 stands for, of its own type or `dtype`, saturated to the type's finite range."""
    dtype = stored.dtype if dtype is None else dtype
    if dtype not in DTYPES:
        raise RuntimeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    n = stored.shape.numel()
    check_tensor(stored.codes, "codes", torch.uint8, shape=(n,))
    check_tensor(stored.scales, "scales", torch.uint8, stored.codes.device, (-(-n // BLOCK),))
    out = torch.empty(stored.shape, dtype=dtype, device=stored.codes.device)
    launch("ckpt8 restore", _lib.load().cnl_ckpt8_restore, out.device, stored.codes.data_ptr(), stored.scales.data_ptr(),
           out.data_ptr(), out.numel(), DTYPES[dtype], format_code(stored.fmt))
    return out


def forward(x: torch.Tensor, kind: str, fmt: Optional[str]):
    """(act(x), Stored8 of x); fmt None keeps nothing."""
    check_tensor(x, "x")
    y = torch.empty_like(x)
    codes, scales = empty_codes(x) if fmt is not None else (None, None)
    launch("activation forward", _lib.load().cnl_act8_forward, x.device, x.data_ptr(), y.data_ptr(),
           None if codes is None else codes.data_ptr(), None if scales is None else scales.data_ptr(), x.numel(),
           DTYPES[x.dtype], format_code(fmt) or _lib.CKPT_INT8, _kind_code(kind))
    return y, None if fmt is None else Stored8(codes, scales, x.shape, x.dtype, fmt)


def backward(stored: Stored8, grad: torch.Tensor, kind: str) -> torch.Tensor:
    """grad * act'(restored input)."""
    check_tensor(grad, "grad", stored.dtype, stored.codes.device, stored.shape)
    g = torch.empty_like(grad)
    launch("activation backward", _lib.load().cnl_act8_backward, grad.device, stored.codes.data_ptr(),
           stored.scales.data_ptr(), grad.data_ptr(), g.data_ptr(), grad.numel(), DTYPES[grad.dtype], format_code(stored.fmt),
           _kind_code(kind))
    return g


class Activation8Function(Function):
    @staticmethod
    def forward(ctx, x, kind, fmt):
        x = x.contiguous()
        check_tensor(x, "x")
        n = x.numel()
        y = torch.empty_like(x)
        # codes and scales in one allocation, the scales behind the codes
        packed = torch.empty(n + -(-n // BLOCK), dtype=torch.uint8, device=x.device)
        ctx.save_for_backward(packed)
        ctx.meta = meta = (DTYPES[x.dtype], format_code(fmt), _kind_code(kind))
        at = packed.data_ptr()
        launch("activation forward", _lib.load().cnl_act8_forward, x.device, x.data_ptr(), y.data_ptr(), at, at + n, n, *meta)
        return y

    @staticmethod
    @first_order
    def backward(ctx, grad):
        (packed,) = ctx.saved_tensors
        grad = grad.contiguous()
        n = grad.numel()
        g = torch.empty_like(grad)
        at = packed.data_ptr()
        launch("activation backward", _lib.load().cnl_act8_backward, grad.device, at, at + n, grad.data_ptr(), g.data_ptr(), n, *ctx.meta)
        return g, None, None


def activation(x: torch.Tensor, kind: str = "gelu", fmt: str = "int8") -> torch.Tensor:
    """act(x); the backward pass takes act' at x as its 8-bit checkpoint holds it, so x itself is not kept alive."""
    if format_code(fmt) == _lib.CKPT_NONE:
        raise RuntimeError("activation needs a format")
    if wants_grad(x):
        return Activation8Function.apply(x, kind, fmt)
    return forward(x.contiguous(), kind, None)[0]


class Activation8(nn.Module):
    """forward(x) -> act(x), kind "gelu" or "silu", its input kept in 8 bits for the backward pass."""

    def __init__(self, kind: str = "gelu", fmt: str = "int8"):
        super().__init__()
        _kind_code(kind)
        if format_code(fmt) == _lib.CKPT_NONE:
            raise RuntimeError("Activation8 needs a format")
        self.kind, self.fmt = kind, fmt

    def forward(self, x):
        return activation(x, self.kind, self.fmt)
