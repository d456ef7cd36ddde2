"""8-bit activation checkpoints, and the linear layer that trains from them.

A training step keeps each layer's input for the weight gradient. Kept as 8-bit
codes it takes a little over half the bytes of bf16, a quarter of fp32, as the
LSTM cells' gate streams do for theirs; unlike those bounded values, activations
need a scale, one for each 32 values of a row:

    e     = max(floor(log2 max|v|) - 6, -126)         kept as the byte e + 127
    code  = clamp(rint(v / 2^e), -127, 127)           int8
    value = code * 2^e                                |value - v| <= max|v| / 127,
                                                      or 2^-127 where that is more

The scale is a power of two, so a kept value has at most seven significant bits
and is exact in bf16 and fp16: products take it as it is. A group with a value
that is not finite restores as NaN throughout.

- :func:`save8` / :func:`load8`: a tensor to codes and back.
- :func:`linear8`: ``x @ weight.T + bias`` with its gradient; only the codes of
  ``x`` live from the forward to the backward pass.
- :func:`weight_grad8`: the gradient of weight and bias from such codes.

GPU tensors run the HIP kernels, CPU tensors a plain torch form of the same
definition.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import ext

GROUP = 32  # values that share a scale
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


@dataclass(frozen=True)
class Saved8:
    """A tensor as 8-bit codes: rows are its last axis, padded to groups of 32."""

    codes: torch.Tensor   # int8  [rows, ceil(F / 32) * 32]
    scales: torch.Tensor  # uint8 [rows, ceil(F / 32)]
    shape: torch.Size
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as [rows, F] with unit stride along a row; copied only if it has to be."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES:
        raise ValueError(f"{what} must be a float32, bfloat16 or float16 tensor, got {getattr(x, 'dtype', type(x))}")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what} must have a last axis that is not empty, got shape {tuple(x.shape)}")
    F = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(x.numel() // F, F)
    return x if F == 1 or x.stride(1) == 1 else x.contiguous()


def codes_eager(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of [rows, F] in plain torch."""
    w = torch.nn.functional.pad(x.float(), (0, -x.shape[1] % GROUP))
    w = w.reshape(x.shape[0], w.shape[1] // GROUP, GROUP)
    field = (w.abs().amax(-1).view(torch.int32) >> 23) & 255
    scale = torch.where(field == 255, 255, (field - 6).clamp_min(1))
    inv = ((254 - scale).clamp_min(0) << 23).view(torch.float32).unsqueeze(-1)
    codes = (w * inv).round().clamp(-127, 127)
    codes = torch.where((scale == 255).unsqueeze(-1), torch.zeros_like(codes), codes)
    return codes.to(torch.int8).flatten(1), scale.to(torch.uint8)


def values_eager(codes: torch.Tensor, scales: torch.Tensor, F: int) -> torch.Tensor:
    """[rows, F] in float32 of codes in plain torch."""
    step = (scales.to(torch.int32) << 23).view(torch.float32)
    step = torch.where(scales == 255, torch.full_like(step, float("nan")), step)
    w = codes.reshape(*scales.shape, GROUP).float() * step.unsqueeze(-1)
    return w.reshape(codes.shape)[:, :F]


def save8(x: torch.Tensor) -> Saved8:
    """The 8-bit codes of ``x``, groups of 32 along its last axis. Codes carry no
    gradient: this is what a backward pass keeps, not a layer."""
    rows = _rows(x, "x")
    if rows.is_cuda:
        codes, scales = ext().save8(rows)
    else:
        codes, scales = codes_eager(rows.detach())
    return Saved8(codes, scales, x.shape, x.dtype)


def _check_saved(saved: Saved8, what: str = "saved") -> int:
    """The row length of ``saved``; raises where its parts do not belong together."""
    if not isinstance(saved, Saved8):
        raise ValueError(f"{what} must be a Saved8, got {type(saved)}")
    shape = torch.Size(saved.shape)
    if len(shape) == 0 or shape[-1] == 0 or saved.dtype not in _DTYPES:
        raise ValueError(f"{what}: no tensor of shape {tuple(shape)} and type {saved.dtype} is kept")
    F = shape[-1]
    N, groups = shape.numel() // F, -(-F // GROUP)
    if (saved.codes.shape != (N, groups * GROUP) or saved.scales.shape != (N, groups)
            or saved.codes.dtype != torch.int8 or saved.scales.dtype != torch.uint8
            or saved.codes.device != saved.scales.device
            or not saved.codes.is_contiguous() or not saved.scales.is_contiguous()):
        raise ValueError(f"{what}: codes and scales do not match shape {tuple(saved.shape)}")
    return F


def load8(saved: Saved8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that ``saved`` stands for, in its own type or in ``dtype``.
    Exact in float32 and bfloat16; float16 where the saved tensor was."""
    F = _check_saved(saved)
    dtype = saved.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    if saved.codes.is_cuda:
        out = ext().load8(saved.codes, saved.scales, F, dtype)
    else:
        out = values_eager(saved.codes, saved.scales, F).to(dtype)
    return out.reshape(saved.shape)


def weight_grad8(
    dy: torch.Tensor, saved: Saved8, *, bias: bool = False, dtype: Optional[torch.dtype] = None
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(dW, db) of a linear layer whose input was kept as ``saved``:
    ``dW = dy^T x8`` as [O, F] and ``db`` the sum of ``dy``'s rows (None without
    ``bias``), in ``dtype`` (default: dy's). Sums are held in 32 bits."""
    F = _check_saved(saved)
    dy2 = _rows(dy, "dy")
    if dy2.shape[0] != saved.codes.shape[0] or dy.shape[:-1] != saved.shape[:-1]:
        raise ValueError(f"dy of shape {tuple(dy.shape)} does not belong to an input of shape {tuple(saved.shape)}")
    if dy2.device != saved.codes.device:
        raise ValueError(f"dy is on {dy2.device}, the codes are on {saved.codes.device}")
    dtype = dy.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    O = dy2.shape[1]
    if dy2.is_cuda:
        if dy2.dtype == torch.float16 and saved.dtype != torch.float16:
            dy2 = dy2.float()  # the kept values are exact in float16 only if they came from it
        dw = torch.empty((O, F), dtype=dtype, device=dy2.device)
        db = torch.empty((O,), dtype=dtype, device=dy2.device) if bias else None
        ext().weight_grad8(dy2, saved.codes, saved.scales, dw, db)
        return dw, db
    dyf = dy2.detach().float()
    dw = dyf.t() @ values_eager(saved.codes, saved.scales, F)
    return dw.to(dtype), dyf.sum(0).to(dtype) if bias else None


class _Linear8(torch.autograd.Function):
    """The CPU form; the GPU's is in hip/autograd.cpp."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        y = torch.nn.functional.linear(x, weight.to(x.dtype), None if bias is None else bias.to(x.dtype))
        saved = save8(x) if ctx.needs_input_grad[1] else None
        ctx.x_shape, ctx.x_dtype = x.shape, x.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(weight, *((saved.codes, saved.scales) if saved is not None else (None, None)))
        return y

    @staticmethod
    def backward(ctx, dy):
        first_order("linear8")
        weight, codes, scales = ctx.saved_tensors
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = torch.matmul(dy, weight.to(ctx.x_dtype))
        if ctx.needs_input_grad[1]:
            dw, _ = weight_grad8(dy, Saved8(codes, scales, ctx.x_shape, ctx.x_dtype), dtype=weight.dtype)
        if ctx.needs_input_grad[2]:
            db = dy.reshape(-1, dy.shape[-1]).sum(0, dtype=torch.float32).to(ctx.bias_dtype)
        return dx, dw, db


def first_order(what: str) -> None:
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what}: the gradient has no gradient of its own (create_graph)")


def linear8(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ weight.T + bias`` as ``torch.nn.functional.linear`` has it, keeping
    the 8-bit codes of ``x`` for the backward pass instead of ``x``.

    ``x`` [..., F] sets the type that the products run in; ``weight`` [O, F] and
    ``bias`` [O] may be of another one (32-bit masters beside 16-bit
    activations), and their gradients come in their own types. Under autocast
    ``x`` is taken in the autocast type. The gradient of ``x`` does not depend on
    the codes; the weight gradient is ``dy^T x8``.
    """
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError("x must be a tensor with at least one axis")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight must be [O, F] with neither empty, got {tuple(weight.shape)}")
    if x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x has {x.shape[-1]} features, weight {weight.shape[1]}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    kind = x.device.type
    for t, what in ((x, "x"), (weight, "weight"), (bias, "bias")):
        if t is not None and t.dtype not in _DTYPES:
            raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
        if t is not None and t.device != x.device:
            raise ValueError(f"{what} is on {t.device}, x on {x.device}")
    if torch.is_autocast_enabled(kind):
        x = x.to(torch.get_autocast_dtype(kind))
    if x.is_cuda:
        return ext().linear8(x, weight, bias)
    with torch.autocast(kind, enabled=False):
        return _Linear8.apply(x, weight, bias)
