"""Gated linear recurrence: the sequence operator that can be split over time.

The LSTM cells (lstm_engine) walk a window token after token, since each gate
reads the last hidden state. Here gates come from the input alone:

    p = [x | r | z]                     one projection, z optional
    f_t = sigmoid(r_t)
    h_t = f_t h_{t-1} + (1 - f_t) x_t   elementwise, held in 32 bits
    y_t = h_t silu(z_t)                 (y_t = h_t without z)

so a long stream is a scan, computed in parallel over its tokens.

- :func:`gated_scan`: a batch of sequences, with its gradient (training, and
  the prompt of a stream).
- :func:`gated_step`: the next token of many streams, each with its state in a
  slot of a resident buffer (online scoring).

GPU tensors run the HIP kernels, CPU tensors a plain torch form of the same
definition.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ext
from .checkpoint8 import _DTYPES, codes_eager, first_order, values_eager

KEEP_EVERY = 16  # tokens between two kept states
_TOP = torch.finfo(torch.float32).max


# ------------------------------------------------------------------ plain torch
def _live(T: int, lengths: Optional[torch.Tensor], device) -> Optional[torch.Tensor]:
    if lengths is None:
        return None
    return (torch.arange(T, device=device)[None] < lengths[:, None]).unsqueeze(-1)


def _gate(r):
    """(holds, small): the smaller of k = sigmoid(-r) and f = sigmoid(r), k where the
    state is held (r >= 0). Either has all its digits that way; 1 - k near k = 1 has
    lost those of f, 1 - f near f = 1 those of k. (From exp, whose bits do not depend on
    a value's place in the tensor; torch.sigmoid's do, by the unit in the last place.)"""
    e = torch.exp(-r.abs())
    return r >= 0, e / (1 + e)


def _next(gate, x, h):
    """f h + k x, as two products: x - h may be more than the largest number."""
    holds, small = gate
    most, rest = torch.where(holds, h, x), torch.where(holds, x, h)
    return (most - small * most) + small * rest


def _scan_eager(p, dim, h0, live, start=None):
    """States before and after every token, float32. ``start``: the kept states,
    from which the recurrence goes on at every KEEP_EVERY-th token."""
    B, T = p.shape[:2]
    x = p[..., :dim]
    holds, small = _gate(p[..., dim : 2 * dim])
    h = h0
    before, after = torch.empty_like(x), torch.empty_like(x)
    for t in range(T):
        if start is not None and t % KEEP_EVERY == 0:
            h = start[:, t // KEEP_EVERY]
        before[:, t] = h
        n = _next((holds[:, t], small[:, t]), x[:, t], h)
        h = n if live is None else torch.where(live[:, t], n, h)
        after[:, t] = h
    return before, after, h


def _forward_eager(p, dim, h0, lengths):
    live = _live(p.shape[1], lengths, p.device)
    pf = p.float()
    before, after, last = _scan_eager(pf, dim, h0, live)
    y = after
    if p.shape[2] == 3 * dim:
        y = y * torch.nn.functional.silu(pf[..., 2 * dim :])
    if live is not None:
        y = torch.where(live, y, torch.zeros_like(y))
    return y.to(p.dtype), last, before[:, ::KEEP_EVERY].contiguous()


def _backward_eager(p, dim, lengths, states, dy, dh):
    """p in float32 as it was kept."""
    live = _live(p.shape[1], lengths, p.device)
    before, after, _ = _scan_eager(p, dim, None, live, states)
    x = p[..., :dim]
    holds, small = _gate(p[..., dim : 2 * dim])
    g, dp = dy.float(), torch.empty_like(p)
    if p.shape[2] == 3 * dim:
        z = p[..., 2 * dim :]
        s = torch.sigmoid(z)
        dp[..., 2 * dim :] = g * (s * (1 + z * (1 - s))) * after
        g = g * z * s
    c = dh
    for t in range(p.shape[1] - 1, -1, -1):
        gt = g[:, t] + c
        less = small[:, t] * gt
        more = gt - small[:, t] * gt.clamp(-_TOP, _TOP)  # an infinite gradient stays so: 1 less a share is more than 0
        dp[:, t, :dim] = torch.where(holds[:, t], less, more)
        dp[:, t, dim : 2 * dim] = (small[:, t] * before[:, t] - small[:, t] * x[:, t]) * more
        n = torch.where(holds[:, t], more, less)
        c = n if live is None else torch.where(live[:, t], n, c)
    if live is not None:
        dp = torch.where(live, dp, torch.zeros_like(dp))
    return dp, c


class _GatedScan(torch.autograd.Function):
    """The CPU form; the GPU's is in hip/autograd.cpp."""

    @staticmethod
    def forward(ctx, p, h0, lengths, dim, keep8):
        y, last, states = _forward_eager(p, dim, h0, lengths)
        codes = scales = None
        if keep8:
            codes, scales = codes_eager(p.reshape(-1, dim))
        ctx.dim, ctx.p_shape, ctx.p_dtype = dim, p.shape, p.dtype
        ctx.save_for_backward(None if keep8 else p, lengths, states, codes, scales)
        return y, last

    @staticmethod
    def backward(ctx, dy, dh):
        first_order("gated_scan")
        p, lengths, states, codes, scales = ctx.saved_tensors
        kept = p.float() if codes is None else values_eager(codes, scales, ctx.dim).reshape(ctx.p_shape)
        dp, dh0 = _backward_eager(kept, ctx.dim, lengths, states, dy, dh)
        return dp.to(ctx.p_dtype), dh0, None, None, None


# -------------------------------------------------------------------- entry points
def _check_projection(p, dim, axes: int, shape: str) -> None:
    if not isinstance(p, torch.Tensor) or p.dtype not in _DTYPES:
        raise ValueError(f"p must be a float32, bfloat16 or float16 tensor, got {getattr(p, 'dtype', type(p))}")
    if not isinstance(dim, int) or dim < 1:
        raise ValueError(f"dim must be a positive int, got {dim!r}")
    if p.dim() != axes or p.shape[-1] not in (2 * dim, 3 * dim):
        raise ValueError(f"p must be {shape} with 2 or 3 parts of {dim}, got shape {tuple(p.shape)}")


def _check_index(t, n: int, p, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64) or t.shape != (n,):
        raise ValueError(f"{what} must be int32 or int64 [{n}], got {getattr(t, 'dtype', type(t))} {tuple(getattr(t, 'shape', ()))}")
    if t.device != p.device:
        raise ValueError(f"{what} is on {t.device}, p on {p.device}")
    return t.contiguous()


def gated_scan(
    p: torch.Tensor,
    dim: int,
    h0: Optional[torch.Tensor] = None,
    lengths: Optional[torch.Tensor] = None,
    *,
    keep: str = "input",
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The recurrence over a batch of sequences: (y [B, T, dim], h_last [B, dim]).

    p        [B, T, 3 * dim] as x | r | z, or [B, T, 2 * dim] as x | r; float32,
             bfloat16 or float16; any strides (a last axis that is not of unit
             stride is copied first)
    h0       [B, dim] float32, the states before the first token; zeros if None
    lengths  [B] int32 or int64: tokens of each sequence; what p holds behind
             them is not looked at, y and the gradient are 0 there, and h_last is
             the state after the last token (h0 for a length of 0). Values
             outside 0..T count as the nearer end.
    keep     what the backward pass keeps of p: "input" keeps p itself, "int8"
             its 8-bit codes (checkpoint8; each part's last axis in groups of 32)
             and takes the gradient at the kept values. States are kept in 32
             bits before every 16th token either way and computed again between.

    y has the type of p, h_last is float32. Gradients: p and h0, once, in reverse
    mode; forward mode and gradients of gradients are refused.

    The same call gives the same bits each time. A sequence's last bits may depend on
    how time is split, which follows from the sizes of the call, padding included.

    A value that is not finite reaches all that depends on it, as one that is not
    finite; whether it is infinite or no number may depend on how time is split.
    """
    _check_projection(p, dim, 3, "[B, T, parts * dim]")
    B, T = p.shape[:2]
    if keep not in ("input", "int8"):
        raise ValueError(f"keep must be 'input' or 'int8', got {keep!r}")
    if h0 is not None:
        if not isinstance(h0, torch.Tensor) or h0.dtype != torch.float32 or h0.shape != (B, dim):
            raise ValueError(f"h0 must be float32 [{B}, {dim}], got {getattr(h0, 'dtype', type(h0))} {tuple(getattr(h0, 'shape', ()))}")
        if h0.device != p.device:
            raise ValueError(f"h0 is on {h0.device}, p on {p.device}")
        h0 = h0.contiguous()
    if lengths is not None:
        lengths = _check_index(lengths, B, p, "lengths")
    if B == 0 or T == 0:  # nothing to scan: differentiable as it stands
        last = p.new_zeros((B, dim), dtype=torch.float32) if h0 is None else h0.clone()
        return p[..., :dim] * 1, last
    if p.stride(2) != 1:
        p = p.contiguous()
    if p.is_cuda:
        return ext().gated_scan(p, dim, h0, lengths, keep == "int8")
    return _GatedScan.apply(p, p.new_zeros((B, dim), dtype=torch.float32) if h0 is None else h0, lengths, dim, keep == "int8")


def gated_step(
    p: torch.Tensor,
    state: torch.Tensor,
    slots: Optional[torch.Tensor] = None,
    *,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """One token of the recurrence for B streams: y [B, dim]; states are updated.

    p      [B, 3 * dim] as x | r | z, or [B, 2 * dim] as x | r
    state  [S, dim] float32, contiguous: one state for each slot
    slots  [B] int32 or int64: the slot of each row; None: row b has slot b, and
           S is B. A slot outside 0..S-1 names no state: its row is padding, y is
           0 there and nothing is written. Rows with the same slot are applied
           one after the other in their order. (Every row is looked for in
           all others: some thousand rows a call, not a hundred thousand.)
    out    where the new states go: ``state`` itself (None), or a buffer of its
           shape that does not overlap it; slots that no row names are left as
           they are there.

    It has no gradient (use :func:`gated_scan`), and refuses inputs that ask for one,
    forward mode's among them.
    """
    if not isinstance(state, torch.Tensor) or state.dtype != torch.float32 or state.dim() != 2 or not state.is_contiguous():
        raise ValueError("state must be contiguous float32 [slots, dim]")
    S, dim = state.shape
    _check_projection(p, dim, 2, "[B, parts * dim]")
    if state.device != p.device:
        raise ValueError(f"state is on {state.device}, p on {p.device}")
    if torch.is_grad_enabled() and (p.requires_grad or state.requires_grad or getattr(out, "requires_grad", False)):
        raise ValueError("gated_step has no gradient: call it under torch.no_grad()")
    B = p.shape[0]
    if slots is not None:
        slots = _check_index(slots, B, p, "slots")
    elif S != B:
        raise ValueError(f"without slots, state needs one row for each of p's {B}, got {S}")
    if out is None:
        out = state
    elif out is not state:
        if (not isinstance(out, torch.Tensor) or out.dtype != torch.float32 or out.shape != state.shape
                or out.device != state.device or not out.is_contiguous()):
            raise ValueError(f"out must be contiguous float32 [{S}, {dim}] on {state.device}")
        a, b, n = out.data_ptr(), state.data_ptr(), 4 * S * dim
        if a != b and a < b + n and b < a + n:
            raise ValueError("out overlaps state: pass state itself, or a buffer of its own")
    if B and p.is_cuda:
        return ext().gated_step(p if p.stride(1) == 1 else p.contiguous(), state, slots, out)
    for t in (p, state, out):
        if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("gated_step has no gradient, no forward mode either")
    y = torch.empty((B, dim), dtype=p.dtype, device=p.device)
    pf = p.detach().float()
    new = {}
    for b in range(B):
        s = b if slots is None else int(slots[b])
        if not 0 <= s < S:
            y[b] = 0
            continue
        h = new.get(s, state[s])
        h = _next(_gate(pf[b, dim : 2 * dim]), pf[b, :dim], h)
        new[s] = h
        y[b] = h * torch.nn.functional.silu(pf[b, 2 * dim :]) if p.shape[1] == 3 * dim else h
    for s, h in new.items():
        out[s] = h
    return y
