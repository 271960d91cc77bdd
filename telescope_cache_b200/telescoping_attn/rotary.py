"""Rotary positions for full-attention layers: tables with position scaling, and
one differentiable launch that rotates a token's queries and keys in either
layout, over a part of the head, at any integer positions.

``apply_rope`` (position.py) is the reference's form: half layout, whole head,
one tensor.  Here q and k go together, are read in place through their strides
(views of a fused projection), and nothing synchronises with the host.
"""

import math
from typing import Optional, Tuple

import torch

from .. import _lib

LAYOUTS = ("half", "interleaved")
SCALINGS = ("none", "linear", "base", "parts")


def rotary_tables(n_pos: int, dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                  original_positions: Optional[int] = None, turns: Tuple[float, float] = (1.0, 32.0),
                  magnitude: float = 1.0, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos / sin [n_pos, dim // 2] fp32 of theta_i = base^(-2i / dim), times
    `magnitude`.  Angles are formed in 64 bits: a fp32 angle at position 131072
    is off by up to 0.004.

    scaling, for contexts `factor` times as long as the frequencies were made for:
        'none'    theta_i
        'linear'  theta_i / factor (positions squeezed into the old range)
        'base'    base * factor^(dim / (dim - 2)): the slowest frequency is
                  divided by `factor`, the fastest stays
        'parts'   per frequency, by the turns it makes over `original_positions`:
                  theta_i with turns[1] or more, theta_i / factor with turns[0]
                  or fewer, linear in the number of turns between
    """
    if dim <= 0 or dim % 2 != 0:
        raise ValueError(f"dim must be positive and even, got {dim}")
    if n_pos <= 0:
        raise ValueError(f"n_pos must be positive, got {n_pos}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not factor > 0:
        raise ValueError(f"factor must be positive, got {factor}")
    if scaling == "none" and factor != 1.0:
        raise ValueError("factor given with scaling='none'")
    if scaling == "base":
        if dim < 4:
            raise ValueError(f"scaling='base' needs dim >= 4, got {dim}")
        base = base * factor ** (dim / (dim - 2))
    theta = float(base) ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    if scaling == "linear":
        theta = theta / factor
    elif scaling == "parts":
        if original_positions is None or original_positions <= 0:
            raise ValueError("scaling='parts' needs original_positions")
        few, many = turns
        if not many > few:
            raise ValueError(f"turns must ascend, got {turns}")
        made = original_positions * theta / (2 * math.pi)
        keep = ((made - few) / (many - few)).clamp(0.0, 1.0)
        theta = keep * theta + (1.0 - keep) * theta / factor
    ang = torch.arange(n_pos, device=device, dtype=torch.float64)[:, None] * theta[None, :]
    return (torch.cos(ang) * magnitude).float(), (torch.sin(ang) * magnitude).float()


class _Rotary(torch.autograd.Function):
    """The rotation is linear: its VJP is the rotation by the negative angle
    (with the tables' magnitude), in the same kernel."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, layout, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.cfg = (layout, inverse, q.dtype)
        return _lib.host(q).rotary(q, k, cos, sin, positions, layout, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        cos, sin, positions = ctx.saved_tensors
        layout, inverse, dtype = ctx.cfg
        # under create_graph the gradient is differentiated in its turn
        turn = _Rotary.apply if torch.is_grad_enabled() else _lib.host(gq).rotary
        dq, dk = turn(gq.to(dtype), None if gk is None else gk.to(dtype), cos, sin, positions, layout, not inverse)
        return dq, dk, None, None, None, None, None


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, *,
           positions: Optional[torch.Tensor] = None, layout: str = "half",
           inverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotated (q [B, N, Hq, D], k [B, N, Hkv, D] or None) in fp32, rounded once.

    The first R = 2 * cos.shape[1] dims of a head rotate, pairs (i, i + R / 2)
    for layout 'half' and (2i, 2i + 1) for 'interleaved'; the others pass
    through.  positions: integers [N] or [B, N], by default 0 .. N - 1; a
    position outside the tables makes the rotated dims of its rows NaN (no
    device value is read on the host).  Differentiable in q and k; inverse=True
    rotates back.  Any strides with a dense head dim are read in place."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    interleaved = layout == "interleaved"
    if torch.is_grad_enabled():
        if cos.requires_grad or sin.requires_grad:
            raise NotImplementedError("gradients with respect to the rotary tables are not supported")
        if q.requires_grad or (k is not None and k.requires_grad):
            return _Rotary.apply(q, k, cos, sin, positions, interleaved, inverse)
    return _lib.host(q).rotary(q, k, cos, sin, positions, interleaved, inverse)


__all__ = ["rotary_tables", "rotary"]
