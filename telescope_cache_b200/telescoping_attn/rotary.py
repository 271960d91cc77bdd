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


def _table(t):
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _dense_head(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _launch(q, k, cos, sin, positions, layout, inverse):
    B, N, Hq, D = q.shape
    q = _dense_head(q)
    a = _lib.RotaryArgs(B=B, N=N, Hq=Hq, Hk=0, D=D, R=2 * cos.shape[1], dtype=_lib.dtype_code(q.dtype),
                        interleaved=layout == "interleaved", inverse=bool(inverse), n_pos=cos.shape[0],
                        cos_t=cos.data_ptr(), sin_t=sin.data_ptr())
    qo = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    a.q, a.q_out = q.data_ptr(), qo.data_ptr()
    a.q_stride_b, a.q_stride_n, a.q_stride_h = q.stride(0), q.stride(1), q.stride(2)
    ko = None
    if k is not None:
        k = _dense_head(k)
        ko = torch.empty(k.shape, device=k.device, dtype=k.dtype)
        a.Hk, a.k, a.k_out = k.shape[2], k.data_ptr(), ko.data_ptr()
        a.k_stride_b, a.k_stride_n, a.k_stride_h = k.stride(0), k.stride(1), k.stride(2)
    if positions is not None:
        a.positions, a.pos_stride_b = positions.data_ptr(), positions.stride(0) if positions.dim() == 2 else 0
    _lib.launch("tc_rotary", q.device, a, _lib.stream_of(q))
    return qo, ko


class _Rotary(torch.autograd.Function):
    """The rotation is linear: its VJP is the rotation by the negative angle
    (with the tables' magnitude), in the same kernel."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, layout, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.cfg = (layout, inverse, q.dtype)
        qo, ko = _launch(q, k, cos, sin, positions, layout, inverse)
        return qo, ko

    @staticmethod
    def backward(ctx, gq, gk):
        cos, sin, positions = ctx.saved_tensors
        layout, inverse, dtype = ctx.cfg
        if gk is None:
            dq, dk = _launch(gq.to(dtype), None, cos, sin, positions, layout, not inverse)
        else:
            dq, dk = _launch(gq.to(dtype), gk.to(dtype), cos, sin, positions, layout, not inverse)
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
    if q.dim() != 4:
        raise ValueError(f"q must be [B, N, H, D], got {tuple(q.shape)}")
    B, N, _, D = q.shape
    if k is not None and (k.dim() != 4 or tuple(k.shape[:2]) != (B, N) or k.shape[3] != D):
        raise ValueError(f"k shape {tuple(k.shape)} incompatible with q {tuple(q.shape)}")
    if k is not None and k.dtype != q.dtype:
        raise ValueError(f"k dtype {k.dtype} must match q dtype {q.dtype}")
    if cos.shape != sin.shape or cos.dim() != 2:
        raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must be one [n_pos, R / 2] shape")
    if 2 * cos.shape[1] > D:
        raise ValueError(f"rotary tables cover dim {2 * cos.shape[1]}, the heads have {D}")
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if positions is None:
        if cos.shape[0] < N:
            raise ValueError(f"rotary tables cover {cos.shape[0]} positions, q has {N}")
    else:
        if positions.dtype.is_floating_point or tuple(positions.shape) not in ((N,), (B, N)):
            raise ValueError(f"positions must be integers [{N}] or [{B}, {N}], got {tuple(positions.shape)} "
                             f"{positions.dtype}")
        if positions.dtype != torch.int32 or positions.stride(-1) != 1:
            positions = positions.to(torch.int32).contiguous()
    _lib.require_cuda(q, k, cos, sin, positions)
    if torch.is_grad_enabled():
        if cos.requires_grad or sin.requires_grad:
            raise NotImplementedError("gradients with respect to the rotary tables are not supported")
        if q.requires_grad or (k is not None and k.requires_grad):
            return _Rotary.apply(q, k, _table(cos), _table(sin), positions, layout, bool(inverse))
    return _launch(q, k, _table(cos), _table(sin), positions, layout, inverse)


__all__ = ["rotary_tables", "rotary"]
