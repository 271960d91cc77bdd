"""Causal attention over whole prompts and packed training rows, with grouped
heads: the full-attention counterpart of ``multilevel_attention_forward`` for
the layers that a hybrid stack does not telescope.

It has the same (out, lse) boundary, so ``apply_attention_sink`` and
``apply_output_gate`` follow it unchanged, and the same ``seq_idx`` as
``short_conv``: ids of the packed examples of a row.
"""

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from .. import _lib
from .attention import _impl_code, device_status


class Segments(NamedTuple):
    """Bounds of the packed examples (segment_bounds): token n of row b sees
    tokens starts[b, n] .. n and is seen by tokens n .. ends[b, n] - 1."""

    starts: torch.Tensor
    ends: torch.Tensor

    def positions(self) -> torch.Tensor:
        """[B, N] int32 position of each token in its example (0 in padding)."""
        n = torch.arange(self.starts.shape[1], device=self.starts.device, dtype=torch.int32)
        return (n - self.starts).clamp_(min=0)


def segment_bounds(seq_idx: torch.Tensor) -> Segments:
    """Bounds of the runs of equal ids of seq_idx [B, N] (integers).  A packed
    example is one run; tokens with a negative id are padding: they see nothing
    and are seen by nothing."""
    if seq_idx.dim() != 2 or seq_idx.dtype.is_floating_point:
        raise ValueError(f"seq_idx must be an integer tensor [B, N], got {tuple(seq_idx.shape)} {seq_idx.dtype}")
    _lib.require_cuda(seq_idx)
    ids = seq_idx if seq_idx.dtype == torch.int32 and seq_idx.is_contiguous() else seq_idx.to(torch.int32).contiguous()
    B, N = ids.shape
    both = torch.empty(2, B, N, device=ids.device, dtype=torch.int32)
    starts, ends = both[0], both[1]
    _lib.launch("tc_segment_bounds", ids.device, B, N, ids.data_ptr(), starts.data_ptr(), ends.data_ptr(),
                _lib.stream_of(ids))
    return Segments(starts, ends)


def _segments(seq_idx, B, N):
    if seq_idx is None:
        return None
    if isinstance(seq_idx, Segments):
        if tuple(seq_idx.starts.shape) != (B, N) or tuple(seq_idx.ends.shape) != (B, N):
            raise ValueError(f"segment bounds {tuple(seq_idx.starts.shape)} != {(B, N)}")
        return seq_idx
    if tuple(seq_idx.shape) != (B, N):
        raise ValueError(f"seq_idx must be an integer tensor [{B}, {N}], got {tuple(seq_idx.shape)}")
    return segment_bounds(seq_idx)


def _check(q, k, v, softcap, scale):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k, v must be [B, N, H, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, N, Hq, Dk = q.shape
    Hkv = k.shape[2]
    if tuple(k.shape) != (B, N, Hkv, Dk):
        raise ValueError(f"k shape {tuple(k.shape)} incompatible with q {tuple(q.shape)}")
    if tuple(v.shape[:3]) != (B, N, Hkv):
        raise ValueError(f"v shape {tuple(v.shape)} incompatible with k {tuple(k.shape)}")
    if Hkv == 0 or Hq % Hkv != 0:
        raise ValueError(f"Hq={Hq} must be divisible by Hkv={Hkv}.")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"q, k, v must share a dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    if softcap is not None and not softcap > 0:
        raise ValueError(f"softcap must be positive, got {softcap}")
    _lib.require_cuda(q, k, v)
    return 1.0 / math.sqrt(Dk) if scale is None else float(scale)


def _dense_head(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _args(q, k, v, seg, softcap, scale, impl):
    B, N, Hq, Dk = q.shape
    return _lib.CausalArgs(
        B=B, N=N, Hq=Hq, Hkv=k.shape[2], Dk=Dk, Dv=v.shape[3], dtype=_lib.dtype_code(q.dtype),
        has_softcap=softcap is not None, softcap=0.0 if softcap is None else softcap, scale=scale,
        q=q.data_ptr(), q_stride_b=q.stride(0), q_stride_n=q.stride(1), q_stride_h=q.stride(2),
        k=k.data_ptr(), k_stride_b=k.stride(0), k_stride_n=k.stride(1), k_stride_h=k.stride(2),
        v=v.data_ptr(), v_stride_b=v.stride(0), v_stride_n=v.stride(1), v_stride_h=v.stride(2),
        starts=None if seg is None else seg.starts.data_ptr(), ends=None if seg is None else seg.ends.data_ptr(),
        dev_status=device_status(q.device).data_ptr(), impl=_impl_code(impl))


def _forward(q, k, v, seg, softcap, scale, impl):
    q, k, v = _dense_head(q), _dense_head(k), _dense_head(v)
    B, N, Hq, _ = q.shape
    out = torch.empty(B, N, Hq, v.shape[3], device=q.device, dtype=q.dtype)
    lse = torch.empty(B, N, Hq, device=q.device, dtype=torch.float32)
    a = _args(q, k, v, seg, softcap, scale, impl)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    _lib.launch("tc_causal_fwd", q.device, a, _lib.stream_of(q))
    return out, lse


def _backward(q, k, v, out, lse, dout, dlse, seg, softcap, scale, impl):
    q, k, v = _dense_head(q), _dense_head(k), _dense_head(v)
    B, N, Hq, Dk = q.shape
    out, dout, lse = out.contiguous(), dout.contiguous(), lse.contiguous()
    dlse = None if dlse is None else dlse.float().contiguous()
    delta = torch.empty(B, N, Hq, device=q.device, dtype=torch.float32)
    dq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    dk = torch.empty(k.shape, device=q.device, dtype=q.dtype)
    dv = torch.empty(v.shape, device=q.device, dtype=q.dtype)
    a = _args(q, k, v, seg, softcap, scale, impl)
    a.lse, a.o, a.dout = lse.data_ptr(), out.data_ptr(), dout.data_ptr()
    a.dlse = None if dlse is None else dlse.data_ptr()
    a.delta, a.dq, a.dk, a.dv = delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    _lib.launch("tc_causal_bwd", q.device, a, _lib.stream_of(q))
    return dq, dk, dv


class _Causal(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts, ends, softcap, scale, impl):
        seg = None if starts is None else Segments(starts, ends)
        out, lse = _forward(q, k, v, seg, softcap, scale, impl)
        ctx.save_for_backward(q, k, v, out, lse, starts, ends)
        ctx.cfg = (softcap, scale, impl)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    def backward(ctx, dout, dlse):
        q, k, v, out, lse, starts, ends = ctx.saved_tensors
        seg = None if starts is None else Segments(starts, ends)
        if dout is None and dlse is None:
            return (None,) * 8
        dout = torch.zeros_like(out) if dout is None else dout.to(out.dtype)
        return _backward(q, k, v, out, lse, dout, dlse, seg, *ctx.cfg) + (None,) * 5


def causal_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                     seq_idx: Union[torch.Tensor, Segments, None] = None, softcap: Optional[float] = None,
                     scale: Optional[float] = None, impl: Optional[str] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [B, N, Hq, Dv], lse [B, N, Hq] fp32 natural log) of causal attention
    of q [B, N, Hq, Dk] over k [B, N, Hkv, Dk], v [B, N, Hkv, Dv]; query head h
    reads key head h // (Hq / Hkv).

    S = c tanh(X / c) (X without softcap), X = scale q.k, scale 1 / sqrt(Dk) by
    default.  seq_idx [B, N]: ids of the row's packed examples, one run each: a
    token attends its own example only; a token with a negative id is padding
    (out 0, lse -inf, zero gradients).  The bounds of segment_bounds may be
    given in its place, so that the layers of a model form them once.

    Differentiable in q, k, v through both results.  bf16 / f16 with Dk = Dv of
    64 or 128 run on the tensor cores (strided q, k, v in place where strides
    and addresses are multiples of 16 bytes), other types and head dims up to
    256 on the CUDA cores.  Products with tokens outside a row's view are formed
    and masked: a NaN or infinity in one example's values reaches the rows of
    its neighbours in the same 128 tokens.  ``impl`` ('simt' | 'tensor' | None)
    pins a kernel family for testing."""
    scale = _check(q, k, v, softcap, scale)
    seg = _segments(seq_idx, q.shape[0], q.shape[1])
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Causal.apply(q, k, v, None if seg is None else seg.starts, None if seg is None else seg.ends, softcap,
                             scale, impl)
    return _forward(q, k, v, seg, softcap, scale, impl)


@torch.no_grad()
def causal_attention_backward(q, k, v, out, lse, dout, *, dlse: Optional[torch.Tensor] = None,
                              seq_idx: Union[torch.Tensor, Segments, None] = None, softcap: Optional[float] = None,
                              scale: Optional[float] = None, impl: Optional[str] = None):
    """(dq, dk, dv) at the (out, lse) boundary of causal_attention, with the
    gradient of lse folded into Delta (the seam that attention_sink_backward
    feeds).  Bit-for-bit repeatable."""
    scale = _check(q, k, v, softcap, scale)
    B, N, Hq, _ = q.shape
    if tuple(out.shape) != (B, N, Hq, v.shape[3]) or out.dtype != q.dtype:
        raise ValueError(f"out shape {tuple(out.shape)} {out.dtype} != {(B, N, Hq, v.shape[3])} {q.dtype}")
    if tuple(dout.shape) != tuple(out.shape) or dout.dtype != out.dtype:
        raise ValueError(f"dout shape {tuple(dout.shape)} {dout.dtype} must match out {tuple(out.shape)} {out.dtype}")
    if tuple(lse.shape) != (B, N, Hq) or lse.dtype != torch.float32:
        raise ValueError("lse must be float32 [B, N, Hq]")
    if dlse is not None and (tuple(dlse.shape) != (B, N, Hq) or not dlse.dtype.is_floating_point):
        raise ValueError(f"dlse must be floating [{B}, {N}, {Hq}], got {tuple(dlse.shape)} {dlse.dtype}")
    _lib.require_cuda(out, lse, dout, dlse)
    return _backward(q, k, v, out, lse, dout, dlse, _segments(seq_idx, B, N), softcap, scale, impl)


__all__ = ["Segments", "segment_bounds", "causal_attention", "causal_attention_backward"]
