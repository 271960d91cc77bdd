"""Causal attention over whole prompts and packed training rows, with grouped
heads: the full-attention counterpart of ``multilevel_attention_forward`` for
the layers that a hybrid stack does not telescope.

It has the same (out, lse) boundary, so ``apply_attention_sink`` and
``apply_output_gate`` follow it unchanged, and the same ``seq_idx`` as
``short_conv``: ids of the packed examples of a row.
"""

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .attention import _impl_code


class Segments(NamedTuple):
    """Bounds of the packed examples (segment_bounds): token n of row b sees
    tokens starts[b, n] .. n and is seen by tokens n .. ends[b, n] - 1.  Neither
    descends along a row; what lies outside the row is cut off at its ends."""

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
    return Segments(*_lib.host(seq_idx).segment_bounds(seq_idx))


def _split(seq_idx):
    """(ids, starts, ends) of a seq_idx that is ids, bounds or None."""
    if isinstance(seq_idx, Segments):
        return None, seq_idx.starts, seq_idx.ends
    return seq_idx, None, None


class _Causal(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts, ends, softcap, scale, impl):
        out, lse, low = _lib.host(q).causal_forward(q, k, v, None, starts, ends, softcap, scale, impl, True)
        ctx.save_for_backward(q, k, v, out, low, lse, starts, ends)
        ctx.cfg = (softcap, scale, impl)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlse):
        q, k, v, out, low, lse, starts, ends = ctx.saved_tensors
        if dout is None and dlse is None:
            return (None,) * 8
        dout = torch.zeros_like(out) if dout is None else dout.to(out.dtype)
        return _lib.host(q).causal_backward(q, k, v, out, low, lse, dout, dlse, None, starts, ends, *ctx.cfg) + (None,) * 5


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

    Differentiable in q, k, v through both results, once and in reverse mode (for
    16-bit types the graph also keeps what the rounding of out left over, a tensor
    of its size).

    bf16 / f16 with Dk = Dv of 64 or 128 run on the tensor cores: strided q, k, v in
    place where strides and addresses are multiples of 16 bytes and no stride is
    zero, with a scale of 1e-30 to 1e30 and a softcap of at most 2048.  Everything
    else, head dims up to 256, runs on the CUDA cores, up to 30 times slower: copy
    16-bit views that do not qualify.  The tensor cores take weights and gradients of
    logits in the type of q: in f16 the latter, up to twice |dout| |v| of a token,
    have to stay below 65504 and well above 6e-8 (a loss scale that fits the other
    f16 gradients does).  Products with tokens outside a row's view are formed and
    masked: a NaN or infinity in one example's values reaches the rows of its
    neighbours in the same 128 tokens.  ``impl`` ('simt' | 'tensor' | None) pins a
    kernel family for testing."""
    code = _impl_code(impl)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if seq_idx is not None and not isinstance(seq_idx, Segments):
            seq_idx = segment_bounds(seq_idx)  # once for both directions
        _, starts, ends = _split(seq_idx)
        return _Causal.apply(q, k, v, starts, ends, softcap, scale, code)
    return _lib.host(q).causal_forward(q, k, v, *_split(seq_idx), softcap, scale, code, False)[:2]


@torch.no_grad()
def causal_attention_backward(q, k, v, out, lse, dout, *, dlse: Optional[torch.Tensor] = None,
                              seq_idx: Union[torch.Tensor, Segments, None] = None, softcap: Optional[float] = None,
                              scale: Optional[float] = None, impl: Optional[str] = None):
    """(dq, dk, dv) at the (out, lse) boundary of causal_attention, with the
    gradient of lse folded into Delta (the seam that attention_sink_backward
    feeds); Delta is taken from the rounded out, where autograd has its leftovers
    too (bf16, values of mean 8: dq off by 1.5e-2 of its norm for autograd's 2.4e-3).
    Bit-for-bit repeatable."""
    return _lib.host(q).causal_backward(q, k, v, out, None, lse, dout, dlse, *_split(seq_idx), softcap, scale,
                                        _impl_code(impl))


__all__ = ["Segments", "segment_bounds", "causal_attention", "causal_attention_backward"]
