"""Causal attention at the edges of its contract: the order of its products, what
a caller may pass for scale, softcap, ids, bounds and addresses.

Tolerances are test_gpu_causal.py's, by check_forward and check_grads."""

import pytest
import torch

from test_gpu_causal import DT, check_forward, ids_of, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap", [None, 20.0])
def test_both_directions_repeat_bit_for_bit(dtype, D, softcap):
    """A score tile that overwrote weights (or a dP tile that overwrote dX) before
    the product that reads them is through would differ from call to call."""
    from telescope_cache_b200 import causal_attention, causal_attention_backward, segment_bounds

    q, k, v = inputs(2, 1900, 8, 2, D, D, DT[dtype], seed=12)
    seg = segment_bounds(torch.stack([ids_of([1900], 1900), ids_of([700, -9, 1191], 1900)]))
    out, lse = causal_attention(q, k, v, seq_idx=seg, softcap=softcap)
    gout = torch.randn_like(out)
    want = causal_attention_backward(q, k, v, out, lse, gout, seq_idx=seg, softcap=softcap)
    for _ in range(30):
        again, again_lse = causal_attention(q, k, v, seq_idx=seg, softcap=softcap)
        assert torch.equal(again, out) and torch.equal(again_lse, lse)
        for a, b in zip(causal_attention_backward(q, k, v, out, lse, gout, seq_idx=seg, softcap=softcap), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64), ("f32", 64), ("f32", 96)])
def test_bounds_that_leave_the_row(dtype, D):
    """A window of 200 tokens whose starts and ends were not cut off at the row's
    ends gives what the cut bounds give."""
    from telescope_cache_b200 import Segments, causal_attention

    N, W = 700, 200
    q, k, v = (t.requires_grad_() for t in inputs(1, N, 4, 2, D, D, DT[dtype], seed=21))
    n = torch.arange(N, device="cuda", dtype=torch.int32)[None]
    wide, cut = Segments(n - W + 1, n + W), Segments((n - W + 1).clamp(min=0), (n + W).clamp(max=N))
    results = []
    for seg in (wide, cut):
        out, lse = causal_attention(q, k, v, seq_idx=seg)
        results.append([out, lse, *torch.autograd.grad(out.float().square().sum() + lse.sum(), (q, k, v))])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    see = (n[:, None] <= n[..., None]) & (n[:, None] > n[..., None] - W)
    check_forward(results[0][0].detach(), results[0][1].detach(), q.detach(), k.detach(), v.detach(), see)


def test_starts_and_ends_go_together():
    from telescope_cache_b200 import Segments, causal_attention

    q, k, v = inputs(1, 20, 2, 1, 64, 64, torch.bfloat16)
    n = torch.zeros(1, 20, device="cuda", dtype=torch.int32)
    for seg in (Segments(n, None), Segments(None, n)):
        with pytest.raises(ValueError, match="go together"):
            causal_attention(q, k, v, seq_idx=seg)
