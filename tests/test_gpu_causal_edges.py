"""Causal attention at the edges of its contract: the order of its products, what
a caller may pass for scale, softcap, ids, bounds and addresses.

Tolerances are test_gpu_causal.py's, by check_forward and check_grads."""

import pytest
import torch

from test_gpu_causal import DT, ids_of, inputs

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
