"""The 8-bit cache at the edges of its contract: prompts of no tokens, values that
are not finite, ids that do not fit 32 bits, softcap and scale."""

import math

import pytest
import torch

from full_attention_reference import quantise
from test_gpu_kv_cache import DT, check, rand, slots

pytestmark = pytest.mark.gpu


def test_a_fresh_prompt_of_no_tokens_empties_its_rows():
    from telescope_cache_b200 import cached_attention, cached_attention_step, init_kv_cache, write_kv_cache

    c = init_kv_cache(4, 40, 2, 64)
    write_kv_cache(c, rand(4, 7, 2, 64, seed=1), rand(4, 7, 2, 64, seed=2))
    none = torch.empty(3, 0, 2, 64, device="cuda")
    write_kv_cache(c, none, none)  # appended: nothing
    assert c.lengths.tolist() == [7, 7, 7, 7]
    write_kv_cache(c, none, none, seq_idx=torch.empty(3, 0, device="cuda", dtype=torch.int32), fresh=True)  # names no row
    assert c.lengths.tolist() == [7, 7, 7, 7] and c.max_length == 7
    write_kv_cache(c, none, none, fresh=True)
    assert c.lengths.tolist() == [0, 0, 0, 7] and c.max_length == 7
    write_kv_cache(c, torch.empty(4, 0, 2, 64, device="cuda"), torch.empty(4, 0, 2, 64, device="cuda"), fresh=True)
    assert c.lengths.tolist() == [0, 0, 0, 0] and c.max_length == 0
    q, k, v = (rand(4, 1, 2, 64, seed=i) for i in range(3))
    out, lse = cached_attention(q, c)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    out, _ = cached_attention_step(q, k, v, c)
    assert c.lengths.tolist() == [1, 1, 1, 1]
    held = quantise(v, "int8")[2]  # one token: the value as held
    assert float((out.cpu().double() - held).abs().max()) <= 2.0 ** -18 * float(held.abs().max())
