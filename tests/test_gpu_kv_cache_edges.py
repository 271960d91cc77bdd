"""The 8-bit cache at the edges of its contract: prompts of no tokens, values that
are not finite, ids that do not fit 32 bits, softcap and scale."""

import math

import pytest
import torch

from full_attention_reference import UNIT, quantise
from test_gpu_kv_cache import DT, formula, rand

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


@pytest.mark.parametrize("dtype,D", [("bf16", 80), ("f32", 80), ("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("N", [1, 30, 3000])
def test_a_query_that_is_not_a_number(dtype, D, N):
    """NaN logits make their own head's result NaN, not an empty row's, whatever
    the number of splits; nothing else changes."""
    from telescope_cache_b200 import cached_attention, init_kv_cache, write_kv_cache

    dt = DT[dtype]
    c = init_kv_cache(2, 3001, 2, D, dtype=dt)
    write_kv_cache(c, rand(2, N, 2, D, dtype=dt, seed=1), rand(2, N, 2, D, dtype=dt, seed=2))
    q = rand(2, 1, 6, D, dtype=dt, seed=3)
    want, want_lse = cached_attention(q, c)
    q[0, 0, 4, 7] = math.nan
    out, lse = cached_attention(q, c)
    bad = torch.zeros(2, 1, 6, dtype=torch.bool, device="cuda")
    bad[0, 0, 4] = True
    assert bool(out[bad].isnan().all()) and bool(lse[bad].isnan().all())
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse[~bad], want_lse[~bad])


@pytest.mark.parametrize("D", [80, 128])
@pytest.mark.parametrize("N", [20, 2000])
def test_a_step_past_the_tables_is_nan(D, N):
    """Lengths that moved on without the host's bound: the rotated query is NaN, and so
    is the result; the other row's is not."""
    from telescope_cache_b200 import cached_attention_step, init_kv_cache, write_kv_cache

    c = init_kv_cache(2, N + 10, 2, D)
    ids = torch.where(torch.arange(N) < torch.tensor([N, 5])[:, None], torch.arange(2)[:, None], -1)
    write_kv_cache(c, rand(2, N, 2, D, seed=1), rand(2, N, 2, D, seed=2), seq_idx=ids.cuda())
    c.max_length = 5
    ang = torch.rand(8, 12, device="cuda")
    q, k, v = (rand(2, 1, h, D, seed=h) for h in (4, 2, 2))
    out, lse = cached_attention_step(q, k, v, c, rope_cos=ang.cos(), rope_sin=ang.sin())
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    assert bool(out[1].isfinite().all()) and bool(lse[1].isfinite().all())
    assert c.lengths.tolist() == [N + 1, 6]


@pytest.mark.parametrize("store", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 40])
def test_an_infinity_makes_its_row_nan(store, dtype, D):
    """Every element of the row, of either sign, written as a prompt or as a step."""
    from telescope_cache_b200 import cached_attention_step, init_kv_cache, read_kv_cache, write_kv_cache

    dt = DT[dtype]
    c = init_kv_cache(2, 8, 2, D, store=store, dtype=dt)
    k, v = rand(2, 4, 2, D, dtype=dt, seed=1), rand(2, 4, 2, D, dtype=dt, seed=2)
    k[0, 1, 0, 3], v[0, 2, 1, 9] = math.inf, -math.inf
    write_kv_cache(c, k, v)
    q, kt, vt = (rand(2, 1, 2, D, dtype=dt, seed=i) for i in (3, 4, 5))
    kt[1, 0, 1, 0], vt[1, 0, 0, 5] = -math.inf, math.inf
    _, _, kn, vn = cached_attention_step(q, kt, vt, c, return_stored=True)
    rk, rv = read_kv_cache(c)
    bk, bv = (torch.zeros(2, 5, 2, dtype=torch.bool, device="cuda") for _ in range(2))
    bk[0, 1, 0] = bv[0, 2, 1] = bk[1, 4, 1] = bv[1, 4, 0] = True
    for r, bad, last in ((rk, bk, kn), (rv, bv, vn)):
        assert bool(r[bad].isnan().all()) and bool(r[~bad].isfinite().all())
        assert torch.equal(last[:, 0].isnan(), r[:, 4].isnan())


@pytest.mark.parametrize("store", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,D,Hq", [("f32", 128, 5), ("f32", 64, 8), ("bf16", 128, 2), ("f32", 80, 3)])
@pytest.mark.parametrize("power", [12, 24, 36, 90])
def test_values_of_very_different_sizes(store, dtype, D, Hq, power):
    """A token with values 2^power times the others' that hardly any head weighs:
    the others' weights keep their bits.  (One head's logits fall towards it, so
    that its weight counts there.)"""
    from telescope_cache_b200 import cached_attention, init_kv_cache, write_kv_cache

    dt, N = DT[dtype], 900
    k, v = rand(1, N, 1, D, dtype=dt, seed=1), rand(1, N, 1, D, dtype=dt, seed=2)
    q = rand(1, 1, Hq, D, dtype=dt, seed=3)
    q[..., 0] = 8.0
    q[:, :, Hq - 1, 0] = -8.0 * power / 90
    k[:, :, :, 0] = 0
    for at in (1, 400, 899):
        k[:, at, :, 0] = -15.0 * D ** 0.5
        v[:, at] *= 2.0 ** power
    c = init_kv_cache(1, N, 1, D, store=store, dtype=dt)
    write_kv_cache(c, k, v)
    out, lse = cached_attention(q, c)
    held = [quantise(t, store)[2][0] for t in (k, v)]
    o, l, size, top = formula(q[0, 0].double().cpu(), *held, None, D ** -0.5)
    # as check(), and the fp32 error of logits of size top in the weights
    err = (out[0, 0].double().cpu() - o).abs()
    assert bool((err <= UNIT[dt] * o.abs() + (2.0 ** -18 + 4 * top * 2.0 ** -23) * size).all()), float((err / size).max())
    assert float((lse[0, 0].double().cpu() - l).abs().max()) <= 1e-5 + 4e-6 * top
