"""The 8-bit cache: codes bit for bit, ragged and packed writes, the attention
over the codes against the formula in 64 bits on the values they stand for.

Tolerances: q and P enter the products with 22 bits, sums are fp32: out is
within UNIT |out| + 2^-18 sum p |v| of exact, lse within 1e-5 + 4e-6 max |logit|
(softcap by 1 - 2 / (e^2x + 1): 1e-6 of the cap)."""

import math

import pytest
import torch

from full_attention_reference import LEAST, UNIT, quantise, rotate

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def rand(*s, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*s, generator=g, device="cuda").to(dtype)


def slots(cache, row, n):
    """(k codes, v codes, k scales, v scales) of the first n slots of a row, [n, Hkv, ...]."""
    return [t[row, :, :n].transpose(0, 1).cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


@pytest.mark.parametrize("store", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("H,Dk,Dv", [(2, 128, 128), (3, 64, 64), (1, 96, 96), (2, 40, 72), (2, 256, 256)])
def test_written_codes_and_values(store, dtype, H, Dk, Dv):
    from telescope_cache_b200 import init_kv_cache, read_kv_cache, write_kv_cache

    B, N, dt = 2, 21, DT[dtype]
    c = init_kv_cache(B, 50, H, Dk, Dv, store=store, dtype=dt)
    parts = [(rand(B, n, H, Dk, dtype=dt, seed=n), rand(B, n, H, Dv, dtype=dt, seed=n + 1)) for n in (N, 1, 5)]
    for i, (k, v) in enumerate(parts):
        k[0, 0, 0] = 0  # a row of zeros
        k[1, 0, H - 1] *= 2.0 ** -10
        write_kv_cache(c, k, v)
    k, v = (torch.cat([p[i] for p in parts], 1) for i in range(2))
    n = k.shape[1]
    assert c.lengths.tolist() == [n, n] and c.max_length == n
    kc, ks, kv = quantise(k, store)
    vc, vs, vv = quantise(v, store)
    for b in range(B):
        got = slots(c, b, n)
        for a, w in zip(got, (kc[b], vc[b], ks[b], vs[b])):
            assert torch.equal(a, w)
    rk, rv = read_kv_cache(c, 30)
    for r, w in ((rk, kv), (rv, vv)):
        assert r.dtype == dt and r.shape[1] == 30
        want = (w.float() if dt == torch.float32 else w).to(dt)  # one fp32 product, one rounding
        assert float((r[:, :n].cpu().double() - want.double()).abs().max()) <= UNIT[dt] * float(w.abs().max())
        assert bool((r[:, n:] == 0).all())


def test_extremes_of_a_row():
    """Infinity and NaN make a row's values NaN and nothing else's; tiny rows are zeros."""
    from telescope_cache_b200 import init_kv_cache, read_kv_cache, write_kv_cache

    for store in ("int8", "fp8"):
        c = init_kv_cache(1, 8, 2, 64, store=store, dtype=torch.float32)
        k = rand(1, 5, 2, 64)
        k[0, 1, 0, 3], k[0, 2, 1, 9], k[0, 3, 0] = math.inf, math.nan, 1e-31
        write_kv_cache(c, k, k)
        rk, _ = read_kv_cache(c)
        bad = torch.zeros(1, 5, 2, dtype=torch.bool, device="cuda")
        bad[0, 1, 0] = bad[0, 2, 1] = True
        assert bool(rk[bad].isnan().any(-1).all()) and bool(rk[~bad].isfinite().all())
        assert bool((rk[0, 3, 0] == 0).all())
        big = torch.full((1, 1, 2, 64), float(torch.finfo(torch.float32).max), device="cuda")
        write_kv_cache(c, big, big, fresh=True)
        assert float((read_kv_cache(c, 1)[0] / big - 1).abs().max()) <= 2.0 ** -22


@pytest.mark.parametrize("N", [1, 6, 130])
def test_packed_and_ragged_writes(N):
    """seq_idx names the cache row of each token: padding, rows out of order, rows
    that get nothing, appended behind what the rows hold."""
    from telescope_cache_b200 import init_kv_cache, write_kv_cache

    c = init_kv_cache(5, 300, 2, 64)
    first_k, first_v = rand(5, 3, 2, 64, seed=1), rand(5, 3, 2, 64, seed=2)
    write_kv_cache(c, first_k, first_v)
    k, v = rand(2, N, 2, 64, seed=3), rand(2, N, 2, 64, seed=4)
    ids = torch.full((2, N), -1, dtype=torch.int32)
    ids[0, : (N + 1) // 2] = 3
    ids[0, (N + 1) // 2:] = 0
    ids[1, N // 3: N - N // 4] = 2
    write_kv_cache(c, k, v, seq_idx=ids.cuda())
    for row in range(5):
        m = (ids == row)
        want_k = torch.cat([first_k[row].cpu(), k.cpu()[m]])
        assert int(c.lengths[row]) == want_k.shape[0]
        kc, ks, _ = quantise(want_k, "int8")
        got = slots(c, row, want_k.shape[0])
        assert torch.equal(got[0], kc) and torch.equal(got[2], ks)
    write_kv_cache(c, k, v, seq_idx=ids.cuda(), fresh=True)
    for row in range(5):
        n = int((ids == row).sum())
        assert int(c.lengths[row]) == (n or 3)


def test_a_token_without_a_slot_is_dropped_and_flagged():
    from telescope_cache_b200 import init_kv_cache, write_kv_cache
    from telescope_cache_b200.telescoping_attn.attention import read_device_status

    read_device_status("cuda:0")
    c = init_kv_cache(2, 4, 1, 64)
    k = rand(1, 6, 1, 64)
    ids = torch.tensor([[0, 0, 0, 0, 0, 7]], device="cuda")
    write_kv_cache(c, k, k, seq_idx=ids, max_tokens=4)  # row 0 gets five tokens, row 7 does not exist
    assert read_device_status("cuda:0") & 2
    assert c.lengths.tolist() == [4, 0]
    assert torch.equal(slots(c, 0, 4)[0], quantise(k[0, :4], "int8")[0])
    assert read_device_status("cuda:0") == 0


def formula(q, k, v, softcap, scale):
    """q [Hq, Dk], k [n, Hkv, Dk], v [n, Hkv, Dv] double -> out, lse, sum p |v|, top."""
    E = q.shape[0] // k.shape[1]
    k, v = k.repeat_interleave(E, 1), v.repeat_interleave(E, 1)
    x = torch.einsum("hd,nhd->hn", q, k) * scale
    if softcap is not None:
        x = softcap * torch.tanh(x / softcap)
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - lse[:, None])
    return torch.einsum("hn,nhd->hd", p, v), lse, torch.einsum("hn,nhd->hd", p, v.abs()), float(x.abs().max())


def check(out, lse, q, values, lengths, dt, softcap=None, scale=None):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    for b, n in enumerate(lengths):
        if n == 0:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        o, l, size, top = formula(q[b].double().cpu(), values[0][b][:n], values[1][b][:n], softcap, scale)
        err = (out[b, 0].double().cpu() - o).abs()
        assert bool((err <= UNIT[dt] * o.abs() + LEAST[dt] + 2.0 ** -18 * size).all()), float((err / size).max())
        cap = 0.0 if softcap is None else 1e-6 * softcap
        assert float((lse[b, 0].double().cpu() - l).abs().max()) <= 1e-5 + 4e-6 * top + cap


@pytest.mark.parametrize("store", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("Hq,Hkv,Dk,Dv", [(1, 1, 128, 128), (8, 2, 64, 64), (16, 2, 128, 128), (9, 1, 128, 128),
                                          (24, 2, 64, 64), (4, 2, 96, 96), (3, 3, 40, 72)])
def test_attention_over_lengths(store, dtype, Hq, Hkv, Dk, Dv):
    """Rows of length zero, one, inside and at the end of tiles and chunks."""
    from telescope_cache_b200 import cached_attention, init_kv_cache, write_kv_cache

    dt = DT[dtype]
    lengths = [0, 1, 15, 16, 17, 64, 65, 333, 700]
    B, N = len(lengths), 700
    k, v = rand(B, N, Hkv, Dk, dtype=dt, seed=1), rand(B, N, Hkv, Dv, dtype=dt, seed=2)
    v[:, ::7] *= 2.0 ** -8  # value rows of very different sizes
    ids = torch.where(torch.arange(N) < torch.tensor(lengths)[:, None], torch.arange(B)[:, None], -1)
    c = init_kv_cache(B, N + 3, Hkv, Dk, Dv, store=store, dtype=dt)
    c.k.fill_(0x7f)  # what lies past a row's end does not matter (e4m3 NaN)
    c.v.fill_(0x7f)
    c.k_scale.fill_(math.nan)
    c.v_scale.fill_(math.inf)
    write_kv_cache(c, k, v, seq_idx=ids.cuda())
    q = rand(B, 1, Hq, Dk, dtype=dt, seed=3)
    values = [quantise(t, store)[2] for t in (k, v)]
    for cap, scale in ((None, None), (20.0, 0.3)):
        out, lse = cached_attention(q, c, softcap=cap, scale=scale)
        assert out.dtype == dt and out.shape == (B, 1, Hq, Dv) and lse.shape == (B, 1, Hq)
        check(out, lse, q[:, 0], values, lengths, dt, cap, scale)
    again = cached_attention(q, c, softcap=20.0, scale=0.3)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)  # bit for bit


@pytest.mark.parametrize("store", ["int8", "fp8"])
@pytest.mark.parametrize("layout,R", [("half", 64), ("interleaved", 64), ("half", 24), ("interleaved", 0)])
@pytest.mark.parametrize("dtype,Hq,Hkv,D", [("bf16", 8, 2, 64), ("f32", 2, 2, 128), ("f16", 18, 2, 128), ("bf16", 2, 1, 80)])
def test_step(store, layout, R, dtype, Hq, Hkv, D):
    """Steps from empty rows on: codes of the rotated key, attention over them,
    lengths; a tried token leaves no trace."""
    from telescope_cache_b200 import cached_attention, cached_attention_step, init_kv_cache, rotary, write_kv_cache

    dt, B, cap = DT[dtype], 3, 80
    g = torch.Generator(device="cuda").manual_seed(5)
    ang = torch.rand(cap, R // 2, generator=g, device="cuda") * 6.28
    cos, sin = ang.cos(), ang.sin()
    c = init_kv_cache(B, cap, Hkv, D, store=store, dtype=dt)
    start = [0, 1, 63]
    k0, v0 = rand(B, 63, Hkv, D, dtype=dt, seed=1), rand(B, 63, Hkv, D, dtype=dt, seed=2)
    ids = torch.where(torch.arange(63) < torch.tensor(start)[:, None], torch.arange(B)[:, None], -1)
    write_kv_cache(c, k0, v0, seq_idx=ids.cuda())
    hist = [[quantise(t, store)[2][b, :n] for b, n in enumerate(start)] for t in (k0, v0)]
    rope = dict(rope_cos=cos, rope_sin=sin, layout=layout) if R else {}
    for s in range(4):
        q, k, v = (rand(B, 1, h, D, dtype=dt, seed=10 * s + i) for i, h in enumerate((Hq, Hkv, Hkv)))
        at = c.lengths.clone()
        tried = cached_attention_step(q, v, k, c, advance=False, **rope)  # another token, not kept
        assert torch.equal(c.lengths, at) and tried[0].shape == q.shape
        out, lse, kn, vn = cached_attention_step(q, k, v, c, softcap=25.0, return_stored=True, **rope)
        assert torch.equal(c.lengths, at + 1)
        # the rotated key in fp32, as rotary gives it
        pos = at[:, None]
        kr = rotary(k.float(), None, cos, sin, positions=pos, layout=layout)[0] if R else k.float()
        qd = rotate(q.cpu(), cos.cpu(), sin.cpu(), pos.long().cpu(), layout) if R else q.double().cpu()
        kc, _, kval = quantise(kr, store)
        vc, _, vval = quantise(v, store)
        for b in range(B):
            n = start[b] + s
            assert torch.equal(c.k[b, :, n].cpu(), kc[b, 0]) and torch.equal(c.v[b, :, n].cpu(), vc[b, 0])
            hist[0][b] = torch.cat([hist[0][b], kval[b]])
            hist[1][b] = torch.cat([hist[1][b], vval[b]])
        for a, w in ((kn, kval), (vn, vval)):
            assert a.dtype == dt and float((a.cpu().double() - w).abs().max()) <= UNIT[dt] * float(w.abs().max())
        check(out, lse, qd[:, 0], hist, [n + s + 1 for n in start], dt, 25.0)
        if not R:
            same, _ = cached_attention(q, c, softcap=25.0)
            assert torch.equal(same, out)
    assert c.max_length == 67


def test_lengths_move_on_across_chunk_ends():
    """A row that grows over a chunk's end, with fewer tokens in the others (their
    spare chunks must not see the moved length)."""
    from telescope_cache_b200 import cached_attention_step, init_kv_cache, read_kv_cache, write_kv_cache

    B, H, D = 4, 2, 128
    c = init_kv_cache(B, 600, H, D)
    ids = torch.where(torch.arange(500) < torch.tensor([62, 126, 500, 0])[:, None], torch.arange(B)[:, None], -1)
    write_kv_cache(c, rand(B, 500, H, D, seed=1), rand(B, 500, H, D, seed=2), seq_idx=ids.cuda())
    for s in range(8):
        q, k, v = (rand(B, 1, H, D, seed=50 + 3 * s + i) for i in range(3))
        cached_attention_step(q, k, v, c)
        assert c.lengths.tolist() == [63 + s, 127 + s, 501 + s, 1 + s]
        rk, _ = read_kv_cache(c)
        for b, n in enumerate((62, 126, 500, 0)):
            want = quantise(k[b, 0], "int8")[2]
            assert float((rk[b, n + s].cpu().double() - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
            assert bool((rk[b, n + s + 1:] == 0).all())


def test_q_of_many_sizes():
    """Queries of 1e-6 and 1e+6 of the usual size keep their 22 bits."""
    from telescope_cache_b200 import cached_attention, init_kv_cache, write_kv_cache

    B, N, H, D = 1, 200, 1, 128
    k, v = rand(B, N, H, D, seed=1), rand(B, N, H, D, seed=2)
    c = init_kv_cache(B, N, H, D, dtype=torch.float32)
    write_kv_cache(c, k, v)
    values = [quantise(t, "int8")[2] for t in (k, v)]
    for f in (1e-6, 1.0, 1e6):
        q = rand(B, 1, 4, D, seed=3) * f
        out, lse = cached_attention(q, c, scale=1 / (f * math.sqrt(D)))
        check(out, lse, q[:, 0], values, [N], torch.float32, scale=1 / (f * math.sqrt(D)))


def test_long_offsets():
    """A cache whose codes pass 2^32 bytes: the last row and head are found."""
    from telescope_cache_b200 import cached_attention, init_kv_cache, read_kv_cache, write_kv_cache

    rows, cap, H, D = 3, 1 << 20, 11, 128  # 4.4e9 codes each of keys and values
    c = init_kv_cache(rows, cap, H, D)
    c.lengths.fill_(cap - 5)
    c.max_length = cap - 5
    k, v = rand(rows, 5, H, D, seed=1), rand(rows, 5, H, D, seed=2)
    write_kv_cache(c, k, v)
    kc, _, kv_ = quantise(k, "int8")
    vc, _, vv = quantise(v, "int8")
    assert torch.equal(c.k[:, :, -5:].cpu().transpose(1, 2), kc) and torch.equal(c.v[:, :, -5:].cpu().transpose(1, 2), vc)
    q = rand(rows, 1, H, D, seed=3, dtype=torch.bfloat16)
    out, lse = cached_attention(q, c)
    # every other key and value is zero: logit 0, value 0
    x = torch.einsum("bhd,bnhd->bhn", q[:, 0].double().cpu(), kv_) / math.sqrt(D)
    total = torch.exp(x).sum(-1) + (cap - 5)
    assert float((lse[:, 0].double().cpu() - total.log()).abs().max()) <= 1e-4
    want = torch.einsum("bhn,bnhd->bhd", torch.exp(x) / total[..., None], vv)
    assert float((out[:, 0].double().cpu() - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())


def test_two_streams():
    from telescope_cache_b200 import cached_attention, init_kv_cache, write_kv_cache

    B, N, H, D = 4, 3000, 4, 128
    c = init_kv_cache(B, N, H, D)
    write_kv_cache(c, rand(B, N, H, D, seed=1), rand(B, N, H, D, seed=2))
    q = rand(B, 1, 16, D, dtype=torch.bfloat16, seed=3)
    want, _ = cached_attention(q, c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(cached_attention(q, c)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_a_negative_length_is_an_empty_row():
    """Lengths set by hand: below zero reads nothing and the next token goes to slot 0."""
    from telescope_cache_b200 import cached_attention, cached_attention_step, init_kv_cache

    for D in (128, 40):
        c = init_kv_cache(2, 100, 2, D)
        c.lengths.copy_(torch.tensor([-7, -1]))
        q, k, v = (rand(2, 1, 2, D, seed=i) for i in range(3))
        out, lse = cached_attention(q, c)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
        cached_attention_step(q, k, v, c)
        assert c.lengths.tolist() == [1, 1]
        assert bool((c.k_scale[:, :, 0] > 0).all()) and bool((c.k_scale[:, :, 1:] == 0).all())


def test_replayed_steps_outlive_a_larger_call():
    """A captured step goes on with its workspace after a larger call on its stream
    took another one, and with lengths that pass those it was planned for."""
    from telescope_cache_b200 import cached_attention, cached_attention_step, init_kv_cache, write_kv_cache

    B, N, H, D = 2, 500, 2, 128
    k, v = rand(B, N, H, D, seed=1), rand(B, N, H, D, seed=2)
    caches = [init_kv_cache(B, 900, H, D) for _ in range(2)]
    for c in caches:
        write_kv_cache(c, k, v)
    q, kt, vt = (rand(B, 1, h, D, dtype=torch.bfloat16, seed=5 + h) for h in (8, H, H))
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cached_attention_step(q, kt, vt, caches[0], advance=False)
    with torch.cuda.graph(graph, stream=s):
        out, lse = cached_attention_step(q, kt, vt, caches[0])
    big = init_kv_cache(8, 6000, 8, D)
    write_kv_cache(big, rand(8, 6000, 8, D, seed=3), rand(8, 6000, 8, D, seed=4))
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cached_attention(rand(8, 1, 64, D, dtype=torch.bfloat16, seed=9), big)
    torch.cuda.synchronize()
    junk = [torch.full((1 << i,), math.nan, device="cuda") for i in range(12, 22)]
    for _ in range(300):
        graph.replay()
        want, wl = cached_attention_step(q, kt, vt, caches[1])
    torch.cuda.synchronize()
    assert len(junk) == 10 and caches[0].lengths.tolist() == caches[1].lengths.tolist() == [800, 800]
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v_scale, caches[1].v_scale)
    # other splits, the same formula: fp32 sums, then one rounding to bf16
    assert float((out.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
    assert float((lse - wl).abs().max()) <= 1e-5 + 8e-6 * float(wl.abs().max())
