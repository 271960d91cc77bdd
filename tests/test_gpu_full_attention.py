"""The full-attention operators together: the layer in training, prompt and token
form, and the refusals of the public calls."""

import math

import pytest
import torch

from full_attention_reference import UNIT, causal, rel, rotate, visible

pytestmark = pytest.mark.gpu


def layer(D, dtype, **kw):
    from telescope_cache_b200.fms_attention import FullMultiHeadAttention

    torch.manual_seed(0)
    m = FullMultiHeadAttention(96, D, D, 4, 2, **kw).to("cuda", dtype)
    with torch.no_grad():
        m.in_proj.weight.mul_(6.0)
        if kw.get("use_sinks"):
            m.sinks.normal_()
    return m


def plain(m, x, seq_idx, see):
    """The layer in 64 bits; parameters and x as double leaves."""
    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}
    x = x.detach().double().requires_grad_()
    B, N, _ = x.shape
    y = x @ p["in_proj.weight"].T
    q, k, v = y.split(m._split, -1)
    q, k, v = q.view(B, N, m.nheads, -1), k.view(B, N, m.kvheads, -1), v.view(B, N, m.kvheads, -1)
    pos = torch.arange(N, device=x.device).expand(B, N)
    if seq_idx is not None:
        start = torch.stack([torch.tensor([next((j for j in range(n, -1, -1) if j == 0 or r[j - 1] != r[j]), 0)
                                           for n in range(N)]) for r in seq_idx.cpu().tolist()]).to(x.device)
        pos = torch.where(seq_idx >= 0, pos - start, 0)
    cos, sin = m._tables(N, x.device)
    q, k = rotate_(q, cos, sin, pos, m.rope_layout), rotate_(k, cos, sin, pos, m.rope_layout)
    out, lse, _, _ = causal(q, k, v, see, m.softcap)
    if m.use_sinks:
        out = out * torch.sigmoid(lse - p["sinks"])[..., None]
    if m.use_gate:
        out = torch.nn.functional.silu(x @ p["gate_proj.weight"].T).view_as(out) * out
    return out.reshape(B, N, -1) @ p["dense.weight"].T, p, x


def rotate_(x, cos, sin, pos, layout):
    """rotate() that autograd passes through."""
    R = 2 * cos.shape[1]
    c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]
    head, tail = x[..., :R], x[..., R:]
    a, b = (head[..., 0::2], head[..., 1::2]) if layout == "interleaved" else (head[..., : R // 2], head[..., R // 2:])
    u, w = a * c - b * s, b * c + a * s
    y = torch.stack([u, w], -1).flatten(-2) if layout == "interleaved" else torch.cat([u, w], -1)
    return torch.cat([y, tail], -1)


def test_rotate_forms_agree():
    x = torch.randn(1, 5, 2, 12, dtype=torch.float64)
    cos, sin = torch.rand(5, 4), torch.rand(5, 4)
    for layout in ("half", "interleaved"):
        pos = torch.arange(5)[None]
        assert torch.allclose(rotate_(x, cos, sin, pos, layout), rotate(x, cos, sin, pos, layout), atol=1e-12)


@pytest.mark.parametrize("dtype,D,kw", [
    (torch.float32, 64, dict(use_sinks=True, use_gate=True, softcap=20.0, rope_dim=32, rope_layout="interleaved")),
    (torch.float32, 48, dict()),
    (torch.bfloat16, 128, dict(use_sinks=True)),
    (torch.bfloat16, 64, dict(softcap=30.0, rope_scaling=dict(scaling="linear", factor=2.0)))])
@pytest.mark.parametrize("packed", [False, True])
def test_layer_trains(dtype, D, kw, packed):
    """Output and the gradient of the input and every parameter.  bf16: a chain of
    five rounded tensors, 8 units of the norm; fp32: products of 96 to 256 terms."""
    m = layer(D, dtype, **kw)
    B, N = 2, 150
    x = torch.randn(B, N, 96, device="cuda").to(dtype).requires_grad_()
    ids = None
    if packed:
        ids = torch.zeros(B, N, dtype=torch.int32, device="cuda")
        ids[0, 40:] = 1
        ids[0, 139:] = -1
        ids[1, 130:] = 7
    see = visible(ids, B, N, "cuda")
    y = m(x, seq_idx=ids)
    want, p, xd = plain(m, x, ids, see)
    tol = 8 * UNIT[dtype] if dtype == torch.bfloat16 else 1e-5
    live = see.any(-1)
    assert rel(y[live], want[live]) <= tol
    g = torch.randn_like(y) * live[..., None]
    params = dict(m.named_parameters())
    got = torch.autograd.grad(y, [x] + list(params.values()), g)
    ref = torch.autograd.grad(want[live], [xd] + [p[n] for n in params], g.double()[live])
    for n, a, b in zip(["x"] + list(params), got, ref):
        assert rel(a, b) <= 2 * tol, n


@pytest.mark.parametrize("store", ["int8", "fp8"])
def test_layer_prompt_then_tokens(store):
    """Packed prompts into the cache, then tokens: each token's output is the full
    layer's at its place, up to the cache's 8 bits (int8: 1/254 of a row's largest
    value, about 1% of its norm; e4m3: 2^-4 at most, 2.6% of the norm)."""
    m = layer(64, torch.float32, use_sinks=True, cache_store=store, rope_layout="interleaved")
    lens, steps = [30, 1, 75], 5
    xs = [torch.randn(1, n + steps, 96, device="cuda") for n in lens]
    packed = torch.cat([x[:, :n] for x, n in zip(xs, lens)] + [torch.zeros(1, 6, 96, device="cuda")], 1)
    ids = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)] + [torch.full((6,), -1)])[None].to("cuda", torch.int32)
    cache = m.new_cache(3, 300, torch.float32, "cuda")
    with torch.no_grad():
        y = m(packed, seq_idx=ids, cache=cache)
        assert cache.lengths.tolist() == lens
        full = [m(x) for x in xs]
        at = 0
        for f, n in zip(full, lens):
            assert rel(y[0, at: at + n], f[0, :n]) <= 1e-5
            at += n
        for s in range(steps):
            x_t = torch.cat([x[:, n + s: n + s + 1] for x, n in zip(xs, lens)])
            out = m.decode(x_t, cache)
            for i, n in enumerate(lens):
                assert rel(out[i, 0], full[i][0, n + s]) <= (0.03 if store == "int8" else 0.08)
    assert cache.lengths.tolist() == [n + steps for n in lens]


def test_graph_capture_of_a_step():
    """A step captured after a first call replays with new inputs and lengths."""
    from telescope_cache_b200 import cached_attention_step, init_kv_cache, write_kv_cache

    c = init_kv_cache(2, 400, 2, 64)
    k = torch.randn(2, 300, 2, 64, device="cuda").bfloat16()
    write_kv_cache(c, k, k)
    q, kt = torch.randn(2, 1, 4, 64, device="cuda").bfloat16(), torch.randn(2, 1, 2, 64, device="cuda").bfloat16()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        cached_attention_step(q, kt, kt, c, advance=False)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out, lse = cached_attention_step(q, kt, kt, c)
    for i in range(3):
        q.normal_()
        kt.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert c.lengths.tolist() == [301 + i, 301 + i]
        c.lengths -= 1
        want, want_lse = cached_attention_step(q, kt, kt, c)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_refusals():
    from telescope_cache_b200 import (cached_attention, cached_attention_step, causal_attention, causal_attention_backward,
                                      init_kv_cache, read_kv_cache, rotary, segment_bounds, write_kv_cache)

    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    q, k = z(2, 8, 4, 64), z(2, 8, 2, 64)
    t = z(8, 32, dt=torch.float32)

    def no(exc, f):
        with pytest.raises(exc):
            f()

    # rotary: shapes, dtypes, tables, positions
    no(ValueError, lambda: rotary(q[0], k, t, t))
    no(ValueError, lambda: rotary(q, k[:, :4], t, t))
    no(ValueError, lambda: rotary(q, k.half(), t, t))
    no(ValueError, lambda: rotary(q, k, t, t[:4]))
    no(ValueError, lambda: rotary(q, k, t[:4], t[:4]))
    no(ValueError, lambda: rotary(q, k, z(8, 33, dt=torch.float32), z(8, 33, dt=torch.float32)))
    no(ValueError, lambda: rotary(q, k, t, t, positions=z(8, dt=torch.float32)))
    no(ValueError, lambda: rotary(q, k, t, t, positions=torch.zeros(7, device="cuda", dtype=torch.int32)))
    no(ValueError, lambda: rotary(q, k, t, t, layout="both"))
    no(TypeError, lambda: rotary(q.double(), k.double(), t, t))
    no(RuntimeError, lambda: rotary(q, k, t.cpu(), t.cpu()))
    no(NotImplementedError, lambda: rotary(q, k, t.clone().requires_grad_(), t))
    # causal attention
    no(ValueError, lambda: causal_attention(q[0], k, k))
    no(ValueError, lambda: causal_attention(q[:, :, :3], k, k))
    no(ValueError, lambda: causal_attention(q, k[:1], k[:1]))
    no(ValueError, lambda: causal_attention(q, k, k[:, :, :1]))
    no(ValueError, lambda: causal_attention(q, k, k.half()))
    no(ValueError, lambda: causal_attention(q, k, k, softcap=0.0))
    no(ValueError, lambda: causal_attention(q, k, k, seq_idx=z(2, 8)))
    no(ValueError, lambda: causal_attention(q, k, k, seq_idx=torch.zeros(2, 7, device="cuda", dtype=torch.int32)))
    no(ValueError, lambda: causal_attention(q, k, k, seq_idx=segment_bounds(torch.zeros(1, 8, device="cuda", dtype=torch.int32))))
    no(NotImplementedError, lambda: causal_attention(z(1, 2, 2, 300), z(1, 2, 2, 300), z(1, 2, 2, 300)))
    no(NotImplementedError, lambda: causal_attention(z(1, 2, 2, 96), z(1, 2, 2, 96), z(1, 2, 2, 96), impl="tensor"))
    out, lse = causal_attention(q, k, k)
    no(ValueError, lambda: causal_attention_backward(q, k, k, out[:, :4], lse, out))
    no(ValueError, lambda: causal_attention_backward(q, k, k, out, lse.half(), out))
    no(ValueError, lambda: causal_attention_backward(q, k, k, out, lse, out.float()))
    no(ValueError, lambda: causal_attention_backward(q, k, k, out, lse, out, dlse=lse[:1]))
    no(ValueError, lambda: segment_bounds(z(2, 8)))
    # cache
    c = init_kv_cache(2, 10, 2, 64)
    no(ValueError, lambda: write_kv_cache(c, k[:, :, :1], k[:, :, :1]))
    no(ValueError, lambda: write_kv_cache(c, k, k[:1]))
    no(ValueError, lambda: write_kv_cache(c, z(3, 1, 2, 64), z(3, 1, 2, 64)))
    no(ValueError, lambda: write_kv_cache(c, z(2, 11, 2, 64), z(2, 11, 2, 64)))
    no(ValueError, lambda: write_kv_cache(c, k, k, seq_idx=torch.zeros(2, 7, device="cuda", dtype=torch.int32)))
    no(ValueError, lambda: read_kv_cache(c, 11))
    no(ValueError, lambda: cached_attention(q, c))
    no(ValueError, lambda: cached_attention(z(3, 1, 4, 64), c))
    no(ValueError, lambda: cached_attention(z(2, 1, 3, 64), c))
    no(ValueError, lambda: cached_attention(z(2, 1, 4, 32), c))
    no(ValueError, lambda: cached_attention(q[:, :1], c, softcap=-1.0))
    q1, k1 = q[:, :1], k[:, :1]
    no(ValueError, lambda: cached_attention_step(q1, k1, k1.half(), c))
    no(ValueError, lambda: cached_attention_step(q1, k1[:1], k1[:1], c))
    no(ValueError, lambda: cached_attention_step(q1, None, None, c))
    no(ValueError, lambda: cached_attention_step(q1, k1, k1, c, rope_cos=t))
    no(ValueError, lambda: cached_attention_step(q1, k1, k1, c, rope_cos=t[:0], rope_sin=t[:0]))
    no(ValueError, lambda: cached_attention_step(q1, k1, k1, c, layout="both"))
    assert c.lengths.tolist() == [0, 0] and c.max_length == 0  # nothing was written on the way
    write_kv_cache(c, z(2, 10, 2, 64), z(2, 10, 2, 64))
    no(ValueError, lambda: cached_attention_step(q1, k1, k1, c))  # full
    no(ValueError, lambda: write_kv_cache(c, k1, k1))
    bad = init_kv_cache(2, 10, 2, 64)
    bad.k = bad.k.transpose(0, 1)
    no(ValueError, lambda: cached_attention(q1, bad))
    bad = init_kv_cache(2, 10, 2, 64)
    bad.store = "int3"
    no(ValueError, lambda: cached_attention(q1, bad))


def test_wide_groups_and_scale():
    """More query heads to a key head than one CTA takes (8), and a scale of one's own."""
    from telescope_cache_b200 import causal_attention

    q, k, v = (torch.randn(1, 200, h, 64, device="cuda").bfloat16() for h in (24, 2, 2))
    out, lse = causal_attention(q, k, v, scale=0.5)
    o, l, top, _ = causal(q.double(), k.double(), v.double(), visible(None, 1, 200, "cuda"), None, 0.5)
    assert rel(out, o) <= 2 * UNIT[torch.bfloat16] and float((lse - l).abs().max()) <= 1e-5 + 2e-5 * top
    assert math.isfinite(float(lse.sum()))
