"""causal_attention and its gradients against the formula in 64 bits.

Tolerances, fixed before the first run.  16-bit types: P is rounded to the type
before the product with V, the result once more: |out - exact| <= UNIT (sum p |v|
+ |out|).  Gradients round P, dX and the result and take Delta from the rounded
out: 4 UNIT of the norm, and UNIT / 16 of the norm of the terms that cancel in
dP - Delta (roundings of out that point every way: 1 / sqrt(D) of their bound).
fp32: sums of up to a few hundred terms in fp32, 64 units of 2^-24 of the norm,
and 4 of the terms' norm.  lse: fp32 sums of exact products, exp2 to 2^-22,
softcap's tanh to 1e-5 of the logit."""

import math

import pytest
import torch

from full_attention_reference import UNIT, causal, gradient_terms, rel, visible

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def inputs(B, N, Hq, Hkv, Dk, Dv, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return r(B, N, Hq, Dk), r(B, N, Hkv, Dk), r(B, N, Hkv, Dv)


def ids_of(lengths, N):
    """Ids of consecutive examples; a negative length is padding of that many tokens."""
    out, at = [], 0
    for i, n in enumerate(lengths):
        out += [i if n > 0 else -1] * abs(n)
    return torch.tensor(out + [len(lengths)] * (N - len(out)), device="cuda", dtype=torch.int32)[:N]


def grad_tol(dtype):
    return 64 * 2.0 ** -24 if dtype == torch.float32 else 4 * UNIT[dtype]


def check_grads(got, want, terms, dtype):
    part = 4 * 2.0 ** -24 if dtype == torch.float32 else UNIT[dtype] / 16
    for a, b, t in zip(got, want, terms):
        off = float((a.double() - b).norm())
        assert off <= grad_tol(dtype) * float(b.norm()) + part * t, (off, float(b.norm()), t)


def check_forward(out, lse, q, k, v, see, softcap=None, scale=None):
    o, l, top, p = causal(q.double(), k.double(), v.double(), see, softcap, scale)
    E = q.shape[2] // k.shape[2]
    size = torch.einsum("bhnm,bmhd->bnhd", p, v.double().abs().repeat_interleave(E, 2))
    unit = UNIT[q.dtype] if q.dtype != torch.float32 else 64 * 2.0 ** -24
    assert bool(((out.double() - o).abs() <= unit * (size + o.abs()) + 1e-5 * size).all())
    empty = ~see.any(-1)
    assert bool((lse[empty] == -math.inf).all()) and bool((out[empty] == 0).all())
    assert bool(((lse.double() - l)[~empty].abs() <= 1e-5 + 2e-5 * top).all())


SHAPES = [  # B, N, Hq, Hkv, Dk, Dv
    (1, 1, 1, 1, 128, 128), (2, 2, 2, 1, 64, 64), (1, 127, 4, 4, 128, 128), (2, 128, 2, 1, 128, 128),
    (1, 129, 8, 1, 64, 64), (1, 257, 6, 2, 128, 128), (2, 300, 4, 2, 64, 64), (1, 640, 2, 2, 128, 128),
    (1, 1000, 3, 1, 64, 64), (1, 65, 2, 2, 32, 32), (1, 70, 2, 1, 96, 96), (1, 50, 2, 1, 64, 128),
    (1, 40, 2, 2, 200, 256)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,N,Hq,Hkv,Dk,Dv", SHAPES)
@pytest.mark.parametrize("softcap", [None, 15.0])
def test_forward(dtype, B, N, Hq, Hkv, Dk, Dv, softcap):
    from telescope_cache_b200 import causal_attention

    q, k, v = inputs(B, N, Hq, Hkv, Dk, Dv, DT[dtype])
    out, lse = causal_attention(q, k, v, softcap=softcap)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    check_forward(out, lse, q, k, v, visible(None, B, N, "cuda"), softcap)


PACKS = [[1, 1, 1, 125, 1, 300], [-5, 100, -60, 7, 200, -30], [400, -1], [127, 1, 128, 129], [-402], [3, -300, 99]]


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64), ("f32", 64), ("bf16", 80)])
@pytest.mark.parametrize("pack", range(len(PACKS)))
def test_packed_forward_and_gradients(dtype, D, pack):
    """Examples that start and end inside tiles, of one token, padding at the
    front, between and at the end, a row of padding alone."""
    from telescope_cache_b200 import causal_attention, segment_bounds

    dt, B, N, Hq, Hkv = DT[dtype], 2, 402, 4, 2
    q, k, v = inputs(B, N, Hq, Hkv, D, D, dt, seed=pack)
    ids = torch.stack([ids_of(PACKS[pack], N), ids_of(PACKS[(pack + 1) % len(PACKS)], N)])
    see = visible(ids, B, N, "cuda")
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out, lse = causal_attention(q, k, v, seq_idx=ids)
    check_forward(out.detach(), lse.detach(), q.detach(), k.detach(), v.detach(), see)
    again, _ = causal_attention(q.detach(), k.detach(), v.detach(), seq_idx=segment_bounds(ids))
    assert torch.equal(again, out.detach())
    gout, glse = torch.randn_like(out), torch.randn_like(lse)
    got = torch.autograd.grad((out, lse), (q, k, v), (gout, glse))
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]
    o, l, _, _ = causal(*x, see)
    some = see.any(-1)
    loss = (o * gout.double()).sum() + (l * glse.double())[some].sum()
    want = torch.autograd.grad(loss, x) if bool(some.any()) else [torch.zeros_like(t) for t in x]
    glse = torch.where(some[..., None], glse, torch.zeros_like(glse))
    check_grads(got, want, gradient_terms(q, k, v, see, gout, glse), dt)
    for a in got:
        assert bool((a[(~some)] == 0).all())  # padding has no gradient


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,N,Hq,Hkv,Dk,Dv", SHAPES)
@pytest.mark.parametrize("softcap", [None, 15.0])
def test_gradients(dtype, B, N, Hq, Hkv, Dk, Dv, softcap):
    from telescope_cache_b200 import causal_attention, causal_attention_backward

    dt = DT[dtype]
    q, k, v = (t.requires_grad_() for t in inputs(B, N, Hq, Hkv, Dk, Dv, dt, seed=3))
    out, lse = causal_attention(q, k, v, softcap=softcap, scale=0.11)
    gout, glse = torch.randn_like(out), torch.randn_like(lse)
    got = torch.autograd.grad((out, lse), (q, k, v), (gout, glse))
    explicit = causal_attention_backward(q, k, v, out, lse, gout, dlse=glse, softcap=softcap, scale=0.11)
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]
    o, l, _, _ = causal(*x, visible(None, B, N, "cuda"), softcap, 0.11)
    want = torch.autograd.grad((o * gout.double()).sum() + (l * glse.double()).sum(), x)
    terms = gradient_terms(q, k, v, visible(None, B, N, "cuda"), gout, glse, softcap, 0.11)
    check_grads(got, want, terms, dt)
    check_grads(explicit, want, terms, dt)  # from the rounded out alone
    # and the same bits from call to call
    for a, c in zip(explicit, causal_attention_backward(q, k, v, out, lse, gout, dlse=glse, softcap=softcap, scale=0.11)):
        assert torch.equal(a, c)
    for a, c in zip(got, torch.autograd.grad(causal_attention(q, k, v, softcap=softcap, scale=0.11), (q, k, v), (gout, glse))):
        assert torch.equal(a, c)


def test_gradients_against_differences():
    """fp32 gradients against central differences of the 64-bit formula along
    random directions (step 1e-4: truncation 1e-8 of the third derivative)."""
    from telescope_cache_b200 import causal_attention

    B, N, Hq, Hkv, D = 1, 70, 4, 2, 64
    q, k, v = (t.requires_grad_() for t in inputs(B, N, Hq, Hkv, D, D, torch.float32, seed=5))
    ids = ids_of([20, -5, 45], N)[None]
    see = visible(ids, B, N, "cuda")
    out, lse = causal_attention(q, k, v, seq_idx=ids, softcap=10.0)
    gout, glse = torch.randn_like(out), torch.randn_like(lse)
    glse = torch.where(see.any(-1)[..., None], glse, torch.zeros_like(glse))
    got = torch.autograd.grad((out, lse), (q, k, v), (gout, glse))

    def f(x):
        o, l, _, _ = causal(*x, see, 10.0)
        return float((o * gout.double()).sum() + torch.nan_to_num(l * glse.double(), nan=0.0).sum())

    x = [t.detach().double() for t in (q, k, v)]
    for i in range(3):
        t = torch.randn_like(x[i])
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + 1e-4 * t, x[i] - 1e-4 * t
        want = (f(up) - f(down)) / 2e-4
        assert abs(float((got[i].double() * t).sum()) - want) <= 1e-4 * float(got[i].double().norm() * t.norm())


@pytest.mark.parametrize("D", [64, 128])
def test_backward_repeats_bit_for_bit(D):
    """Warps of a last block with few rows run ahead of those with work."""
    from telescope_cache_b200 import causal_attention, causal_attention_backward

    q, k, v = inputs(4, 912, 16, 4, D, D, torch.bfloat16, seed=8)
    out, lse = causal_attention(q, k, v)
    gout = torch.randn_like(out)
    want = causal_attention_backward(q, k, v, out, lse, gout)
    for _ in range(50):
        for a, b in zip(causal_attention_backward(q, k, v, out, lse, gout), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("D", [72, 128])
def test_gradients_of_many_blocks(D):
    """fp32 with enough blocks of keys for every SM, and a tail of 6 tokens."""
    from telescope_cache_b200 import causal_attention

    dt, B, N, Hq, Hkv = torch.float32, 37, 70, 8, 4
    q, k, v = (t.requires_grad_() for t in inputs(B, N, Hq, Hkv, D, D, dt, seed=6))
    out, lse = causal_attention(q, k, v, scale=0.11)
    gout, glse = torch.randn_like(out), torch.randn_like(lse)
    got = torch.autograd.grad((out, lse), (q, k, v), (gout, glse))
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]
    see = visible(None, B, N, "cuda")
    o, l, _, _ = causal(*x, see, None, 0.11)
    want = torch.autograd.grad((o * gout.double()).sum() + (l * glse.double()).sum(), x)
    check_grads(got, want, gradient_terms(q, k, v, see, gout, glse, None, 0.11), dt)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64), ("f32", 64)])
def test_strided_views(dtype, D):
    """q, k, v as views of a fused projection, with heads before tokens, and with
    a base address 2 or 4 bytes off."""
    from telescope_cache_b200 import causal_attention

    dt, B, N, Hq, Hkv = DT[dtype], 2, 150, 4, 2
    x = torch.randn(B, N, (Hq + 2 * Hkv) * D, device="cuda").to(dt)
    a = [t.view(B, N, -1, D) for t in x.split([Hq * D, Hkv * D, Hkv * D], -1)]
    b = [torch.randn(B, h, N, D, device="cuda").to(dt).transpose(1, 2) for h in (Hq, Hkv, Hkv)]
    y = torch.randn(B * N * (Hq + 2 * Hkv) * D + 1, device="cuda").to(dt)[1:]
    c = [t.view(B, N, -1, D) for t in y.split([B * N * Hq * D, B * N * Hkv * D, B * N * Hkv * D])]
    e = [torch.randn(B, N, D, h, device="cuda").to(dt).transpose(2, 3) for h in (Hq, Hkv, Hkv)]
    for views in (a, b, c, e):
        dense = [t.contiguous() for t in views]
        out, lse = causal_attention(*views)
        check_forward(out, lse, *dense, visible(None, B, N, "cuda"))
        v1 = [t.detach().requires_grad_() for t in views]
        v2 = [t.detach().requires_grad_() for t in dense]
        g = torch.randn_like(out)
        for s, t in zip(torch.autograd.grad(causal_attention(*v1)[0], v1, g),
                        torch.autograd.grad(causal_attention(*v2)[0], v2, g)):
            assert rel(s, t) <= grad_tol(dt)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_large_logits_and_masked_extremes(dtype):
    """Logits of +-1e3, and the largest values of the type in keys that no query
    of interest sees: the first example's rows are as without them."""
    from telescope_cache_b200 import causal_attention

    dt, B, N, Hq, Hkv, D = DT[dtype], 1, 400, 2, 1, 64
    q, k, v = inputs(B, N, Hq, Hkv, D, D, dt, seed=9)
    q = (q.float() * 12).to(dt)
    k = (k.float() * 12).to(dt)
    out, lse = causal_attention(q, k, v)
    o, l, top, _ = causal(q.double(), k.double(), v.double(), visible(None, B, N, "cuda"))
    assert top > 500
    # a logit of size top carries an fp32 error of top 2^-23: relative error of P
    assert rel(out, o) <= UNIT[dt] + 4 * top * 2.0 ** -23
    assert float((lse.double() - l).abs().max()) <= 1e-5 + 4 * top * 2.0 ** -23
    ids = ids_of([130, 270], N)[None]
    base, base_lse = causal_attention(q, k, v, seq_idx=ids)
    big = float(torch.finfo(dt).max)
    k2, v2 = k.clone(), v.clone()
    k2[:, 256:], v2[:, 256:] = -big, big
    got, got_lse = causal_attention(q, k2, v2, seq_idx=ids)
    assert torch.equal(got[:, :130], base[:, :130]) and torch.equal(got_lse[:, :130], base_lse[:, :130])


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64), ("f32", 64)])
def test_nan_of_later_tiles_stays_there(dtype, D):
    """A NaN in a key's and value's row never reaches queries that precede its
    128-token block."""
    from telescope_cache_b200 import causal_attention

    q, k, v = inputs(1, 600, 2, 1, D, D, DT[dtype], seed=4)
    base, _ = causal_attention(q, k, v)
    k2, v2 = k.clone(), v.clone()
    k2[:, 384], v2[:, 384] = math.nan, math.inf
    got, lse = causal_attention(q, k2, v2)
    assert torch.equal(got[:, :384], base[:, :384])
    assert bool(lse[:, 384:].isnan().all()) and bool(got[:, 384:].isnan().all())


def test_sink_follows():
    """The (out, lse) boundary composes with the framework's sink, gradients
    through both."""
    from telescope_cache_b200 import apply_attention_sink, causal_attention

    B, N, Hq, Hkv, D = 1, 90, 4, 2, 64
    q, k, v = (t.requires_grad_() for t in inputs(B, N, Hq, Hkv, D, D, torch.float32, seed=8))
    sinks = torch.randn(Hq, device="cuda", requires_grad=True)
    y = apply_attention_sink(*causal_attention(q, k, v), sinks)
    g = torch.randn_like(y)
    got = torch.autograd.grad(y, (q, k, v, sinks), g)
    x = [t.detach().double().requires_grad_() for t in (q, k, v, sinks)]
    see = visible(None, B, N, "cuda")
    o, l, _, _ = causal(*x[:3], see)
    want = torch.autograd.grad(o * torch.sigmoid(l - x[3])[..., None], x, g.double())
    check_grads(got[:3], want[:3], [2 * t for t in gradient_terms(q, k, v, see, g, l.detach())], torch.float32)
    assert rel(got[3], want[3]) <= 2 * grad_tol(torch.float32)


def test_empty_batch_and_other_stream():
    from telescope_cache_b200 import causal_attention

    q, k, v = inputs(2, 200, 4, 2, 128, 128, torch.bfloat16)
    out, lse = causal_attention(q[:, :0], k[:, :0], v[:, :0])
    assert out.shape == (2, 0, 4, 128) and lse.shape == (2, 0, 4)
    want, _ = causal_attention(q, k, v)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, _ = causal_attention(q, k, v)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("N", [1, 31, 1024, 1025, 5000])
def test_segment_bounds(N):
    from telescope_cache_b200 import segment_bounds

    g = torch.Generator().manual_seed(N)
    ids = torch.randint(-1, 3, (3, N), generator=g).repeat_interleave(3, 1)[:, :N]
    ids[2] = 0
    seg = segment_bounds(ids.cuda())
    for b in range(3):
        for n in range(N):
            s, e = n, n + 1
            while s > 0 and ids[b, s - 1] == ids[b, n] and b < 2:
                s -= 1
            while e < N and ids[b, e] == ids[b, n] and b < 2:
                e += 1
            if b == 2:
                s, e = 0, N
            if ids[b, n] < 0:
                s, e = n + 1, n
            if n % 97 == 0 or N < 100:
                assert (int(seg.starts[b, n]), int(seg.ends[b, n])) == (s, e), (b, n)
    pos = seg.positions()
    assert bool((pos >= 0).all()) and torch.equal(pos[2].cpu(), torch.arange(N, dtype=torch.int32))


def test_second_derivatives_are_refused():
    """They are not built: an error, not zeros."""
    from telescope_cache_b200 import causal_attention

    q, k, v = (t.requires_grad_() for t in inputs(1, 20, 2, 1, 64, 64, torch.float32, seed=2))
    out, _ = causal_attention(q, k, v)
    (dq,) = torch.autograd.grad(out.square().sum(), (q,), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dq.square().sum().backward()
