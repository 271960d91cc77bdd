"""Causal attention at the edges of its contract: the order of its products, what
a caller may pass for scale, softcap, ids, bounds and addresses.

Tolerances are test_gpu_causal.py's, by check_forward and check_grads."""

import pytest
import torch

from full_attention_reference import causal, gradient_terms, rel, visible
from test_gpu_causal import DT, check_forward, check_grads, grad_tol, ids_of, inputs

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


@pytest.mark.parametrize("D", [64, 128])
def test_c_entries_take_any_address(D):
    """Results one element off a 16-byte boundary: the forward's out and what its
    rounding left over, the backward's three gradients, one at a time."""
    from telescope_cache_b200 import _lib

    dt, B, N, Hq, Hkv = torch.bfloat16, 1, 200, 4, 2
    q, k, v = inputs(B, N, Hq, Hkv, D, D, dt, seed=31)
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    strides = {f"{n}_stride_{a}": t.stride(i) for n, t in (("q", q), ("k", k), ("v", v)) for i, a in enumerate("bnh")}
    args = _lib.CausalArgs(B=B, N=N, Hq=Hq, Hkv=Hkv, Dk=D, Dv=D, dtype=_lib.dtype_code(dt), scale=D ** -0.5,
                           q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), **strides)
    gout = torch.randn_like(q)

    def run(off):  # the named results start one element late
        def room(name, *shape, dtype=dt):
            n = torch.Size(shape).numel()
            return torch.empty(n + 8, device="cuda", dtype=dtype)[int(name == off):][:n].view(shape)

        r = {n: room(n, B, N, Hq, D) for n in ("out", "out_low", "dq")} | {n: room(n, B, N, Hkv, D) for n in ("dk", "dv")}
        lse, delta = (torch.empty(B, N, Hq, device="cuda") for _ in range(2))
        for n, t in r.items():
            setattr(args, n, t.data_ptr())
        args.lse, args.delta, args.o, args.o_low, args.dout = (t.data_ptr() for t in (lse, delta, r["out"], r["out_low"], gout))
        assert lib.tc_causal_fwd(args, stream) == 0 and lib.tc_causal_bwd(args, stream) == 0
        torch.cuda.synchronize()
        return r, lse

    base, base_lse = run(None)
    check_forward(base["out"], base_lse, q, k, v, visible(None, B, N, "cuda"))
    for off in base:
        got, lse = run(off)
        check_forward(got["out"], lse, q, k, v, visible(None, B, N, "cuda"))
        for n in ("dq", "dk", "dv"):
            assert rel(got[n], base[n].double()) <= 2 * grad_tol(dt)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap", [None, 15.0])
@pytest.mark.parametrize("scale", [-0.11, 0.0, 1e-35])
def test_any_finite_scale(dtype, D, softcap, scale):
    from telescope_cache_b200 import causal_attention

    dt, B, N, Hq, Hkv = DT[dtype], 1, 300, 4, 2
    q, k, v = (t.requires_grad_() for t in inputs(B, N, Hq, Hkv, D, D, dt, seed=17))
    see = visible(None, B, N, "cuda")
    # softcap and negative scale: logits beyond the cap, where a series would leave tanh
    q.data.mul_(8)
    out, lse = causal_attention(q, k, v, softcap=softcap, scale=scale)
    check_forward(out.detach(), lse.detach(), q.detach(), k.detach(), v.detach(), see, softcap, scale)
    gout, glse = torch.randn_like(out), torch.randn_like(lse)
    got = torch.autograd.grad((out, lse), (q, k, v), (gout, glse))
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]
    o, l, _, _ = causal(*x, see, softcap, scale)
    want = torch.autograd.grad((o * gout.double()).sum() + (l * glse.double()).sum(), x)
    terms = gradient_terms(q, k, v, see, gout, glse, softcap, scale)
    if dt == torch.float16 and scale == 1e-35:  # dq, dk are far below its smallest number
        assert bool((got[0] == 0).all()) and bool((got[1] == 0).all())
        got, want, terms = got[2:], want[2:], terms[2:]
    check_grads(got, want, terms, dt)


def test_scales_that_are_refused():
    from telescope_cache_b200 import cached_attention, causal_attention, init_kv_cache

    q, k, v = inputs(1, 20, 2, 1, 64, 64, torch.bfloat16)
    c = init_kv_cache(1, 10, 1, 64)
    for scale in (float("nan"), float("inf"), -float("inf"), 1e39):
        with pytest.raises(ValueError, match="scale"):
            causal_attention(q, k, v, scale=scale)
        with pytest.raises(ValueError, match="scale"):
            cached_attention(q[:, :1], c, scale=scale)
    with pytest.raises(NotImplementedError):  # the tensor-core kernels need it positive
        causal_attention(q, k, v, scale=-1.0, impl="tensor")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap", [1e-7, 1e-3, 1500.0, 1e5, 1e7])
def test_any_softcap(dtype, D, softcap):
    """Caps far below and above the logits.  One query is large: its logits pass the
    larger caps while those of its neighbours stay small beside them."""
    from telescope_cache_b200 import causal_attention

    dt, B, N, Hq, Hkv = DT[dtype], 1, 300, 4, 2
    q, k, v = inputs(B, N, Hq, Hkv, D, D, dt, seed=18)
    if softcap < 1e-5 and dtype != "f16":  # logits around the cap (f16 has no numbers so small)
        q.mul_(1e-8)
    elif softcap > 1000:
        q[:, 7] *= softcap / 30 if dtype != "f16" else min(softcap / 30, 8000.0)
    see = visible(None, B, N, "cuda")
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out, lse = causal_attention(q, k, v, softcap=softcap)
    check_forward(out.detach(), lse.detach(), q.detach(), k.detach(), v.detach(), see, softcap)
    gout, glse = torch.randn_like(out), torch.randn_like(lse)
    gout[:, 7], glse[:, 7] = 0, 0  # the neighbours' gradients are what is looked at
    got = torch.autograd.grad((out, lse), (q, k, v), (gout, glse))
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]
    o, l, _, _ = causal(*x, see, softcap)
    want = torch.autograd.grad((o * gout.double()).sum() + (l * glse.double()).sum(), x)
    check_grads(got, want, gradient_terms(q, k, v, see, gout, glse, softcap), dt)


def test_softcaps_that_are_refused():
    from telescope_cache_b200 import cached_attention, causal_attention, init_kv_cache

    q, k, v = inputs(1, 20, 2, 1, 64, 64, torch.bfloat16)
    c = init_kv_cache(1, 10, 1, 64)
    for softcap in (float("nan"), float("inf"), 0.0, -2.0, 1e-50, 1e39):
        with pytest.raises(ValueError, match="softcap"):
            causal_attention(q, k, v, softcap=softcap)
        with pytest.raises(ValueError, match="softcap"):
            cached_attention(q[:, :1], c, softcap=softcap)


@pytest.mark.parametrize("N", [5, 300, 2500])
def test_ids_of_64_bits(N):
    """Ids that agree in their low 32 bits, or whose low 32 bits are negative, are
    what they are in 64."""
    from telescope_cache_b200 import causal_attention, segment_bounds

    ids = ids_of([N // 3, -(N // 5), N // 4], N)[None].long()
    want = segment_bounds(ids.int())
    for wide in (ids * 2 ** 32 + 7, ids * 2 ** 40 + 2 ** 31, 2 ** 62 - ids):
        wide = torch.where(ids < 0, -(2 ** 33), wide)
        for t in (wide, wide.expand(3, N), wide.repeat_interleave(2, 1)[:, ::2]):
            got = segment_bounds(t)
            for a, b in zip(got, want):
                assert a.dtype == torch.int32 and torch.equal(a, b.expand(t.shape[0], N))
    for small in (torch.int8, torch.uint8, torch.int16):
        t = ids.to(small) if small != torch.uint8 else ids.clamp(min=0).to(small)
        got, ref = segment_bounds(t), segment_bounds(t.int())
        assert torch.equal(got.starts, ref.starts) and torch.equal(got.ends, ref.ends)
    q, k, v = inputs(1, N, 2, 1, 64, 64, torch.bfloat16, seed=2)
    wide = torch.where(ids < 0, -1, ids * 2 ** 32 + 2 ** 31)
    assert torch.equal(causal_attention(q, k, v, seq_idx=wide)[0], causal_attention(q, k, v, seq_idx=want)[0])


def test_positions_of_64_bits():
    from telescope_cache_b200 import rotary

    q, k, _ = inputs(1, 5, 2, 1, 64, 64, torch.float32)
    ang = torch.rand(8, 32, device="cuda")
    pos = torch.tensor([0, 2 ** 32 + 1, -(2 ** 32) + 2, 2 ** 33, 7], device="cuda")
    y, _ = rotary(q, k, ang.cos(), ang.sin(), positions=pos)
    want, _ = rotary(q, k, ang.cos(), ang.sin(), positions=torch.tensor([0, -1, -1, -1, 7], device="cuda"))
    assert bool(y[:, 1:4].isnan().all()) and torch.equal(y[:, [0, 4]], want[:, [0, 4]]) and bool(y[:, [0, 4]].isfinite().all())


def test_cache_rows_of_64_bits():
    from telescope_cache_b200 import init_kv_cache, write_kv_cache
    from telescope_cache_b200.telescoping_attn.attention import read_device_status

    read_device_status("cuda:0")
    c = init_kv_cache(2, 8, 1, 64)
    k = torch.randn(1, 6, 1, 64, device="cuda")
    ids = torch.tensor([[0, 0, 2 ** 32, 2 ** 32 + 1, -(2 ** 32) + 1, 1]], device="cuda")
    write_kv_cache(c, k, k, seq_idx=ids)
    assert read_device_status("cuda:0") & 2  # rows that do not exist
    assert c.lengths.tolist() == [2, 1]


def test_tangents_are_refused():
    """Forward-mode derivatives are not built: an error, not a result without one."""
    import torch.autograd.forward_ad as fwd
    from telescope_cache_b200 import cached_attention, causal_attention, init_kv_cache, rotary

    q, k, v = inputs(1, 20, 2, 1, 64, 64, torch.float32)
    ang = torch.rand(20, 32, device="cuda")
    c = init_kv_cache(1, 10, 1, 64)
    with fwd.dual_level():
        for i in range(3):
            x = [q, k, v]
            x[i] = fwd.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|forward AD|jvp"):
                causal_attention(*x)
            if i < 2:
                with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|forward AD|jvp"):
                    rotary(*x[:2], ang.cos(), ang.sin())
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|forward AD|jvp"):
            cached_attention(fwd.make_dual(q[:, :1], torch.ones_like(q[:, :1])), c)
        out, _ = causal_attention(q, k, v)  # none of them dual: as ever
    assert bool(out.isfinite().all())


def rounded_gradients(q, k, v, gout, glse, see, scale, dt):
    """dq, dk in 64 bits, and as they are with dX rounded to dt before its products and
    the results after them: what a kernel with 16-bit operands cannot avoid."""
    E = q.shape[2] // k.shape[2]
    p = causal(q, k, v, see, None, scale)[3]
    dp = torch.einsum("bnhd,bmhd->bhnm", gout, v.repeat_interleave(E, 2))
    dx = p * (dp - (p * dp).sum(-1, keepdim=True) + glse.permute(0, 2, 1)[..., None])
    out = []
    for x, r in ((dx, lambda t: t), (dx.float().to(dt).double(), lambda t: t.float().to(dt).double())):
        dq = r(torch.einsum("bhnm,bmhd->bnhd", x, k.repeat_interleave(E, 2)) * scale)
        dk = r(torch.einsum("bhnm,bnhd->bmhd", x, q).unflatten(2, (-1, E)).sum(3) * scale)
        out.append((dq, dk))
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N,mean,sharp,example", [(40, 8.0, 1, 40), (128, 8.0, 1, 5), (128, 0.0, 1, 3), (700, 8.0, 1, 700),
                                                  (700, 8.0, 4, 700), (700, 2.0, 4, 90), (700, 0.0, 4, 700)])
def test_gradients_of_values_that_share_a_mean(dtype, D, N, mean, sharp, example):
    """dP - Delta is small beside its terms there.  Delta comes from the forward's
    rounded weights: normalised by their own sum, each adds a rounding of its share
    of dX, at most as much again as the rounding of dX itself: with it and the
    result's, three for two, sqrt(3 / 2) = 1.22 of what rounded_gradients leaves."""
    from telescope_cache_b200 import causal_attention

    dt, Hq, Hkv, scale = DT[dtype], 4, 2, D ** -0.5
    q, k, v = inputs(1, N, Hq, Hkv, D, D, dt, seed=23)
    q, v = (q.float() * sharp).to(dt), (v.float() + mean).to(dt)
    ids = (torch.arange(N, device="cuda") // example)[None]
    see = visible(ids, 1, N, "cuda")
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out, lse = causal_attention(q, k, v, seq_idx=ids)
    gout, glse = torch.randn_like(out), torch.randn_like(lse)
    got = torch.autograd.grad((out, lse), (q, k), (gout, glse))
    want, near = rounded_gradients(*(t.detach().double() for t in (q, k, v, gout, glse)), see, scale, dt)
    for a, w, n in zip(got, want, near):
        assert rel(a, w) <= 1.25 * rel(n, w), (rel(a, w), rel(n, w))
