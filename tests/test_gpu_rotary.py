"""rotary against the formula in 64 bits: layouts, partial heads, strides,
positions, types, gradients.

Tolerance: the result is rounded once (UNIT of the type) after three fp32
operations on the pair (4 roundings of 2^-24 of |x1| + |x2| at most)."""

import pytest
import torch

from full_attention_reference import UNIT, rotate

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def inputs(B, N, Hq, Hk, D, R, dtype, n_pos=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, N, (Hq + 2 * Hk) * D, generator=g, device="cuda").to(dtype)
    q, k, _ = x.split([Hq * D, Hk * D, Hk * D], -1)
    ang = torch.rand(n_pos or max(N, 1), R // 2, generator=g, device="cuda") * 6.28
    return q.view(B, N, Hq, D), k.view(B, N, Hk, D), ang.cos(), ang.sin()


def check(got, x, cos, sin, pos, layout, dtype, inverse=False):
    want = rotate(x, cos, sin, pos, layout, inverse)
    R = 2 * cos.shape[1]
    size = x[..., :R].double().abs().amax(-1, keepdim=True) * 2
    assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous()
    assert bool(((got.double() - want).abs() <= UNIT[dtype] * want.abs() + 4 * 2.0 ** -24 * size).all())
    assert torch.equal(got[..., R:], x[..., R:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,N,Hq,Hk,D,R", [
    (1, 1, 1, 1, 64, 64), (64, 1, 16, 16, 128, 128), (2, 77, 16, 4, 128, 64), (1, 513, 5, 1, 96, 32),
    (3, 9, 3, 3, 64, 24), (2, 5, 4, 2, 50, 10), (1, 300, 8, 2, 256, 256), (2, 3, 2, 1, 64, 2),
    (2, 2000, 16, 4, 128, 128), (1, 1500, 9, 3, 128, 24)])
def test_formula(layout, dtype, B, N, Hq, Hk, D, R):
    from telescope_cache_b200 import rotary

    dt = DT[dtype]
    q, k, cos, sin = inputs(B, N, Hq, Hk, D, R, dt)
    pos = torch.arange(N, device="cuda").expand(B, N)
    qr, kr = rotary(q, k, cos, sin, layout=layout)
    check(qr, q, cos, sin, pos, layout, dt)
    check(kr, k, cos, sin, pos, layout, dt)
    one, none = rotary(q, None, cos, sin, layout=layout)
    assert none is None and torch.equal(one, qr)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("kind", ["rows", "shared", "int64"])
def test_positions(layout, kind):
    from telescope_cache_b200 import rotary

    B, N = 3, 41
    q, k, cos, sin = inputs(B, N, 4, 2, 64, 64, torch.float32, n_pos=100)
    pos = torch.randint(0, 100, (N,) if kind == "shared" else (B, N), device="cuda",
                        dtype=torch.int64 if kind == "int64" else torch.int32)
    qr, kr = rotary(q, k, cos, sin, positions=pos, layout=layout)
    p = pos.long().expand(B, N)
    check(qr, q, cos, sin, p, layout, torch.float32)
    check(kr, k, cos, sin, p, layout, torch.float32)
    back, _ = rotary(qr, None, cos, sin, positions=pos, layout=layout, inverse=True)
    # two rotations: twice the single tolerance of a unit rotation
    assert float((back - q).abs().max()) <= 16 * 2.0 ** -24 * float(q.abs().max())


def test_position_outside_the_tables_is_nan_and_only_there():
    from telescope_cache_b200 import rotary

    q, k, cos, sin = inputs(1, 6, 2, 1, 64, 32, torch.bfloat16, n_pos=4)
    pos = torch.tensor([0, 3, 4, -1, 2 ** 31 - 1, 1], device="cuda")
    qr, kr = rotary(q, k, cos, sin, positions=pos)
    bad = torch.tensor([False, False, True, True, True, False], device="cuda")
    for y, x in ((qr, q), (kr, k)):
        assert bool(y[0, bad, :, :32].isnan().all()) and bool(y[0, ~bad].isfinite().all())
        assert torch.equal(y[..., 32:], x[..., 32:])


def test_strides_and_alignment():
    """Transposed heads, a base that is 2 bytes off, a dim that is not dense."""
    from telescope_cache_b200 import rotary

    B, N, H, D = 2, 33, 4, 64
    _, _, cos, sin = inputs(B, N, H, H, D, D, torch.bfloat16)
    pos = torch.arange(N, device="cuda").expand(B, N)
    x = torch.randn(B * N * H * D + 1, device="cuda").to(torch.bfloat16)
    views = [x[: -1].view(B, H, N, D).transpose(1, 2), x[1:].view(B, N, H, D), x[: -1].view(B, N, D, H).transpose(2, 3),
             x[: -1].view(N, B, H, D).transpose(0, 1)]
    for v in views:
        for layout in ("half", "interleaved"):
            qr, kr = rotary(v, v, cos, sin, layout=layout)
            check(qr, v, cos, sin, pos, layout, torch.bfloat16)
            assert torch.equal(qr, kr)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", list(DT))
def test_gradients(layout, dtype):
    """The VJP against the formula's, and (fp32) against differences."""
    from telescope_cache_b200 import rotary

    dt = DT[dtype]
    B, N, Hq, Hk, D, R = 2, 19, 4, 2, 64, 32
    q, k, cos, sin = inputs(B, N, Hq, Hk, D, R, dt)
    cos, sin = cos * 1.25, sin * 1.25  # tables may carry a magnitude
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    qr, kr = rotary(q, k, cos, sin, layout=layout)
    dq, dk = torch.autograd.grad((qr, kr), (q, k), (gq, gk))
    pos = torch.arange(N, device="cuda").expand(B, N)
    check(dq, gq, cos, sin, pos, layout, dt, inverse=True)
    check(dk, gk, cos, sin, pos, layout, dt, inverse=True)
    if dt == torch.float32:
        t = torch.randn_like(q)
        f = lambda x: float((rotate(x.detach(), cos, sin, pos, layout) * gq.double()).sum())  # noqa: E731
        want = (f(q.double() + t.double()) - f(q.double() - t.double())) / 2  # linear: exact
        assert abs(float((dq.double() * t.double()).sum()) - want) <= 1e-5 * float(dq.norm() * t.norm())


def test_gradient_of_one_alone():
    from telescope_cache_b200 import rotary

    q, k, cos, sin = inputs(1, 7, 2, 2, 64, 64, torch.float32)
    q = q.detach().requires_grad_()
    qr, kr = rotary(q, k, cos, sin)
    (dq,) = torch.autograd.grad(qr.sum(), q)
    check(dq, torch.ones_like(q), cos, sin, torch.arange(7, device="cuda")[None], "half", torch.float32, inverse=True)
    (d2,) = torch.autograd.grad(rotary(q, None, cos, sin)[0].sum(), q)
    assert torch.equal(dq, d2)


def test_empty_and_other_stream():
    from telescope_cache_b200 import rotary

    q, k, cos, sin = inputs(2, 64, 4, 2, 64, 64, torch.bfloat16)
    e, _ = rotary(q[:, :0], k[:, :0], cos, sin)
    assert e.shape == (2, 0, 4, 64)
    want, _ = rotary(q, k, cos, sin)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, _ = rotary(q, k, cos, sin)
    s.synchronize()
    assert torch.equal(got, want)


def test_agrees_with_apply_rope():
    from telescope_cache_b200 import apply_rope, rope_tables, rotary

    q, k, _, _ = inputs(2, 40, 4, 2, 64, 64, torch.float32)
    cos, sin = rope_tables(40, 64, device="cuda")
    got, _ = rotary(q, k, cos, sin)
    want = apply_rope(q, torch.arange(40, device="cuda")[None, :, None], cos, sin)
    assert float((got - want).abs().max()) <= 8 * 2.0 ** -24 * float(q.abs().max())


def test_second_derivatives():
    """y = Rx, g = R^T (2 Rx) = 2 x for tables of magnitude one: d(g^2)/dx = 8 x."""
    from telescope_cache_b200 import rotary, rotary_tables

    cos, sin = rotary_tables(9, 32, device="cuda")
    q, k = (torch.randn(2, 9, h, 32, device="cuda", requires_grad=True) for h in (4, 2))
    yq, yk = rotary(q, k, cos, sin)
    g = torch.autograd.grad(yq.square().sum() + yk.square().sum(), (q, k), create_graph=True)
    for x, dx in zip((q, k), torch.autograd.grad(sum(t.square().sum() for t in g), (q, k))):
        # four rotations, each two products and a sum of at most sqrt(2) of the pair's size
        assert float((dx - 8 * x).abs().max()) <= 4 * 6 * 2.0 ** -24 * 8 * float(x.abs().max()) + 8 * 4 * 2.0 ** -24
