"""Host side of the full-attention operators, without a GPU: tables, refusals,
the layer's parameters."""

import math

import pytest
import torch

from telescope_cache_b200 import _lib, causal_attention, init_kv_cache, rotary, rotary_tables, segment_bounds
from telescope_cache_b200.fms_attention import FullMultiHeadAttention


def theta(dim, base=10000.0):
    return [base ** (-2 * i / dim) for i in range(dim // 2)]


def check_tables(cos, sin, freqs, n, magnitude=1.0):
    assert cos.dtype == torch.float32 and tuple(cos.shape) == (n, len(freqs)) == tuple(sin.shape)
    for p in (0, 1, n // 2, n - 1):
        for i, f in enumerate(freqs):
            # one fp32 rounding of a 64-bit value
            assert abs(float(cos[p, i]) - magnitude * math.cos(p * f)) <= 2.0 ** -23 * max(1.0, magnitude)
            assert abs(float(sin[p, i]) - magnitude * math.sin(p * f)) <= 2.0 ** -23 * max(1.0, magnitude)


def test_tables_of_each_scaling():
    n, dim = 40000, 16
    check_tables(*rotary_tables(n, dim), theta(dim), n)
    check_tables(*rotary_tables(n, dim, 500000.0, magnitude=1.3), theta(dim, 500000.0), n, 1.3)
    check_tables(*rotary_tables(n, dim, scaling="linear", factor=4.0), [t / 4 for t in theta(dim)], n)
    base = 10000.0 * 4.0 ** (dim / (dim - 2))
    check_tables(*rotary_tables(n, dim, scaling="base", factor=4.0), theta(dim, base), n)
    assert abs(theta(dim, base)[-1] * 4 / theta(dim)[-1] - 1) < 1e-12  # the slowest one: exactly the factor


def test_tables_by_parts():
    n, dim, orig, few, many, f = 5000, 32, 1000, 2.0, 8.0, 8.0
    want = []
    for t in theta(dim):
        turns = orig * t / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - few) / (many - few)))
        want.append(keep * t + (1 - keep) * t / f)
    cos, sin = rotary_tables(n, dim, scaling="parts", factor=f, original_positions=orig, turns=(few, many))
    check_tables(cos, sin, want, n)
    assert want[0] == theta(dim)[0] and want[-1] == theta(dim)[-1] / f and any(a not in (b, b / f) for a, b in zip(want, theta(dim)))


@pytest.mark.parametrize("kw", [dict(dim=7), dict(dim=0), dict(n_pos=0), dict(scaling="other"), dict(factor=0.0, scaling="linear"),
                                dict(factor=2.0), dict(scaling="base", dim=2, factor=2.0), dict(scaling="parts", factor=2.0),
                                dict(scaling="parts", factor=2.0, original_positions=100, turns=(4.0, 4.0))])
def test_tables_refuse(kw):
    args = dict(n_pos=8, dim=8)
    args.update(kw)
    with pytest.raises(ValueError):
        rotary_tables(**args)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rotary(x, None, torch.zeros(4, 4), torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        causal_attention(x, x, x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        segment_bounds(torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="layout"):
        rotary(x, None, torch.zeros(4, 4), torch.zeros(4, 4), layout="other")
    with pytest.raises(KeyError):
        causal_attention(x, x, x, impl="other")


def test_cache_refuses():
    for kw in (dict(rows=0), dict(capacity=0), dict(kvheads=0), dict(k_dim=0), dict(v_dim=0), dict(store="int4")):
        args = dict(rows=1, capacity=4, kvheads=1, k_dim=8, device="cpu")
        args.update(kw)
        with pytest.raises(ValueError):
            init_kv_cache(**args)
    with pytest.raises(TypeError):
        init_kv_cache(1, 4, 1, 8, dtype=torch.float64, device="cpu")


def test_host_extension_checks_shapes_first():
    """Shapes are refused before any device is looked at, with Python's exceptions."""
    _lib._load_host()
    h = _lib._HOST
    q, k = torch.zeros(2, 4, 4, 8), torch.zeros(2, 4, 2, 8)
    t = torch.zeros(4, 4)
    for args in ((q[0], None, t, t), (q, k[:, :3], t, t), (q, k.half(), t, t), (q, k, t, t[:2]), (q, k, torch.zeros(4, 5), torch.zeros(4, 5))):
        with pytest.raises(ValueError):
            h.rotary(*args, None, False, False)
    for args in ((q[0], k, k), (q, k[:1], k[:1]), (q, k, k[:, :, :1]), (q[:, :, :3], k, k), (q, k.half(), k)):
        with pytest.raises(ValueError):
            h.causal_forward(*args, None, None, None, None, None, 0, False)
    with pytest.raises(ValueError, match="softcap"):
        h.causal_forward(q, k, k, None, None, None, -1.0, None, 0, False)
    for seq in (torch.zeros(2, 4), torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(ValueError):
            h.segment_bounds(seq)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        h.causal_forward(q, k, k, None, None, None, None, None, 0, False)


def test_layer_parameters():
    m = FullMultiHeadAttention(32, 8, 8, 4, 2, use_bias=True, use_sinks=True, use_gate=True)
    shapes = {n: tuple(p.shape) for n, p in m.named_parameters()}
    assert shapes == {"in_proj.weight": (64, 32), "in_proj.bias": (64,), "dense.weight": (32, 32), "dense.bias": (32,),
                      "sinks": (4,), "gate_proj.weight": (32, 32)}
    for kw in (dict(kvheads=3), dict(rope_dim=10), dict(rope_dim=3), dict(rope_layout="x")):
        args = dict(emb_dim=32, emb_kq=8, emb_v=8, nheads=4, kvheads=2)
        args.update(kw)
        with pytest.raises(ValueError):
            FullMultiHeadAttention(**args)


def test_a_cleared_cache_is_empty():
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            c = init_kv_cache(3, 4, 1, 8, device="cpu")
            c.lengths.fill_(2)
        c.max_length = 2
        c.clear()
        assert c.lengths.tolist() == [0, 0, 0] and c.max_length == 0
