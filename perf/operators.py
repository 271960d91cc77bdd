"""What is measured of the full-attention operators: rotary positions, causal attention over packed sequences, and the
8-bit key / value cache with the attention that reads it.

Sizes are those of this repository's configurations (16 or 32 heads of 128, 8192 to 131072 tokens, batches of 64 at
decode, the 4-head fp32 shape of 1024 x 64) or generic ones around them; no case stands for a particular model.

    rotary   q, k -> rotated q, k (and, in training, their gradients); one pass over the data
    causal   (out, lse) of causal attention with grouped heads over packed examples (and, in training, dq, dk, dv)
    write    a prompt's keys and values quantised into the cache as they are written, and read back
    step     one token of every sequence: rotate, quantise and write its key and value, attend over the cache
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the token's q and k of 64 sequences at decode: latency alone counts
        dict(name="rotary token", op="rotary", B=64, N=1, Hq=16, Hkv=16, D=128, R=128, layout="half", dtype="bf16",
             grad=False, packed=False),
        # a training step's q and k, views of the fused projection, half of each head rotated, positions restarting
        # at every packed example; with the gradients: bandwidth alone counts
        dict(name="rotary train", op="rotary", B=4, N=16384, Hq=16, Hkv=4, D=128, R=64, layout="interleaved",
             dtype="f16", grad=True, packed=True),
        # a batch of short prompts of an odd length
        dict(name="causal short", op="causal", B=4, N=197, Hq=8, Hkv=2, D=64, dtype="f16", grad=False, examples=1,
             pad=0, softcap=0.0),
        # prefill of packed prompts of very different lengths with a padded tail
        dict(name="causal prompt", op="causal", B=2, N=8192, Hq=16, Hkv=4, D=128, dtype="bf16", grad=False,
             examples=7, pad=100, softcap=0.0),
        # a training step over packed documents with the softcap of the training configuration
        dict(name="causal train", op="causal", B=2, N=4096, Hq=16, Hkv=16, D=128, dtype="bf16", grad=True, examples=5,
             pad=0, softcap=50.0),
        # a training step over one long document
        dict(name="causal train long", op="causal", B=1, N=16384, Hq=8, Hkv=2, D=128, dtype="bf16", grad=True,
             examples=1, pad=0, softcap=0.0),
        # the fp32 parity shape (4 heads of 64, 1024 tokens)
        dict(name="causal train f32", op="causal", B=1, N=1024, Hq=4, Hkv=4, D=64, dtype="f32", grad=True, examples=1,
             pad=0, softcap=0.0),
        # hand-off of a batch of prompts of different lengths into the cache
        dict(name="cache write", op="write", B=4, N=16384, Hkv=16, D=128, dtype="bf16", store="int8", ragged=True),
        # a batch of short prompts of an odd length and small heads
        dict(name="cache write short", op="write", B=64, N=77, Hkv=4, D=64, dtype="f16", store="fp8", ragged=False),
        # one sequence, a short cache: latency alone counts
        dict(name="step small", op="step", B=1, L=1024, Hq=16, Hkv=16, D=128, dtype="bf16", store="int8",
             layout="half", softcap=0.0, ragged=False),
        # serving: 64 sequences of different lengths up to 32768, four query heads to a key head
        dict(name="step batch", op="step", B=64, L=32768, Hq=16, Hkv=4, D=128, dtype="bf16", store="int8",
             layout="half", softcap=0.0, ragged=True),
        # one sequence with a long cache in 8-bit floating point
        dict(name="step long", op="step", B=1, L=131072, Hq=32, Hkv=8, D=128, dtype="bf16", store="fp8",
             layout="interleaved", softcap=50.0, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "causal", "causal", "write", "step", "step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    E = rng.choice([1, 2, 4, 8])
    if op == "rotary":
        N = _log(rng, 1, 32768)
        return dict(op=op, B=max(1, min(64, _log(rng, 1, 131072) // N)), N=N, Hq=Hkv * E, Hkv=Hkv, D=D,
                    R=rng.choice([D, D, D // 2, 24]), layout=rng.choice(["half", "interleaved"]), dtype=dtype,
                    grad=rng.random() < 0.5, packed=rng.random() < 0.5)
    if op == "causal":
        N = _log(rng, 1, 2048 if dtype == "f32" else 8192)
        B = max(1, min(4, 8192 // N))
        while B * Hkv * E * N * N > 2 ** 31:
            E, Hkv = (E // 2, Hkv) if E > 1 else (1, Hkv // 2)
        return dict(op=op, B=B, N=N, Hq=Hkv * E, Hkv=Hkv, D=D, dtype=dtype, grad=rng.random() < 0.5,
                    examples=min(N, rng.choice([1, 2, 5, 13])), pad=rng.choice([0, 0, N // 7]),
                    softcap=rng.choice([0.0, 0.0, 30.0, 50.0]))
    store = rng.choice(["int8", "fp8"])
    if op == "write":
        N = _log(rng, 1, 16384)
        return dict(op=op, B=max(1, min(64, _log(rng, 1, 65536) // N)), N=N, Hkv=Hkv, D=D, dtype=dtype, store=store,
                    ragged=rng.random() < 0.5)
    L = _log(rng, 1, 65536)
    B = max(1, min(64, _log(rng, 64, 262144) // L))
    return dict(op=op, B=B, L=L, Hq=Hkv * E, Hkv=Hkv, D=D, dtype=dtype, store=store,
                layout=rng.choice(["half", "interleaved"]), softcap=rng.choice([0.0, 0.0, 50.0]),
                ragged=rng.random() < 0.5)


# --------------------------------------------------------------------------------------------------------- inputs
def _ids(case, examples, pad):
    """[B, N] example ids of packed rows (the same cuts for every seed), -1 in the padded tail."""
    B, N = case["B"], case["N"]
    g = torch.Generator().manual_seed(1000 * examples + N)
    order = torch.rand(B, max(N - 1, 1), generator=g).argsort(1)[:, : examples - 1] + 1
    cuts = order.sort(1).values
    ids = torch.searchsorted(cuts.contiguous(), torch.arange(N).expand(B, N).contiguous(), right=True)
    return torch.where(torch.arange(N) < N - pad, ids, -1).to(torch.int32)


def _starts(ids):
    """[B, N] first token of each token's run of equal ids."""
    at = torch.arange(ids.shape[1], device=ids.device).expand_as(ids)
    new = torch.ones_like(ids, dtype=torch.bool)
    new[:, 1:] = ids[:, 1:] != ids[:, :-1]
    return torch.where(new, at, 0).cummax(1).values


def _lengths(case):
    """Tokens of every cache row, the same for every seed: all of them, or spread evenly over [1, all]."""
    most = case["N"] if case["op"] == "write" else case["L"]
    if not case["ragged"]:
        return torch.full((case["B"],), most, dtype=torch.int32)
    g = torch.Generator().manual_seed(7 * case["B"] + most)
    n = 1 + (torch.rand(case["B"], generator=g) * most).long()
    n[0] = most
    return n.clamp(max=most).to(torch.int32)


def _tables(n_pos, dim):
    """cos, sin [n_pos, dim / 2] of positions scaled down by 4 above the 8192 that the frequencies were made for."""
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv / (4.0 if n_pos > 8192 else 1.0)
    return ang.cos().float(), ang.sin().float()


def _quantise(x, store):
    """Codes (uint8) and one scale per row of x [..., D]: 8-bit integers kept with 128 added, or e4m3 floats."""
    top = 127.0 if store == "int8" else 448.0
    x = x.float()
    amax = x.abs().amax(-1)
    tiny = amax < 1e-30
    top = torch.full_like(amax, top)  # a tensor: a scalar's quotient would be a product with a rounded reciprocal
    inv = torch.where(tiny, torch.zeros_like(amax), top / amax)
    y = x * inv[..., None]
    if store == "int8":
        codes = (y.round() + 128.0).to(torch.uint8)
    else:
        codes = y.to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, torch.where(tiny, torch.zeros_like(amax), amax / top)


def _values(codes, store):
    return codes.float() - 128.0 if store == "int8" else codes.view(torch.float8_e4m3fn).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    s = dict(case=case)
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    if case["op"] == "rotary":
        N, Hq = case["N"], case["Hq"]
        s["cos"], s["sin"] = _tables(N, case["R"])
        q, k, _ = normal(B, N, (Hq + 2 * Hkv) * D).split([Hq * D, Hkv * D, Hkv * D], -1)
        s["q"], s["k"] = q.view(B, N, Hq, D), k.view(B, N, Hkv, D)
        s["positions"] = None
        if case["packed"]:
            ids = _ids(case, min(N, 6), 0).cuda()
            s["positions"] = (torch.arange(N, device="cuda") - _starts(ids)).to(torch.int32)
        if case["grad"]:
            s["gq"], s["gk"] = normal(B, N, Hq, D), normal(B, N, Hkv, D)
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
    elif case["op"] == "causal":
        N, Hq = case["N"], case["Hq"]
        q, k, v = normal(B, N, (Hq + 2 * Hkv) * D).split([Hq * D, Hkv * D, Hkv * D], -1)
        s["q"], s["k"], s["v"] = q.view(B, N, Hq, D), k.view(B, N, Hkv, D), v.view(B, N, Hkv, D)
        packed = case["examples"] > 1 or case["pad"] > 0
        s["seq_idx"] = _ids(case, case["examples"], case["pad"]).cuda() if packed else None
        if case["grad"]:
            s["gout"] = normal(B, N, Hq, D)
            s["glse"] = torch.randn(B, N, Hq, generator=g, device="cuda")
            for name in ("q", "k", "v"):
                s[name] = s[name].detach().requires_grad_()
    elif case["op"] == "write":
        N = case["N"]
        s["k"], s["v"] = normal(B, N, Hkv, D), normal(B, N, Hkv, D)
        lengths = _lengths(case).cuda()
        rows = torch.arange(B, device="cuda", dtype=torch.int32)[:, None].expand(B, N)
        s["seq_idx"] = torch.where(torch.arange(N, device="cuda") < lengths[:, None], rows, -1)
        s["codes"] = [torch.zeros(B, Hkv, N, D, device="cuda", dtype=torch.uint8) for _ in range(2)]
        s["scales"] = [torch.zeros(B, Hkv, N, device="cuda") for _ in range(2)]
        s["lengths"] = torch.zeros(B, device="cuda", dtype=torch.int32)
    else:
        L, Hq = case["L"], case["Hq"]
        s["cos"], s["sin"] = _tables(L + 1, D)
        s["q"], s["k"], s["v"] = normal(B, 1, Hq, D), normal(B, 1, Hkv, D), normal(B, 1, Hkv, D)
        s["codes"], s["scales"] = [], []
        for _ in range(2):
            codes = torch.empty(B, Hkv, L + 1, D, device="cuda", dtype=torch.uint8)
            scales = torch.empty(B, Hkv, L + 1, device="cuda")
            for b in range(B):  # a sequence at a time: a few buffers of one sequence instead of the whole batch's
                codes[b], scales[b] = _quantise(normal(Hkv, L + 1, D), case["store"])
            s["codes"].append(codes)
            s["scales"].append(scales)
        s["lengths"] = _lengths(case).cuda()
    return s


# ------------------------------------------------------------------------------------------------------ the passes
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _cache(s):
    from telescope_cache_b200 import KVCache

    c = s["case"]
    return KVCache(k=s["codes"][0], v=s["codes"][1], k_scale=s["scales"][0], v_scale=s["scales"][1],
                   lengths=s["lengths"], store=c["store"], dtype=DTYPES[c["dtype"]],
                   max_length=0 if c["op"] == "write" else c["L"])


def _own_rotary(s):
    from telescope_cache_b200 import rotary

    q, k = rotary(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], layout=s["case"]["layout"])
    if not s["case"]["grad"]:
        return dict(q=q, k=k)
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
    return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk)


def _own_causal(s):
    from telescope_cache_b200 import causal_attention

    out, lse = causal_attention(s["q"], s["k"], s["v"], seq_idx=s["seq_idx"], softcap=s["case"]["softcap"] or None)
    if not s["case"]["grad"]:
        return dict(out=out, lse=lse)
    dq, dk, dv = torch.autograd.grad((out, lse), (s["q"], s["k"], s["v"]), (s["gout"], s["glse"]))
    return dict(out=out.detach(), lse=lse.detach(), dq=dq, dk=dk, dv=dv)


def _own_write(s):
    from telescope_cache_b200 import read_kv_cache, write_kv_cache

    cache = _cache(s)
    write_kv_cache(cache, s["k"], s["v"], seq_idx=s["seq_idx"], fresh=True)
    k, v = read_kv_cache(cache)
    return dict(k=k, v=v, lengths=cache.lengths)


def _own_step(s):
    from telescope_cache_b200 import cached_attention_step

    # advance=False: the token is tried at its place and the sequence keeps its length, so every pass is the same
    out, lse, k_new, v_new = cached_attention_step(
        s["q"], s["k"], s["v"], _cache(s), rope_cos=s["cos"], rope_sin=s["sin"], layout=s["case"]["layout"],
        softcap=s["case"]["softcap"] or None, advance=False, return_stored=True)
    return dict(out=out, lse=lse, k_new=k_new, v_new=v_new)


def _rotate(x, c, s, layout):
    """x [..., D] in 32 bits rotated by tables c, s [..., R / 2] that broadcast against it; dims from R on stay."""
    R = 2 * c.shape[-1]
    y = x.clone()
    if layout == "half":
        x1, x2 = x[..., : R // 2], x[..., R // 2: R]
        y[..., : R // 2], y[..., R // 2: R] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x[..., 0:R:2], x[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


@torch.no_grad()
def _plain_rotary(s):
    case = s["case"]
    c, n = s["cos"], s["sin"]
    if s["positions"] is not None:
        c, n = c[s["positions"].long()], n[s["positions"].long()]
    c, n = c[..., None, :], n[..., None, :]
    dt = s["q"].dtype
    r = dict(q=_rotate(s["q"].float(), c, n, case["layout"]).to(dt), k=_rotate(s["k"].float(), c, n, case["layout"]).to(dt))
    if case["grad"]:
        r["dq"] = _rotate(s["gq"].float(), c, -n, case["layout"]).to(dt)
        r["dk"] = _rotate(s["gk"].float(), c, -n, case["layout"]).to(dt)
    return r


@torch.no_grad()
def _plain_causal(s):
    case = s["case"]
    B, N, Hq, D = s["q"].shape
    Hkv, dt, cap, scale = case["Hkv"], s["q"].dtype, case["softcap"], 1.0 / math.sqrt(D)
    q = s["q"].float().view(B, N, Hkv, Hq // Hkv, D)
    k, v = s["k"].float(), s["v"].float()
    at = torch.arange(N, device=q.device)
    see = (at[None, :] <= at[:, None])[None]
    if s["seq_idx"] is not None:
        i = s["seq_idx"]
        see = see & (i[:, :, None] == i[:, None, :]) & (i >= 0)[:, :, None]
    see = see[:, None, None]  # [B or 1, 1, 1, N, N]
    x = torch.einsum("bnhed,bmhd->bhenm", q, k).mul_(scale)
    t = None
    if cap:
        t = x.div_(cap).tanh_()
        x = t * cap
    x = x.masked_fill(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m.isfinite(), m, 0.0)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).squeeze(-1)  # [B, Hkv, E, N]; -inf where a row sees nothing
    p.div_(torch.where(total > 0, total, 1.0))
    out = torch.einsum("bhenm,bmhd->bnhed", p, v)
    r = dict(out=out.reshape(B, N, Hq, D).to(dt), lse=lse.permute(0, 3, 1, 2).reshape(B, N, Hq))
    if not case["grad"]:
        return r
    g = s["gout"].float().view(B, N, Hkv, Hq // Hkv, D)
    delta = (g * out).sum(-1) - s["glse"].view(B, N, Hkv, Hq // Hkv)
    r["dv"] = torch.einsum("bhenm,bnhed->bmhd", p, g).to(dt)
    ds = torch.einsum("bnhed,bmhd->bhenm", g, v).sub_(delta.permute(0, 2, 3, 1)[..., None]).mul_(p).mul_(scale)
    if cap:
        ds.mul_(t.square_().neg_().add_(1.0))
    r["dq"] = torch.einsum("bhenm,bmhd->bnhed", ds, k).reshape(B, N, Hq, D).to(dt)
    r["dk"] = torch.einsum("bhenm,bnhed->bmhd", ds, q).to(dt)
    return r


@torch.no_grad()
def _plain_write(s):
    case = s["case"]
    live = s["seq_idx"] >= 0  # row b's own tokens, from its first slot on
    r = {}
    for i, name in enumerate(("k", "v")):
        codes, scales = _quantise(s[name].transpose(1, 2), case["store"])
        s["codes"][i].copy_(torch.where(live[:, None, :, None], codes, s["codes"][i]))
        s["scales"][i].copy_(torch.where(live[:, None, :], scales, s["scales"][i]))
        back = _values(s["codes"][i], case["store"]) * s["scales"][i][..., None]
        back = torch.where(live[:, None, :, None], back, 0.0)
        r[name] = back.transpose(1, 2).to(s[name].dtype)
    s["lengths"].copy_(live.sum(1))
    r["lengths"] = s["lengths"]
    return r


@torch.no_grad()
def _plain_step(s):
    case = s["case"]
    B, _, Hq, D = s["q"].shape
    Hkv, L, cap, dt = case["Hkv"], case["L"], case["softcap"], s["q"].dtype
    at = s["lengths"].long()
    c, n = s["cos"][at][:, None, None], s["sin"][at][:, None, None]
    q = _rotate(s["q"].float(), c, n, case["layout"]).view(B, Hkv, Hq // Hkv, D)
    new = (_rotate(s["k"].float(), c, n, case["layout"]), s["v"].float())
    row = torch.arange(B, device=q.device)
    r, kv = {}, []
    for i, name in enumerate(("k_new", "v_new")):
        codes, scales = _quantise(new[i][:, 0], case["store"])
        s["codes"][i][row, :, at], s["scales"][i][row, :, at] = codes, scales
        r[name] = (_values(codes, case["store"]) * scales[..., None])[:, None].to(dt)
        kv.append(_values(s["codes"][i], case["store"]).mul_(s["scales"][i][..., None]))
    x = torch.einsum("bhed,bhmd->bhem", q, kv[0]) / math.sqrt(D)
    if cap:
        x = (x / cap).tanh() * cap
    x = x.masked_fill(torch.arange(L + 1, device=q.device) > at[:, None, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = (x - m).exp()
    total = p.sum(-1, keepdim=True)
    r["lse"] = (m + total.log()).reshape(B, 1, Hq)
    r["out"] = torch.einsum("bhem,bhmd->bhed", p / total, kv[1]).reshape(B, 1, Hq, D).to(dt)
    return r


_own = dict(rotary=_own_rotary, causal=_own_causal, write=_own_write, step=_own_step)
_plain = dict(rotary=_plain_rotary, causal=_plain_causal, write=_plain_write, step=_plain_step)


# ---------------------------------------------------------------------------------------------------------- floors
def work(case):
    """Each input read once and each output written once; products as multiply and add."""
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        n = B * case["N"] * (case["Hq"] + Hkv) * D * (2 if case["grad"] else 1)
        return {"bytes": 2 * n * e + 2 * 4 * case["N"] * (case["R"] // 2), "flops": 3 * n * case["R"] // D}
    if case["op"] == "causal":
        N, Hq = case["N"], case["Hq"]
        ids = _ids(case, case["examples"], case["pad"])
        seen = torch.where(ids >= 0, torch.arange(N) - _starts(ids) + 1, 0)
        pairs = int(seen.sum()) * Hq
        q, kv = B * N * Hq, B * N * Hkv
        if not case["grad"]:
            return {"bytes": e * D * (2 * q + 2 * kv) + 4 * q, "flops": 4 * D * pairs}
        return {"bytes": e * D * (4 * q + 4 * kv) + 8 * q, "flops": 14 * D * pairs}
    tokens = int(_lengths(case).sum())
    if case["op"] == "write":
        # read the values, write codes and scales, read them, write the values they stand for (zeros past the end)
        return {"bytes": 2 * Hkv * (tokens * (e * D + 2 * (D + 4)) + B * case["N"] * e * D), "flops": 8 * tokens * Hkv * D}
    Hq = case["Hq"]
    return {"bytes": 2 * Hkv * tokens * (D + 4) + B * (2 * Hq + 4 * Hkv) * D * e + 4 * B * Hq,
            "flops": 4 * D * Hq * (tokens + B)}


# ------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return dict(rotary=_exact_rotary, causal=_exact_causal, write=_exact_write, step=_exact_step)[case["op"]](case, s)


def _turn(x, ang_cos, ang_sin, layout, sign=1.0):
    """Each pair as a complex number times cos + i sin."""
    x = x.detach().double()
    R = 2 * ang_cos.shape[-1]
    w = torch.complex(ang_cos.double(), sign * ang_sin.double())
    part = x[..., :R]
    pairs = part.unflatten(-1, (2, R // 2)).transpose(-1, -2) if layout == "half" else part.unflatten(-1, (R // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
    z = z.transpose(-1, -2).flatten(-2) if layout == "half" else z.flatten(-2)
    return torch.cat([z, x[..., R:]], -1)


def _exact_rotary(case, s):
    B, N = case["B"], case["N"]
    pos = torch.arange(N, device="cuda").expand(B, N) if s["positions"] is None else s["positions"].long()
    c, n = s["cos"][pos].unsqueeze(2), s["sin"][pos].unsqueeze(2)
    r = {name: _turn(s[name], c, n, case["layout"]) for name in ("q", "k")}
    if case["grad"]:
        r |= {"d" + name: _turn(s["g" + name], c, n, case["layout"], -1.0) for name in ("q", "k")}
    return r


def _exact_causal(case, s):
    """One (sequence, query head) at a time; a query sees the tokens of its own example up to itself."""
    B, N, Hq, D = s["q"].shape
    E, cap, scale = Hq // case["Hkv"], case["softcap"], D ** -0.5
    q, k, v = (s[name].detach().double() for name in ("q", "k", "v"))
    r = dict(out=torch.zeros_like(q), lse=torch.empty(B, N, Hq, device="cuda", dtype=torch.float64))
    if case["grad"]:
        r |= dict(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    lower = torch.ones(N, N, device="cuda", dtype=torch.bool).tril()
    for b in range(B):
        see = lower
        if s["seq_idx"] is not None:
            i = s["seq_idx"][b]
            see = lower & (i[None] == i[:, None]) & (i[:, None] >= 0)
        some = see.any(1)
        for h in range(Hq):
            y = q[b, :, h] @ k[b, :, h // E].T * scale
            slope = None
            if cap:
                y = torch.tanh(y / cap)
                slope = 1 - y * y
                y = y * cap
            y = torch.where(see, y, -math.inf)
            lse = torch.logsumexp(y, 1)
            w = torch.where(some[:, None], torch.exp(y - lse[:, None]), 0.0)
            w = torch.where(see, w, 0.0)
            r["out"][b, :, h], r["lse"][b, :, h] = w @ v[b, :, h // E], lse
            if case["grad"]:
                g = s["gout"][b, :, h].double()
                r["dv"][b, :, h // E] += w.T @ g
                y = g @ v[b, :, h // E].T
                # d loss / d logit = w (g . v - sum_j w_j g . v_j + glse)
                y = w * (y - (w * y).sum(1, keepdim=True) + s["glse"][b, :, h, None].double())
                y = y * scale if slope is None else y * slope * scale
                r["dq"][b, :, h] = y @ k[b, :, h // E]
                r["dk"][b, :, h // E] += y.T @ q[b, :, h]
            del y, w, slope
    return r


def _stored(x, store):
    """The values that the cache's codes of x [..., D] stand for, in 64 bits but for the held scale's 32."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    if store == "int8":
        held = (amax / 127).float().double()
        return torch.where(amax < 1e-30, 0.0, (x * 127 / amax).round() * held)
    held = (amax / 448).float().double()
    y = x * 448 / amax
    # e4m3: three bits behind the leading one, none below 2^-9
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(amax < 1e-30, 0.0, ((y / step).round() * step).clamp(-448, 448) * held)


def _exact_write(case, s):
    lengths = _lengths(case).cuda()
    live = (torch.arange(case["N"], device="cuda") < lengths[:, None])[..., None, None]
    return {name: torch.where(live, _stored(s[name], case["store"]), 0.0) for name in ("k", "v")} | dict(lengths=lengths)


def _exact_step(case, s):
    B, _, Hq, D = s["q"].shape
    E, cap = Hq // case["Hkv"], case["softcap"]
    r = dict(out=torch.empty(B, 1, Hq, D, device="cuda", dtype=torch.float64),
             lse=torch.empty(B, 1, Hq, device="cuda", dtype=torch.float64))
    k_new, v_new = [], []
    for b in range(B):
        at = int(s["lengths"][b])
        q = _turn(s["q"][b, 0], s["cos"][at], s["sin"][at], case["layout"])
        new = (_stored(_turn(s["k"][b, 0], s["cos"][at], s["sin"][at], case["layout"]), case["store"]),
               _stored(s["v"][b, 0], case["store"]))
        k_new.append(new[0][None])
        v_new.append(new[1][None])
        k, v = (torch.cat([_values(s["codes"][i][b, :, :at], case["store"]).double()
                           * s["scales"][i][b, :, :at, None].double(), new[i][:, None]], 1).repeat_interleave(E, 0)
                for i in range(2))
        y = (k @ q[:, :, None])[..., 0] / math.sqrt(D)  # [Hq, at + 1]
        y = cap * torch.tanh(y / cap) if cap else y
        r["lse"][b, 0] = torch.logsumexp(y, -1)
        r["out"][b, 0] = (torch.softmax(y, -1)[:, None] @ v)[:, 0]
    return r | dict(k_new=torch.stack(k_new), v_new=torch.stack(v_new))
