"""Plain 64-bit forms of the full-attention operators, one row or head at a time,
and the roundings that the tests allow.

UNIT is twice the largest relative error of one rounding to the type: an output
that is rounded once is within UNIT of its value with room for the fp32 error
before it.
LEAST is the smallest step of the type: a result below its normal range (f16:
2^-14) is off by half of that however it was formed.
"""

import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -22}
LEAST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}


def rotate(x, cos, sin, positions, layout, inverse=False):
    """x [B, N, H, D] double; positions [B, N]; pairs as complex numbers."""
    R = 2 * cos.shape[1]
    c, s = cos.double()[positions][:, :, None], sin.double()[positions][:, :, None]
    s = -s if inverse else s
    y = x.double().clone()
    for i in range(R // 2):
        a, b = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + R // 2)
        xa, xb = x[..., a].double(), x[..., b].double()
        y[..., a] = xa * c[..., i] - xb * s[..., i]
        y[..., b] = xb * c[..., i] + xa * s[..., i]
    return y


def visible(seq_idx, B, N, device):
    """[B, N, N] bool: query i sees key j <= i with no other id between them."""
    out = torch.zeros(B, N, N, dtype=torch.bool)
    ids = torch.zeros(B, N, dtype=torch.long) if seq_idx is None else seq_idx.cpu().long()
    for b in range(B):
        start = 0
        for i in range(N):
            if i and ids[b, i] != ids[b, i - 1]:
                start = i
            if ids[b, i] >= 0:
                out[b, i, start: i + 1] = True
    return out.to(device)


def causal(q, k, v, see, softcap=None, scale=None):
    """(out, lse, largest |logit|) in double; autograd reaches q, k, v."""
    B, N, Hq, D = q.shape
    E = Hq // k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    k, v = k.repeat_interleave(E, 2), v.repeat_interleave(E, 2)
    x = torch.einsum("bnhd,bmhd->bhnm", q, k) * scale
    if softcap is not None:
        x = softcap * torch.tanh(x / softcap)
    top = float(x.detach().abs().max()) if x.numel() else 0.0
    see = see[:, None]
    x = torch.where(see, x, torch.full_like(x, -1e300))
    m = x.detach().amax(-1, keepdim=True)
    e = torch.where(see, torch.exp(x - m), torch.zeros_like(x))
    total = e.sum(-1, keepdim=True)
    empty = total == 0
    p = e / torch.where(empty, torch.ones_like(total), total)
    lse = torch.where(empty, torch.full_like(total, -math.inf), m + torch.log(torch.where(empty, torch.ones_like(total), total)))
    return torch.einsum("bhnm,bmhd->bnhd", p, v), lse[..., 0].permute(0, 2, 1), top, p


def quantise(x, store):
    """(codes, scales, values) of the rows of x in fp32, one IEEE operation at a
    time on the CPU; values in double."""
    x = x.detach().cpu().float()
    top = torch.full(x.shape[:-1], 127.0 if store == "int8" else 448.0)
    amax = x.abs().amax(-1)
    zero = amax < 1e-30
    inv = torch.where(zero, torch.zeros(()), top / amax)
    scale = torch.where(zero, torch.zeros(()), amax / top)
    y = x * inv[..., None]
    if store == "int8":
        codes = (y.round() + 128).to(torch.uint8)
        vals = codes.double() - 128
    else:
        e = y.to(torch.float8_e4m3fn)
        codes, vals = e.view(torch.uint8), e.double()
    return codes, scale, vals * scale[..., None].double()


def rel(got, want):
    n = float(want.double().norm())
    return float((got.double() - want.double()).norm()) / n if n else float(got.double().norm())


def gradient_terms(q, k, v, see, gout, glse, softcap=None, scale=None):
    """Norms of the sums of absolute terms behind dq, dk, dv: what fp32 and 16-bit
    roundings are relative to.  dS = P (dP - Delta) cancels (a token that sees
    itself alone has dP = Delta - dlse), its terms do not."""
    E = q.shape[2] // k.shape[2]
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    with torch.no_grad():
        q, k, v, gout = (t.double() for t in (q, k, v, gout))
        p = causal(q, k, v, see, softcap, scale)[3]
        dp = torch.einsum("bnhd,bmhd->bhnm", gout.abs(), v.abs().repeat_interleave(E, 2))
        delta = (p * dp).sum(-1, keepdim=True) + glse.double().abs().permute(0, 2, 1)[..., None]
        ds = p * (dp + delta) * scale
        dq = torch.einsum("bhnm,bmhd->bnhd", ds, k.abs().repeat_interleave(E, 2))
        dk = torch.einsum("bhnm,bnhd->bmhd", ds, q.abs())
        dv = torch.einsum("bhnm,bnhd->bmhd", p, gout.abs())
        return [float(t.norm()) for t in (dq, dk.unflatten(2, (-1, E)).sum(3), dv.unflatten(2, (-1, E)).sum(3))]
