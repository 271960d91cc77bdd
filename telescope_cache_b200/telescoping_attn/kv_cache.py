"""8-bit key / value cache of a full-attention layer: rows are quantised as they
are written and attended as codes, so a decode step reads a little over half
of a bf16 cache's bytes.

A token's key (or value) of one head is D codes and one fp32 scale.  'int8':
scale = amax / 127, code = round(x * (127 / amax)), kept with 128 added in a
byte; 'fp8': the same with 448 and an e4m3 float.  The codes are a function of
the values alone (IEEE quotient and product, round to nearest even): whichever
kernel writes a value, it writes the same code.
"""

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .. import _lib
from .rotary import LAYOUTS

STORES = {"int8": 0, "fp8": 1}


@dataclass
class KVCache:
    """One layer's cache: k [rows, Hkv, capacity, Dk] and v [..., Dv] codes
    (uint8), k_scale / v_scale [rows, Hkv, capacity] fp32, lengths [rows] int32
    tokens held, store 'int8' | 'fp8', dtype of the values read back.

    max_length is the host's upper bound of the lengths: it plans the split of
    the attention and refuses a write that may not fit; calls keep it current
    without reading the device.  Whoever sets `lengths` by hand sets it too."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    lengths: torch.Tensor
    store: str
    dtype: torch.dtype
    max_length: int = 0

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def clear(self) -> None:
        """Forget every row's tokens, and the bound with them: the cache for another batch."""
        with torch.inference_mode():  # the cache may have been made under it
            self.lengths.zero_()
        self.max_length = 0


def init_kv_cache(rows: int, capacity: int, kvheads: int, k_dim: int, v_dim: Optional[int] = None, *,
                  store: str = "int8", dtype: torch.dtype = torch.bfloat16, device=None) -> KVCache:
    """An empty cache of `rows` sequences of up to `capacity` tokens."""
    v_dim = k_dim if v_dim is None else v_dim
    if min(rows, capacity, kvheads, k_dim, v_dim) <= 0:
        raise ValueError("rows, capacity, kvheads and head dims must be positive")
    if store not in STORES:
        raise ValueError(f"store must be one of {tuple(STORES)}, got {store!r}")
    _lib.dtype_code(dtype)
    device = torch.device("cuda") if device is None else torch.device(device)
    zeros = lambda *s, t: torch.zeros(*s, device=device, dtype=t)  # noqa: E731
    return KVCache(k=zeros(rows, kvheads, capacity, k_dim, t=torch.uint8),
                   v=zeros(rows, kvheads, capacity, v_dim, t=torch.uint8),
                   k_scale=zeros(rows, kvheads, capacity, t=torch.float32),
                   v_scale=zeros(rows, kvheads, capacity, t=torch.float32),
                   lengths=zeros(rows, t=torch.int32), store=store, dtype=dtype)


def _parts(c: KVCache):
    """The cache as the host extension takes it."""
    store = STORES.get(c.store)
    if store is None:
        raise ValueError(f"store must be one of {tuple(STORES)}, got {c.store!r}")
    return c.k, c.v, c.k_scale, c.v_scale, c.lengths, store


def write_kv_cache(cache: KVCache, k: torch.Tensor, v: torch.Tensor, *,
                   seq_idx: Optional[torch.Tensor] = None, fresh: bool = False,
                   max_tokens: Optional[int] = None) -> None:
    """Quantise k [B, N, Hkv, Dk], v [B, N, Hkv, Dv] into the cache, behind the
    tokens that its rows hold, or (fresh=True) from slot 0 on in place of them.

    Without seq_idx, batch row b goes to cache row b.  With seq_idx [B, N]
    integers, token (b, n) goes to cache row seq_idx[b, n] (negative: nowhere):
    packed prompts and padded batches alike; a cache row's tokens are one run,
    in order, and rows that no token names keep what they hold (cache.clear()
    empties them all).  max_tokens: the most tokens that any row gets (by default N;
    for packed prompts, the longest).  Raises when a row may not fit; a token whose row or slot does not exist all the same is dropped and
    flagged in the device status word."""
    most = k.shape[1] if max_tokens is None else int(max_tokens)
    end = (0 if fresh else cache.max_length) + most
    if end > cache.capacity:
        raise ValueError(f"{end} tokens may not fit the cache's capacity of {cache.capacity}")
    _lib.host(k).kv_write(*_parts(cache), k, v, seq_idx, fresh)
    # rows that a fresh call does not name keep what they hold
    whole = fresh and seq_idx is None and k.shape[0] == cache.k.shape[0]
    cache.max_length = most if whole else max(cache.max_length, end)


def read_kv_cache(cache: KVCache, length: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k [rows, length, Hkv, Dk], v [..., Dv]) that the codes of the first
    `length` (default max_length) slots stand for, in cache.dtype; zeros past a
    row's own length."""
    length = cache.max_length if length is None else int(length)
    return _lib.host(cache.k).kv_read(*_parts(cache), length, cache.dtype)


def cached_attention(q_t: torch.Tensor, cache: KVCache, *, softcap: Optional[float] = None,
                     scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [B, 1, Hq, Dv], lse [B, 1, Hq] fp32) of one query per sequence,
    q_t [B, 1, Hq, Dk] (already rotated), over the tokens that rows 0 .. B - 1 of
    the cache hold; an empty row gives out 0 and lse -inf.  For serving: the results
    have no gradients."""
    out, lse, _, _ = _lib.host(q_t).kv_attend(*_parts(cache), cache.dtype, cache.max_length, q_t, None, None, None, None,
                                              False, softcap, scale, False, False)
    return out, lse


def cached_attention_step(q_t: torch.Tensor, k_t: torch.Tensor, v_t: torch.Tensor, cache: KVCache, *,
                          rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                          layout: str = "half", softcap: Optional[float] = None, scale: Optional[float] = None,
                          advance: bool = True, return_stored: bool = False):
    """One token of every sequence in one launch: rotate q_t [B, 1, Hq, Dk] and
    k_t [B, 1, Hkv, Dk] to position lengths[b] (with tables, as rotary does),
    quantise the key and v_t [B, 1, Hkv, Dv] into slot lengths[b], attend over
    lengths[b] + 1 tokens, and move the lengths on (advance=False: the token is
    tried at its place and the next call writes there again).

    Returns (out [B, 1, Hq, Dv], lse [B, 1, Hq] fp32), and with return_stored
    the key and value that the written codes stand for, [B, 1, Hkv, D].  The results
    have no gradients."""
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if k_t is None or v_t is None:
        raise ValueError("a step needs the token's key and value")
    r = _lib.host(q_t).kv_attend(*_parts(cache), cache.dtype, cache.max_length, q_t, k_t, v_t, rope_cos, rope_sin,
                                 layout == "interleaved", softcap, scale, advance, return_stored)
    if advance:
        cache.max_length += 1
    return r if return_stored else r[:2]


__all__ = ["KVCache", "init_kv_cache", "write_kv_cache", "read_kv_cache", "cached_attention", "cached_attention_step"]
