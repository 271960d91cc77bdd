"""8-bit key / value cache of a full-attention layer: rows are quantised as they
are written and attended as codes, so a decode step reads a little over half
of a bf16 cache's bytes.

A token's key (or value) of one head is D codes and one fp32 scale.  'int8':
scale = amax / 127, code = round(x * (127 / amax)), kept with 128 added in a
byte; 'fp8': the same with 448 and an e4m3 float.  The codes are a function of
the values alone (IEEE quotient and product, round to nearest even): whichever
kernel writes a value, it writes the same code.
"""

import ctypes
import math
from dataclasses import dataclass
from typing import Dict, Optional, Tuple, Union

import torch

from .. import _lib
from .attention import device_status
from .causal import Segments, segment_bounds
from .rotary import LAYOUTS, _table

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


def _cache_args(c: KVCache):
    k, v = c.k, c.v
    if k.dim() != 4 or v.dim() != 4 or k.shape[:3] != v.shape[:3]:
        raise ValueError(f"cache k {tuple(k.shape)} and v {tuple(v.shape)} must be [rows, Hkv, capacity, D]")
    if k.dtype != torch.uint8 or v.dtype != torch.uint8 or c.k_scale.dtype != torch.float32 or \
            c.v_scale.dtype != torch.float32 or c.lengths.dtype != torch.int32:
        raise ValueError("cache codes must be uint8, scales float32 and lengths int32")
    if c.k_scale.shape != k.shape[:3] or c.v_scale.shape != k.shape[:3] or c.lengths.shape != k.shape[:1]:
        raise ValueError("cache scales must be [rows, Hkv, capacity] and lengths [rows]")
    if not (k.is_contiguous() and v.is_contiguous() and c.k_scale.is_contiguous() and c.v_scale.is_contiguous()
            and c.lengths.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    store = STORES.get(c.store)
    if store is None:
        raise ValueError(f"store must be one of {tuple(STORES)}, got {c.store!r}")
    _lib.require_cuda(k, v, c.k_scale, c.v_scale, c.lengths)
    return _lib.KVCacheArgs(rows=k.shape[0], Hkv=k.shape[1], Dk=k.shape[3], Dv=v.shape[3], capacity=k.shape[2],
                            store=store, k=k.data_ptr(), v=v.data_ptr(), k_scale=c.k_scale.data_ptr(),
                            v_scale=c.v_scale.data_ptr(), lengths=c.lengths.data_ptr())


def _dense_head(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


@torch.no_grad()
def write_kv_cache(cache: KVCache, k: torch.Tensor, v: torch.Tensor, *,
                   seq_idx: Union[torch.Tensor, None] = None, fresh: bool = False,
                   max_tokens: Optional[int] = None) -> None:
    """Quantise k [B, N, Hkv, Dk], v [B, N, Hkv, Dv] into the cache, behind the
    tokens that its rows hold, or (fresh=True) from slot 0 on in place of them.

    Without seq_idx, batch row b goes to cache row b.  With seq_idx [B, N]
    integers, token (b, n) goes to cache row seq_idx[b, n] (negative: nowhere):
    packed prompts and padded batches alike; a cache row's tokens are one run,
    in order, and rows that no token names keep what they hold.  max_tokens:
    the most tokens that any row gets (by default N).  Raises when a row may not
    fit; a token whose row or slot does not exist all the same is dropped and
    flagged in the device status word."""
    c = _cache_args(cache)
    if k.dim() != 4 or v.dim() != 4 or k.shape[:3] != v.shape[:3] or k.dtype != v.dtype:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} do not go together")
    B, N = k.shape[:2]
    if (k.shape[2], k.shape[3], v.shape[3]) != (c.Hkv, c.Dk, c.Dv):
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} do not fit the cache's {c.Hkv} heads of {c.Dk}, {c.Dv}")
    if seq_idx is None and B > c.rows:
        raise ValueError(f"batch of {B} into a cache of {c.rows} rows")
    most = N if max_tokens is None else int(max_tokens)
    end = (0 if fresh else cache.max_length) + most
    if end > c.capacity:
        raise ValueError(f"{end} tokens may not fit the cache's capacity of {c.capacity}")
    _lib.require_cuda(k, v, seq_idx)
    k, v = _dense_head(k), _dense_head(v)
    a = _lib.KVWriteArgs(B=B, N=N, dtype=_lib.dtype_code(k.dtype), fresh=bool(fresh),
                         k=k.data_ptr(), k_stride_b=k.stride(0), k_stride_n=k.stride(1), k_stride_h=k.stride(2),
                         v=v.data_ptr(), v_stride_b=v.stride(0), v_stride_n=v.stride(1), v_stride_h=v.stride(2),
                         dev_status=device_status(k.device).data_ptr())
    seg = ids = None
    if seq_idx is not None:
        if tuple(seq_idx.shape) != (B, N) or seq_idx.dtype.is_floating_point:
            raise ValueError(f"seq_idx must be an integer tensor [{B}, {N}], got {tuple(seq_idx.shape)}")
        ids = seq_idx.to(torch.int32).contiguous()
        seg = segment_bounds(ids)
        a.seq_idx, a.starts = ids.data_ptr(), seg.starts.data_ptr()
    _lib.launch("tc_kv_write", k.device, c, a, _lib.stream_of(k))
    # fresh rows hold at most `most`; rows that the call does not name keep theirs
    cache.max_length = most if fresh and seq_idx is None and B == c.rows else max(cache.max_length, end)


@torch.no_grad()
def read_kv_cache(cache: KVCache, length: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k [rows, length, Hkv, Dk], v [..., Dv]) that the codes of the first
    `length` (default max_length) slots stand for, in cache.dtype; zeros past a
    row's own length."""
    c = _cache_args(cache)
    length = cache.max_length if length is None else int(length)
    if not 0 <= length <= c.capacity:
        raise ValueError(f"length {length} outside [0, {c.capacity}]")
    dev = cache.k.device
    k = torch.empty(c.rows, length, c.Hkv, c.Dk, device=dev, dtype=cache.dtype)
    v = torch.empty(c.rows, length, c.Hkv, c.Dv, device=dev, dtype=cache.dtype)
    if length:
        _lib.launch("tc_kv_read", dev, c, length, _lib.dtype_code(cache.dtype), k.data_ptr(), v.data_ptr(),
                    _lib.stream_of(cache.k))
    return k, v


# Workspace of the split attention: one per device and stream, since calls on one
# stream run in order.  The arrival counts are zero between calls.
_WORK: Dict[tuple, list] = {}


def _workspace(device, stream: int, floats: int, counts: int):
    key = (device.index, stream)
    w = _WORK.get(key)
    if w is None:
        w = _WORK[key] = [None, None]
    if floats and (w[0] is None or w[0].numel() < floats):
        w[0] = torch.empty(floats, device=device, dtype=torch.float32)
    if w[1] is None or w[1].numel() < counts:
        w[1] = torch.zeros(max(counts, 4096), device=device, dtype=torch.int32)
    return w


def _attend(cache, q_t, k_t, v_t, cos, sin, layout, softcap, scale, advance, stored):
    c = _cache_args(cache)
    if q_t.dim() != 4 or q_t.shape[1] != 1:
        raise ValueError(f"q_t must be [B, 1, Hq, Dk], got {tuple(q_t.shape)}")
    B, _, Hq, Dk = q_t.shape
    if Dk != c.Dk or B > c.rows:
        raise ValueError(f"q_t {tuple(q_t.shape)} incompatible with the cache's {c.rows} rows, {c.Hkv} heads of {c.Dk}")
    if Hq % c.Hkv != 0:
        raise ValueError(f"Hq={Hq} must be divisible by Hkv={c.Hkv}.")
    if softcap is not None and not softcap > 0:
        raise ValueError(f"softcap must be positive, got {softcap}")
    _lib.require_cuda(q_t, k_t, v_t, cos, sin)
    dev = q_t.device
    q_t = _dense_head(q_t)
    out = torch.empty(B, 1, Hq, c.Dv, device=dev, dtype=q_t.dtype)
    lse = torch.empty(B, 1, Hq, device=dev, dtype=torch.float32)
    most = min(cache.max_length + (1 if k_t is not None else 0), c.capacity)
    a = _lib.KVAttendArgs(B=B, Hq=Hq, max_tokens=most, dtype=_lib.dtype_code(q_t.dtype), q=q_t.data_ptr(),
                          q_stride_b=q_t.stride(0), q_stride_h=q_t.stride(2), has_softcap=softcap is not None,
                          softcap=1.0 if softcap is None else softcap,
                          scale=1.0 / math.sqrt(Dk) if scale is None else scale, out=out.data_ptr(), lse=lse.data_ptr(),
                          dev_status=device_status(dev).data_ptr())
    k_new = v_new = None
    if k_t is not None:
        k_t, v_t = _dense_head(k_t), _dense_head(v_t)
        a.k_t, a.k_stride_b, a.k_stride_h = k_t.data_ptr(), k_t.stride(0), k_t.stride(2)
        a.v_t, a.v_stride_b, a.v_stride_h = v_t.data_ptr(), v_t.stride(0), v_t.stride(2)
        if cos is not None:
            cos, sin = _table(cos), _table(sin)
            a.rope_cos, a.rope_sin, a.R, a.n_pos = cos.data_ptr(), sin.data_ptr(), 2 * cos.shape[1], cos.shape[0]
            a.interleaved = layout == "interleaved"
        a.advance = bool(advance)
        if stored:
            k_new = torch.empty(B, 1, c.Hkv, c.Dk, device=dev, dtype=cache.dtype)
            v_new = torch.empty(B, 1, c.Hkv, c.Dv, device=dev, dtype=cache.dtype)
            a.k_new, a.v_new, a.new_dtype = k_new.data_ptr(), v_new.data_ptr(), _lib.dtype_code(cache.dtype)
    stream = torch.cuda.current_stream(dev).cuda_stream
    floats = _lib.lib().tc_kv_attend_scratch_floats(c, B, Hq, most)
    counts = B * (c.Hkv * ((Hq // c.Hkv + 7) // 8) + 1)
    work, done = _workspace(dev, stream, floats, counts)
    if floats:
        a.scratch, a.scratch_floats = work.data_ptr(), work.numel()
    a.counters, a.num_counters = done.data_ptr(), done.numel()
    _lib.launch("tc_kv_attend", dev, c, a, ctypes.c_void_p(stream))
    return out, lse, k_new, v_new


@torch.no_grad()
def cached_attention(q_t: torch.Tensor, cache: KVCache, *, softcap: Optional[float] = None,
                     scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out [B, 1, Hq, Dv], lse [B, 1, Hq] fp32) of one query per sequence,
    q_t [B, 1, Hq, Dk] (already rotated), over the tokens that rows 0 .. B - 1 of
    the cache hold; an empty row gives out 0 and lse -inf."""
    return _attend(cache, q_t, None, None, None, None, "half", softcap, scale, False, False)[:2]


@torch.no_grad()
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
    the key and value that the written codes stand for, [B, 1, Hkv, D]."""
    if k_t.dim() != 4 or v_t.dim() != 4 or q_t.dim() != 4 or k_t.shape[:2] != q_t.shape[:2] or \
            v_t.shape[:3] != k_t.shape[:3]:
        raise ValueError(f"q_t {tuple(q_t.shape)}, k_t {tuple(k_t.shape)}, v_t {tuple(v_t.shape)} do not go together")
    if q_t.dtype != k_t.dtype or q_t.dtype != v_t.dtype:
        raise ValueError(f"q_t, k_t, v_t must share a dtype, got {q_t.dtype}, {k_t.dtype}, {v_t.dtype}")
    if (k_t.shape[2], k_t.shape[3], v_t.shape[3]) != (cache.k.shape[1], cache.k.shape[3], cache.v.shape[3]):
        raise ValueError(f"k_t {tuple(k_t.shape)}, v_t {tuple(v_t.shape)} do not fit the cache")
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    if (rope_cos is None) != (rope_sin is None):
        raise ValueError("rope_cos and rope_sin go together")
    if rope_cos is not None:
        if rope_cos.shape != rope_sin.shape or rope_cos.dim() != 2 or 2 * rope_cos.shape[1] > q_t.shape[3]:
            raise ValueError(f"rope tables {tuple(rope_cos.shape)}, {tuple(rope_sin.shape)} must be [n_pos, R / 2] with "
                             f"R <= {q_t.shape[3]}")
        if rope_cos.shape[0] <= cache.max_length:
            raise ValueError(f"rope tables cover {rope_cos.shape[0]} positions; the token may be at {cache.max_length}")
    if cache.max_length >= cache.capacity:
        raise ValueError(f"a row may be full: max_length {cache.max_length}, capacity {cache.capacity}")
    r = _attend(cache, q_t, k_t, v_t, rope_cos, rope_sin, layout, softcap, scale, advance, return_stored)
    if advance:
        cache.max_length += 1
    return r if return_stored else r[:2]


__all__ = ["KVCache", "init_kv_cache", "write_kv_cache", "read_kv_cache", "cached_attention", "cached_attention_step"]
