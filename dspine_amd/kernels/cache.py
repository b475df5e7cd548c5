"""The paged KV cache of one layer: writing a round's keys and values into its slots and reading
slots back.

The reference leaves the cache to SGLang; here its slots are the ones ``verify_step`` gathers and
``commit_accept`` hands out (page size 1: a position lies in slot ``page_table[b, position]``).
A cache holds bfloat16 or float16 values, or 8-bit codes (OCP e4m3 or int8) with a float32 scale
for each (slot, head): value = code * scale.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from dspine_amd import _lib

_CACHE = {torch.bfloat16: _lib.DSV_BF16, torch.float16: _lib.DSV_F16, torch.float8_e4m3fn: _lib.DSV_E4M3,
          torch.int8: _lib.DSV_I8}
_ACT = {torch.bfloat16: _lib.DSV_BF16, torch.float16: _lib.DSV_F16}
_OUT = {torch.float32: _lib.DSV_F32, **_ACT}
QUANTISED = (torch.float8_e4m3fn, torch.int8)


@dataclass
class KVCache:
    """k and v [num_slots, heads, dim] (bfloat16, float16, float8_e4m3fn or int8; any strides with
    the last dimension contiguous and every row on a 16-byte boundary; dim a multiple of 16 up to
    256), with k_scale and v_scale float32 [num_slots, heads] for the 8-bit types."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None


def new_cache(num_slots: int, heads: int, dim: int, *, dtype: torch.dtype = torch.bfloat16, device) -> KVCache:
    """A zeroed cache."""
    if dtype not in _CACHE:
        raise ValueError(f"unsupported cache dtype {dtype}")
    k, v = (torch.zeros((num_slots, heads, dim), dtype=dtype, device=device) for _ in range(2))
    if dtype not in QUANTISED:
        return KVCache(k, v)
    return KVCache(k, v, *(torch.zeros((num_slots, heads), device=device) for _ in range(2)))


def _rows(t, name):
    """(address, row stride, head stride) of t [., heads, dim]; its rows must be contiguous and start
    on 16-byte boundaries.  The stride of a dimension of one says nothing: 0."""
    at, size = t.data_ptr(), t.element_size()
    n, heads, dim = t.shape
    if t.is_contiguous():
        row, head = heads * dim, dim
    else:
        row, head, last = t.stride()
        if last != 1 and dim != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
        row, head = row if n > 1 else 0, head if heads > 1 else 0
    if at % 16 or row * size % 16 or head * size % 16:
        raise ValueError(f"{name} must have its rows on 16-byte boundaries")
    return at, row, head


def _distinct(t, name):
    """Refuse a tensor to be written whose elements share memory."""
    if t.is_contiguous():
        return
    reach = 1
    for stride, size in sorted((t.stride(i), t.shape[i]) for i in range(t.ndim) if t.shape[i] > 1):
        if stride < reach:
            raise ValueError(f"{name} must not overlap itself")
        reach = stride * (size - 1) + reach


def tensors_of(cache: KVCache):
    return cache.k, cache.v, cache.k_scale, cache.v_scale


def cache_fields(cache: KVCache, *, write: bool = False) -> _lib.KvCache:
    """The ``dsv_kv_cache`` of a cache, checked but for its device."""
    k, v, ks, vs = cache.k, cache.v, cache.k_scale, cache.v_scale
    shape, dtype = k.shape, k.dtype
    code = _CACHE.get(dtype)
    if len(shape) != 3 or v.shape != shape or code is None or v.dtype != dtype:
        raise ValueError("a cache's k and v must be [num_slots, heads, dim] of one supported dtype")
    slots, heads, dim = shape
    if dim % 16 or not 16 <= dim <= 256 or slots < 1 or heads < 1:
        raise ValueError("a cache needs slots, heads and a dim that is a multiple of 16 up to 256")
    k_at, k_slot, k_head = _rows(k, "cache k")
    v_at, v_slot, v_head = _rows(v, "cache v")
    quant = code in (_lib.DSV_E4M3, _lib.DSV_I8)
    if (ks is not None) != quant or (vs is not None) != quant:
        raise ValueError("scales belong to the 8-bit caches, both of them")
    scales = (None, None, 0, 0, 0, 0)
    if quant:
        for name, t in (("k_scale", ks), ("v_scale", vs)):
            if t.shape != shape[:2] or t.dtype != torch.float32:
                raise ValueError(f"{name} must be float32 [num_slots, heads]")
        scales = (ks.data_ptr(), vs.data_ptr(), *ks.stride(), *vs.stride())
    if write:
        for name, t in (("cache k", k), ("cache v", v), ("k_scale", ks), ("v_scale", vs)):
            if t is not None:
                _distinct(t, name)
    return _lib.KvCache(k_at, v_at, code, heads, dim, 0, slots, k_slot, k_head, v_slot, v_head, *scales)


def _check_slots(slots):
    if slots.ndim != 1 or slots.dtype not in (torch.int32, torch.int64) or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int32/int64 vector")
    return int(slots.dtype == torch.int64)


def write_kv(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """k, v [n, heads, dim] (bfloat16 or float16, 16-byte-aligned rows; slices of a fused projection
    are fine) into the cache's ``slots`` [n], on the current stream.

    An 8-bit cache gets, for each (token, head), the scale max |x| * (1 / top) and the codes
    rne(x * (top / max |x|)), top 448 (e4m3) or 127 (int8); a row whose largest magnitude is below
    2^-100 becomes zeros, a row with a NaN or an infinity the scale NaN over zero codes, so that it
    reads back as NaN.  A 16-bit cache takes its own type.  Slots outside [0, num_slots) (padding) are
    skipped; the others must be distinct, or which token a repeated slot holds is undefined."""
    i64 = _check_slots(slots)
    c = cache_fields(cache, write=True)
    shape = (slots.numel(), c.heads, c.dim)
    if tuple(k.shape) != shape or tuple(v.shape) != shape or k.dtype not in _ACT or v.dtype != k.dtype:
        raise ValueError("k and v must be bfloat16 or float16 [len(slots), heads, dim]")
    if cache.k.dtype not in QUANTISED and cache.k.dtype != k.dtype:
        raise ValueError("a 16-bit cache holds its own dtype only")
    if shape[0] == 0:
        return
    k_at, k_row, k_head = _rows(k, "k")
    v_at, v_row, v_head = _rows(v, "v")
    dev = _lib.require_cuda(*tensors_of(cache), k, v, slots)
    _lib.launch("dsv_kv_write", dev, _lib.load().dsv_kv_write, c, k_at, v_at, _ACT[k.dtype], shape[0], k_row, k_head, v_row,
                v_head, slots.data_ptr(), i64)


def read_kv(cache: KVCache, slots: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16, out=None):
    """(k, v) [n, heads, dim] of the cache's ``slots`` [n] as ``dtype`` (bfloat16, float16 or
    float32): code * scale, rounded once.  Slots may repeat; one outside [0, num_slots) reads as zeros.
    ``out``: a pair of contiguous tensors to fill."""
    i64 = _check_slots(slots)
    c = cache_fields(cache)
    shape = (slots.numel(), c.heads, c.dim)
    if out is None:
        if dtype not in _OUT:
            raise ValueError(f"unsupported dtype {dtype} (expected float32, bfloat16 or float16)")
        out = tuple(torch.empty(shape, dtype=dtype, device=cache.k.device) for _ in range(2))
    k, v = out
    for t in (k, v):
        if tuple(t.shape) != shape or t.dtype not in _OUT or t.dtype != k.dtype or not t.is_contiguous():
            raise ValueError("out must be two contiguous [len(slots), heads, dim] tensors of one supported dtype")
        if shape[0] and t.data_ptr() % 16:
            raise ValueError("out must start on a 16-byte boundary")
    dev = _lib.require_cuda(*tensors_of(cache), k, v, slots)
    _lib.launch("dsv_kv_read", dev, _lib.load().dsv_kv_read, c, k.data_ptr(), v.data_ptr(), _OUT[k.dtype], shape[0],
                slots.data_ptr(), i64)
    return k, v
