"""Attention of a round's drafted nodes over the paged KV cache: what the target forward runs in
every layer between writing the nodes' keys and values (``kernels.cache.write_kv``) and the logits
that ``verification.tree.accept_greedy_tree`` or ``verify_step`` accept from.  The reference leaves
it to SGLang's attention backends, which its chains reach through ``prefix_lens`` and the page table.
"""

from __future__ import annotations

import math

import torch

from dspine_amd import _lib
from dspine_amd.kernels.cache import _ACT, QUANTISED, KVCache, _distinct, _rows, cache_fields, tensors_of
from dspine_amd.verify import Workspace, scratch

MAX_NODES = 64


def tree_attention(q: torch.Tensor, cache: KVCache, *, T: int, page_table: torch.Tensor, prefix_lens: torch.Tensor,
                   verify_lens: torch.Tensor | None = None, row_offsets: torch.Tensor | None = None,
                   masks: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                   lse: torch.Tensor | None = None, workspace: Workspace | None = None) -> torch.Tensor:
    """q [rows, q_heads, dim] (bfloat16 or float16; a 16-bit cache's own type) against the cache;
    returns out, of q's shape and dtype.

    Request b has ``verify_lens[b]`` nodes (int32 [bs], clamped into [0, T]; default T; T <= 64) on the
    rows ``b*T + i`` or ``row_offsets[b] + i``.  Its node i sees the positions before ``prefix_lens[b]``
    (int32 [bs]) and, of the window at ``prefix_lens[b] + j``, the nodes j whose bit is set in
    ``masks[b, i]`` (int64 [bs, T], ``verification.tree.tree_masks``; any mask is taken as it is), or
    without masks the chain j <= i.  Position p lies in slot ``page_table[b, p]`` (int32 [bs, L]);
    positions past L and slots outside the cache hold nothing.  Query head h reads cache head
    ``h // (q_heads // heads)``; ``scale`` defaults to 1 / sqrt(dim).  A node that sees nothing gets zeros;
    rows of no node are left as they were.  ``lse`` (float32 [rows, q_heads]) receives log sum exp of the
    scaled scores (-inf for such a node).  T == 1 is ordinary single-token decoding.

    The work is split over the positions, so a call needs scratch memory, which it allocates on the
    current stream (in a captured graph: in the graph's own pool) or takes from ``workspace``; two calls
    that may run at once must not be given one workspace, and one whose buffer a captured graph uses must live as
    long as the graph."""
    a, dev, out = attention_args(q, cache, T=T, page_table=page_table, prefix_lens=prefix_lens, verify_lens=verify_lens,
                                 row_offsets=row_offsets, masks=masks, scale=scale, out=out, lse=lse)
    if a is not None:
        held = with_workspace(a, dev, workspace)  # (until the launch)
        _lib.launch("dsv_tree_attention", dev, _lib.load().dsv_tree_attention, a)
        del held
    return out


def attention_args(q, cache, *, T, page_table, prefix_lens, verify_lens, row_offsets, masks, scale, out, lse, also=()):
    """(the ``dsv_tree_attention_args`` but for the workspace, or None without rows; the device; out), checked;
    ``also``: tensors that have to be on the same device."""
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3 or dtype not in _ACT:
        raise ValueError("q must be bfloat16 or float16 [rows, q_heads, dim]")
    c = cache_fields(cache)
    rows, heads, dim = shape
    if dim != c.dim or heads < 1 or heads % c.heads:
        raise ValueError("q must have the cache's dim and a multiple of its heads")
    if cache.k.dtype not in QUANTISED and cache.k.dtype != dtype:
        raise ValueError("queries and a 16-bit cache must be of one dtype")
    T = int(T)
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"T {T} outside [1, {MAX_NODES}]")
    if prefix_lens.ndim != 1 or prefix_lens.dtype != torch.int32 or not prefix_lens.is_contiguous():
        raise ValueError("prefix_lens must be contiguous int32 [bs]")
    bs = prefix_lens.shape[0]
    if bs < 1:
        raise ValueError("empty attention batch")
    if row_offsets is None and rows != bs * T:
        raise ValueError(f"dense layout needs q rows == bs*T ({rows} != {bs}*{T})")
    if row_offsets is not None and (row_offsets.shape != (bs,) or row_offsets.dtype not in (torch.int32, torch.int64)
                                    or not row_offsets.is_contiguous()):
        raise ValueError("row_offsets must be a contiguous int32/int64 vector of batch size")
    if verify_lens is not None and (verify_lens.shape != (bs,) or verify_lens.dtype != torch.int32
                                    or not verify_lens.is_contiguous()):
        raise ValueError("verify_lens must be contiguous int32 [bs]")
    if masks is not None and (masks.shape != (bs, T) or masks.dtype != torch.int64 or not masks.is_contiguous()):
        raise ValueError("masks must be contiguous int64 [bs, T]")
    pages = page_table.shape
    if len(pages) != 2 or pages[0] != bs or page_table.dtype != torch.int32 or pages[1] < 1:
        raise ValueError("page_table must be int32 [bs, L]")
    page_stride, last = page_table.stride()
    if last != 1 and pages[1] > 1:
        raise ValueError("page_table rows must be contiguous")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not abs(scale) <= 2.0 ** 100:
        raise ValueError("scale must be finite, at most 2^100")
    own = out is None
    if own:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype:
        raise ValueError("out must have q's shape and dtype")
    if lse is not None and (lse.shape != (rows, heads) or lse.dtype != torch.float32 or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous float32 [rows, q_heads]")
    if rows:
        q_at, q_row, q_head = _rows(q, "q")
        if own:
            out_at, out_row, out_head = out.data_ptr(), heads * dim, dim
        else:
            out_at, out_row, out_head = _rows(out, "out")
            _distinct(out, "out")
    dev = _lib.require_cuda(q, *tensors_of(cache), page_table, prefix_lens, verify_lens, row_offsets, masks, out, lse,
                            *also)
    if rows == 0:
        return None, dev, out
    ptr = _lib.ptr
    return _lib.TreeAttentionArgs(
        c, q_at, out_at, ptr(lse), _ACT[dtype], heads, rows, q_row, q_head, out_row, out_head, bs, T,
        prefix_lens.data_ptr(), ptr(verify_lens), ptr(row_offsets),
        int(row_offsets is not None and row_offsets.dtype == torch.int64), scale, ptr(masks), page_table.data_ptr(),
        page_stride, pages[1], None, 0), dev, out


def with_workspace(a, dev, workspace):
    """Give a call its scratch memory; returns what holds it."""
    buf = scratch(workspace, _lib.load().dsv_tree_attention_workspace_bytes(a.bs, a.T, a.cache.heads, a.q_heads, a.cache.dim), dev)
    a.workspace, a.workspace_bytes = buf.data_ptr(), buf.numel()
    return buf
