"""Attention over a long context's best blocks.

A request's context is cut into blocks of 16 to 128 positions.  Of every block that a round or a prompt
finishes, ``index_blocks`` keeps the least and largest key elements of each cache head; from them and a
round's queries ``score_blocks`` bounds every block's attention scores at a small part of the keys' bytes;
``select_blocks`` picks the best of each (request, cache head), and ``block_attention`` is
``kernels.attention.tree_attention`` over those, the unfinished block and the window.  A request's nodes and
the query heads of a cache head choose together; a chain's drafts given as requests of one node (T == 1,
``prefix_lens`` counting the drafts before them) choose each for itself, and a prompt's queries in groups of up
to 64.  The reference leaves the cache and its attention to SGLang, which reads the whole context.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from dspine_amd import _lib
from dspine_amd.kernels.attention import MAX_NODES, attention_args, with_workspace
from dspine_amd.kernels.cache import _ACT, KVCache, _rows, cache_fields, tensors_of
from dspine_amd.verify import Workspace

BLOCK_SIZES = (16, 32, 64, 128)
MAX_BLOCKS = 32768  # of a request, that select_blocks ranks


@dataclass
class BlockIndex:
    """bounds [rows, heads, 2, dim] (bfloat16 or float16, contiguous): of the block that a row is for, each
    head's least and largest key elements; a block has ``block_size`` (16, 32, 64 or 128) positions and
    begins at a multiple of it.  Rows belong to blocks by a block table, as slots do to positions by a page
    table: requests that share slots share the rows of their finished blocks."""

    bounds: torch.Tensor
    block_size: int


def new_block_index(rows: int, heads: int, dim: int, *, block_size: int = 64, dtype: torch.dtype = torch.bfloat16,
                    device) -> BlockIndex:
    """A zeroed index of one layer."""
    if dtype not in _ACT:
        raise ValueError(f"unsupported index dtype {dtype}")
    index = BlockIndex(torch.zeros((rows, heads, 2, dim), dtype=dtype, device=device), block_size)
    index_fields(index)
    return index


def _check_size(block_size):
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"a block has 16, 32, 64 or 128 positions, got {block_size}")
    return int(block_size)


def index_fields(index: BlockIndex) -> _lib.BlockIndexC:
    """The ``dsv_block_index`` of an index, checked but for its device."""
    x = index.bounds
    shape, code = x.shape, _ACT.get(x.dtype)
    if len(shape) != 4 or shape[2] != 2 or code is None or not x.is_contiguous():
        raise ValueError("an index's bounds must be contiguous bfloat16 or float16 [rows, heads, 2, dim]")
    rows, heads, _, dim = shape
    if dim % 16 or not 16 <= dim <= 256 or rows < 1 or heads < 1:
        raise ValueError("an index needs rows, heads and a dim that is a multiple of 16 up to 256")
    at = x.data_ptr()
    if at % 16:
        raise ValueError("an index's bounds must start on a 16-byte boundary")
    return _lib.BlockIndexC(at, code, heads, dim, _check_size(index.block_size), rows)


def _check_table(t, name, bs):
    """(address, row stride, columns)"""
    shape = t.shape
    if len(shape) != 2 or shape[0] != bs or t.dtype != torch.int32 or shape[1] < 1:
        raise ValueError(f"{name} must be int32 [bs, L]")
    row, last = t.stride()
    if last != 1 and shape[1] > 1:
        raise ValueError(f"{name} rows must be contiguous")
    return t.data_ptr(), row, shape[1]


def _check_lens(t, name, bs=None):
    if t.ndim != 1 or t.dtype != torch.int32 or not t.is_contiguous() or (bs is not None and t.shape[0] != bs):
        raise ValueError(f"{name} must be contiguous int32 [bs]")
    return t.shape[0]


def index_blocks(index: BlockIndex, cache: KVCache, *, page_table: torch.Tensor, block_table: torch.Tensor,
                 from_lens: torch.Tensor, to_lens: torch.Tensor, longest: int | None = None) -> None:
    """The bounds of the blocks that each request finished as it grew from ``from_lens[b]`` to ``to_lens[b]``
    positions (int32 [bs]) whose keys are written: of each block j with from // block_size <= j < to // block_size into
    index row ``block_table[b, j]`` (int32 [bs, L]), on the current stream.  ``page_table`` is that of these positions: after
    a commit the request table's rows as the commit left them, not the window's of the attention before it.

    Keys are what ``read_kv`` gives in float32, rounded once to the index's type (so a bound may lie half a step inside), those
    that are finite but past its range to its largest number; a NaN makes both bounds of its element NaN.  Positions
    past ``page_table`` (int32 [bs, L]) and slots outside the cache do not count, a block of nothing else gets zeros.  Blocks
    past ``block_table`` and rows outside the index are skipped; the rows of a call must be distinct.  ``longest``: the most
    positions that any request grew by (default: the page table's width); a growth beyond it is not indexed."""
    x, c = index_fields(index), cache_fields(cache)
    if (x.heads, x.dim) != (c.heads, c.dim):
        raise ValueError("the index and the cache must have the same heads and dim")
    bs = _check_lens(from_lens, "from_lens")
    _check_lens(to_lens, "to_lens", bs)
    pages, table = _check_table(page_table, "page_table", bs), _check_table(block_table, "block_table", bs)
    longest = pages[2] if longest is None else int(longest)
    if longest < 0:
        raise ValueError(f"longest {longest} is negative")
    dev = _lib.require_cuda(index.bounds, *tensors_of(cache), page_table, block_table, from_lens, to_lens)
    _lib.launch("dsv_index_blocks", dev, _lib.load().dsv_index_blocks, x, c, *pages, *table, from_lens.data_ptr(),
                to_lens.data_ptr(), bs, longest)


def score_blocks(q: torch.Tensor, index: BlockIndex, *, T: int, block_table: torch.Tensor, prefix_lens: torch.Tensor,
                 verify_lens: torch.Tensor | None = None, row_offsets: torch.Tensor | None = None,
                 scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """float32 [bs, heads, L]: for each block j of ``block_table`` (int32 [bs, L]) the largest, over the request's nodes and
    the query heads of a cache head, of scale * sum_d max(q_d least_d, q_d largest_d), which no scaled score of the block's
    keys exceeds (but for the bounds' rounding).

    q [rows, q_heads, dim] of the index's dtype, ``T``, ``prefix_lens``, ``verify_lens`` and ``row_offsets`` as in
    ``tree_attention``; 0 < ``scale``, default 1 / sqrt(dim).  Blocks from prefix_lens[b] // block_size on, rows outside the
    index and requests without nodes (one whose row lies outside q is none) get -inf.  A NaN among a block's terms makes its
    score NaN, whichever node it is of: a query with a NaN, a NaN bound, an infinite one beside a query of zero, infinities of
    both signs.  ``out``: a contiguous tensor to fill."""
    if q.ndim != 3 or q.dtype not in _ACT:
        raise ValueError("q must be bfloat16 or float16 [rows, q_heads, dim]")
    x = index_fields(index)
    rows, heads, dim = q.shape
    if dim != x.dim or heads < 1 or heads % x.heads:
        raise ValueError("q must have the index's dim and a multiple of its heads")
    if index.bounds.dtype != q.dtype:
        raise ValueError("queries and index must be of one dtype")
    T = int(T)
    if not 1 <= T <= MAX_NODES:
        raise ValueError(f"T {T} outside [1, {MAX_NODES}]")
    bs = _check_lens(prefix_lens, "prefix_lens")
    if bs < 1:
        raise ValueError("empty attention batch")
    if row_offsets is None and rows != bs * T:
        raise ValueError(f"dense layout needs q rows == bs*T ({rows} != {bs}*{T})")
    if row_offsets is not None and (row_offsets.shape != (bs,) or row_offsets.dtype not in (torch.int32, torch.int64)
                                    or not row_offsets.is_contiguous()):
        raise ValueError("row_offsets must be a contiguous int32/int64 vector of batch size")
    if verify_lens is not None:
        _check_lens(verify_lens, "verify_lens", bs)
    table = _check_table(block_table, "block_table", bs)
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not 0.0 < scale <= 2.0 ** 100:
        raise ValueError("scale must be positive, at most 2^100")
    shape = (bs, x.heads, table[2])
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=q.device)
    elif out.shape != shape or out.dtype != torch.float32 or not out.is_contiguous():
        raise ValueError("out must be contiguous float32 [bs, heads, L]")
    q_at, q_row, q_head = _rows(q, "q") if rows else (None, 0, 0)
    dev = _lib.require_cuda(q, index.bounds, block_table, prefix_lens, verify_lens, row_offsets, out)
    a = _lib.ScoreBlocksArgs(x, q_at, out.data_ptr(), heads, 0, rows, q_row, q_head, bs, T, prefix_lens.data_ptr(),
                             _lib.ptr(verify_lens), _lib.ptr(row_offsets),
                             int(row_offsets is not None and row_offsets.dtype == torch.int64), scale, *table)
    _lib.launch("dsv_score_blocks", dev, _lib.load().dsv_score_blocks, a)
    return out


def select_blocks(scores: torch.Tensor, count: int, *, prefix_lens: torch.Tensor, block_size: int, first: int = 0,
                  last: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """int32 [bs, heads, count]: of each (request, head)'s n = min(prefix_lens[b] // block_size, L) finished blocks
    the ``first`` first, the ``last`` last and, to make ``count``, those of the largest ``scores`` (float32 [bs, heads, L],
    contiguous, L <= 32768; ties to the lowest block, NaN as -inf), in ascending order, then -1 where n < count.
    first + last <= count."""
    shape = scores.shape
    if len(shape) != 3 or scores.dtype != torch.float32 or not scores.is_contiguous():
        raise ValueError("scores must be contiguous float32 [bs, heads, L]")
    bs, heads, cols = shape
    if not 1 <= cols <= MAX_BLOCKS:
        raise ValueError(f"1 to {MAX_BLOCKS} blocks of a request are ranked, got {cols}")
    if bs < 1 or heads < 1:
        raise ValueError("empty selection batch")
    _check_lens(prefix_lens, "prefix_lens", bs)
    block_size, count, first, last = _check_size(block_size), int(count), int(first), int(last)
    if count < 1 or first < 0 or last < 0 or first + last > count or count > 2 ** 24:
        raise ValueError(f"count {count} has to hold the first {first} and the last {last} blocks")
    shape = (bs, heads, count)
    if out is None:
        out = torch.empty(shape, dtype=torch.int32, device=scores.device)
    elif out.shape != shape or out.dtype != torch.int32 or not out.is_contiguous():
        raise ValueError("out must be contiguous int32 [bs, heads, count]")
    dev = _lib.require_cuda(scores, prefix_lens, out)
    _lib.launch("dsv_select_blocks", dev, _lib.load().dsv_select_blocks, scores.data_ptr(), bs, heads, cols,
                prefix_lens.data_ptr(), block_size, count, first, last, out.data_ptr())
    return out


def block_attention(q: torch.Tensor, cache: KVCache, *, T: int, blocks: torch.Tensor, block_size: int,
                    page_table: torch.Tensor, prefix_lens: torch.Tensor, verify_lens: torch.Tensor | None = None,
                    row_offsets: torch.Tensor | None = None, masks: torch.Tensor | None = None,
                    scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                    workspace: Workspace | None = None) -> torch.Tensor:
    """``tree_attention`` (its arguments, rows, masks, workspace and results) where of the context a cache head h's
    queries see only the blocks ``blocks[b, h, i]``, i < min(count, prefix_lens[b] // block_size) (int32 [bs, heads, count],
    contiguous; ``select_blocks``), and the positions from the last finished block's end on.  An entry that names no
    finished block (-1 among them) holds nothing; one that names a block again counts it again."""
    block_size = _check_size(block_size)
    lists, k = blocks.shape, cache.k.shape
    if (len(lists) != 3 or lists[:1] != prefix_lens.shape[:1] or len(k) != 3 or lists[1] != k[1] or lists[2] < 1
            or blocks.dtype != torch.int32 or not blocks.is_contiguous()):
        raise ValueError("blocks must be contiguous int32 [bs, heads, count]")
    a, dev, out = attention_args(q, cache, T=T, page_table=page_table, prefix_lens=prefix_lens, verify_lens=verify_lens,
                                 row_offsets=row_offsets, masks=masks, scale=scale, out=out, lse=lse, also=(blocks,))
    if a is not None:
        held = with_workspace(a, dev, workspace)  # (until the launch)
        _lib.launch("dsv_block_attention", dev, _lib.load().dsv_block_attention,
                    _lib.BlockAttentionArgs(a, blocks.data_ptr(), lists[2], block_size))
        del held
    return out
