"""Requests that share, give up and move their cache slots, around the rounds that ``verify_step`` and ``commit_accept``
run.

The request table (``req_to_token`` int32 [rows, L]; row r holds the slots of request r's ``seq_lens[r]`` positions) is
the one ``commit_accept`` writes.  ``shared`` (int32 [num_slots], zeros to begin with) counts the requests beyond the first
that hold a slot, so requests that share nothing need no entry in it: slots that are handed out or that
``commit_accept`` frees have 0 there.  A block table (``kernels.blocks``) is such a table too, with its own lengths
(finished blocks) and its own ``shared``.  The reference leaves all of this to SGLang's pools.
"""

from __future__ import annotations

import torch

from dspine_amd import _lib
from dspine_amd.kernels.cache import _distinct, slot_rows
from dspine_amd.verify import Workspace, scratch

_INT = (torch.int32, torch.int64)


def _check_requests(req_to_token, seq_lens):
    t, shape, dtype = req_to_token, req_to_token.shape, seq_lens.dtype
    if len(shape) != 2 or t.dtype != torch.int32 or shape[0] < 1 or shape[1] < 1 or (t.stride(1) != 1 and shape[1] > 1):
        raise ValueError("req_to_token must be row-contiguous int32 [rows, L]")
    _distinct(t, "req_to_token")
    if seq_lens.shape != shape[:1] or dtype not in _INT or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32/int64 vector of the table's rows")
    stride = t.stride(0) if shape[0] > 1 else shape[1]
    return t.data_ptr(), shape[0], stride, shape[1], seq_lens.data_ptr(), int(dtype == torch.int64)


def _check_shared(shared):
    if shared.ndim != 1 or shared.dtype != torch.int32 or not shared.is_contiguous() or shared.numel() < 1:
        raise ValueError("shared must be a contiguous int32 vector of the pool's slots")


def _check_rows(rows, name):
    if rows.ndim != 1 or rows.dtype not in _INT or not rows.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32/int64 vector")
    return int(rows.dtype == torch.int64)


def fork_requests(req_to_token: torch.Tensor, seq_lens: torch.Tensor, shared: torch.Tensor, parents: torch.Tensor,
                  children: torch.Tensor) -> None:
    """Row ``children[i]`` becomes a copy of row ``parents[i]`` (int32 or int64 [n]): the parent's slots, each with
    one holder more in ``shared``, and its length; on the current stream.  A parent may have any number of children;
    the children must be distinct, hold nothing (what they held is not released) and be no parents of the call, or what the
    tables then hold is undefined.  Rows outside the table and pairs of equal rows are skipped.  Later positions get slots
    of their own as always, so nothing has to be copied on a write."""
    table = _check_requests(req_to_token, seq_lens)
    _check_shared(shared)
    i64 = _check_rows(parents, "parents")
    if _check_rows(children, "children") != i64 or children.shape != parents.shape:
        raise ValueError("parents and children must be of one length and dtype")
    dev = _lib.require_cuda(req_to_token, seq_lens, shared, parents, children)
    _lib.launch("dsv_fork_requests", dev, _lib.load().dsv_fork_requests, *table, shared.data_ptr(), shared.numel(),
                parents.data_ptr(), children.data_ptr(), i64, parents.numel())


def free_requests(req_to_token: torch.Tensor, seq_lens: torch.Tensor, shared: torch.Tensor, rows: torch.Tensor, *,
                  free_slots: torch.Tensor | None = None, free_count: torch.Tensor | None = None,
                  workspace: Workspace | None = None):
    """The requests in ``rows`` (int32 or int64 [n]; one named again counts once, rows outside the table are skipped) end:
    their lengths become 0 and each of their slots loses a holder.  Returns ``(free_slots, free_count)``: the slots that
    nobody else holds in ascending order (int64; entries past the count are left as they were) and their number
    (int32 [1]).  ``free_slots``: a vector to fill; one shorter than the slots that are freed gets the first of
    them, so give it room for the rows' lengths."""
    table = _check_requests(req_to_token, seq_lens)
    _check_shared(shared)
    i64 = _check_rows(rows, "rows")
    if free_slots is None:
        room = min(shared.numel(), rows.numel() * req_to_token.shape[1])
        free_slots = torch.empty(room, dtype=torch.int64, device=shared.device)
    elif free_slots.ndim != 1 or free_slots.dtype != torch.int64 or not free_slots.is_contiguous():
        raise ValueError("free_slots must be a contiguous int64 vector")
    if free_count is None:
        free_count = torch.empty(1, dtype=torch.int32, device=shared.device)
    elif free_count.dtype != torch.int32 or free_count.numel() < 1:
        raise ValueError("free_count must be int32 [1]")
    dev = _lib.require_cuda(req_to_token, seq_lens, shared, rows, free_slots, free_count)
    lib = _lib.load()
    buf = scratch(workspace, lib.dsv_free_requests_workspace_bytes(shared.numel()), dev)
    _lib.launch("dsv_free_requests", dev, lib.dsv_free_requests, *table, shared.data_ptr(), shared.numel(),
                rows.data_ptr(), i64, rows.numel(), free_slots.data_ptr(), free_slots.numel(), free_count.data_ptr(),
                buf.data_ptr(), buf.numel())
    return free_slots, free_count


def compact_requests(req_to_token: torch.Tensor, seq_lens: torch.Tensor, rows: torch.Tensor, caches, *,
                     shared: torch.Tensor | None = None, moves: torch.Tensor | None = None,
                     counts: torch.Tensor | None = None, workspace: Workspace | None = None):
    """The used slots of a pool to its front: with U distinct slots in the requests ``rows`` (int32 or int64 [n]), which must
    be all that hold any, those at or above U move, in ascending order, into the unused ones below U, in ascending order.
    The rows' entries, ``shared`` and every tensor of ``caches`` (a ``KVCache``, a ``BlockIndex`` for a block table, or
    a list of them: the model's layers) follow; what lies in a slot that was moved from stays there.  Returns ``(moves,
    counts)``: int64 [2, >= num_slots // 2], from and to, and int32 [2], U and the number of moves; entries past it are
    left as they were.  A slot that none of ``rows`` holds is unused, and may be written over: slots that are kept outside the
    table (padding's, a prefix cache's) need a row of their own among them.  Slots of drafts that no length counts yet are not
    held: call between rounds."""
    table = _check_requests(req_to_token, seq_lens)
    i64 = _check_rows(rows, "rows")
    parts, tensors, slots = slot_rows(caches)
    if shared is not None:
        _check_shared(shared)
        if shared.numel() != slots:
            raise ValueError("shared must count the caches' slots")
    if moves is None:
        moves = torch.empty((2, slots // 2), dtype=torch.int64, device=tensors[0].device)
    elif moves.ndim != 2 or moves.shape[0] != 2 or moves.shape[1] < slots // 2 or moves.dtype != torch.int64 \
            or not moves.is_contiguous():
        raise ValueError("moves must be contiguous int64 [2, num_slots // 2] or wider")
    if counts is None:
        counts = torch.empty(2, dtype=torch.int32, device=tensors[0].device)
    elif counts.dtype != torch.int32 or counts.numel() < 2 or not counts.is_contiguous():
        raise ValueError("counts must be contiguous int32 [2]")
    dev = _lib.require_cuda(req_to_token, seq_lens, rows, *tensors, shared, moves, counts)
    lib = _lib.load()
    buf = scratch(workspace, lib.dsv_compact_requests_workspace_bytes(slots), dev)
    room = moves.shape[1]
    _lib.launch("dsv_compact_requests", dev, lib.dsv_compact_requests, *table, _lib.ptr(shared), slots, rows.data_ptr(), i64,
                rows.numel(), parts, len(parts), moves.data_ptr(), moves.data_ptr() + 8 * room, room, counts.data_ptr(),
                buf.data_ptr(), buf.numel())
    return moves, counts
