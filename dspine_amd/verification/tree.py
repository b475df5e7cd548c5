"""Greedy verification of drafted trees.

The reference drafts and verifies chains (``verification/caps.py:32-59``); this is the same
acceptance over a tree of at most 64 nodes: node 0 is the last accepted token, every other node
hangs below an earlier one (``parents``), and the accepted drafts are the path of nodes that the
target's argmaxes take.  A chain (``parents[b, i] = i - 1``) accepts what ``accept_greedy`` does.
"""

from __future__ import annotations

import torch

from dspine_amd import _lib
from dspine_amd.verify import Workspace

MAX_NODES = 64


def _check_parents(parents):
    if parents.ndim != 2 or parents.dtype != torch.int32 or not parents.is_contiguous():
        raise ValueError("parents must be contiguous int32 [bs, T]")
    if not 1 <= parents.shape[1] <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {parents.shape[1]}")


def tree_masks(parents: torch.Tensor, masks: torch.Tensor | None = None, depths: torch.Tensor | None = None):
    """(masks int64 [bs, T], depths int32 [bs, T]) of drafted trees given by ``parents`` int32 [bs, T]:
    bit j of ``masks[b, i]`` says that node j is node i or an ancestor of it (what ``tree_attention``
    takes; bit 63 is the sign), ``depths`` counts the ancestors (a node's position is prefix + depth).
    ``parents[b, 0]`` is -1; a later node whose parent is not an earlier node is a root of its own."""
    _check_parents(parents)
    if masks is None:
        masks = torch.empty(parents.shape, dtype=torch.int64, device=parents.device)
    if depths is None:
        depths = torch.empty(parents.shape, dtype=torch.int32, device=parents.device)
    for name, t, dtype in (("masks", masks, torch.int64), ("depths", depths, torch.int32)):
        if t.shape != parents.shape or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {dtype} [bs, T]")
    dev = _lib.require_cuda(parents, masks, depths)
    _lib.launch("dsv_tree_masks", dev, _lib.load().dsv_tree_masks, parents.data_ptr(), parents.shape[0],
                parents.shape[1], masks.data_ptr(), depths.data_ptr())
    return masks, depths


def accept_greedy_tree(*, candidates: torch.Tensor, parents: torch.Tensor, next_token_logits: torch.Tensor,
                       prefix_lens: torch.Tensor, verify_lens: torch.Tensor | None = None, outputs=None,
                       path: torch.Tensor | None = None, workspace: Workspace | None = None):
    """Returns ``((accept i32, commit i32, bonus i64, output i64 [bs, T], new_seq i32), path i32 [bs, T])``.

    candidates [bs, T] int64: the nodes' tokens, node 0 the last accepted one; next_token_logits
    [bs*T, V] (bfloat16 or float32): row ``b*T + i`` follows node i.  From node 0 the path moves to the child
    that carries the argmax of the node it is at (lowest id on ties, NaN as -inf; of several such children
    the first) until none does; nodes at or past ``verify_lens[b]`` (int32 [bs], clamped into [1, T]) are not
    there and their rows are not read.  accept counts the moves, bonus is the last node's argmax, output holds the
    accepted tokens, the bonus, then zeros; ``path`` the nodes of the path (node 0 first), then -1 --
    what ``commit_accept(path=...)`` and a caller that gathers the path's hidden states take."""
    _check_parents(parents)
    if candidates.shape != parents.shape or candidates.dtype != torch.int64 or not candidates.is_contiguous():
        raise ValueError("candidates must be contiguous int64 [bs, T]")
    bs, T = candidates.shape
    if bs < 1:
        raise ValueError("empty verification batch")
    logits = next_token_logits
    if logits.ndim != 2 or logits.shape[0] != bs * T or logits.shape[1] < 1 or (logits.stride(1) != 1
                                                                               and logits.shape[1] > 1):
        raise ValueError("Greedy tree acceptance needs row-contiguous [bs*T, V] logits")
    if prefix_lens.shape != (bs,) or prefix_lens.dtype != torch.int32 or not prefix_lens.is_contiguous():
        raise ValueError("prefix_lens must be contiguous int32 [bs]")
    if verify_lens is not None and (verify_lens.shape != (bs,) or verify_lens.dtype != torch.int32
                                    or not verify_lens.is_contiguous()):
        raise ValueError("verify_lens must be contiguous int32 [bs]")
    if outputs is None:
        dev = candidates.device
        outputs = (torch.empty(bs, device=dev, dtype=torch.int32),
                   torch.empty(bs, device=dev, dtype=torch.int32),
                   torch.empty(bs, device=dev, dtype=torch.int64),
                   torch.empty((bs, T), device=dev, dtype=torch.int64),
                   torch.empty(bs, device=dev, dtype=torch.int32))
    if path is None:
        path = torch.empty((bs, T), device=candidates.device, dtype=torch.int32)
    if len(outputs) != 5:
        raise ValueError("Expected accept/commit/bonus/output/new_seq buffers")
    shapes = ((bs,), (bs,), (bs,), (bs, T), (bs,), (bs, T))
    dtypes = (torch.int32, torch.int32, torch.int64, torch.int64, torch.int32, torch.int32)
    for t, shape, dtype in zip((*outputs, path), shapes, dtypes):
        if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
            raise ValueError("output buffers must be contiguous (i32 [bs], i32 [bs], i64 [bs], i64 [bs, T], i32 [bs]) "
                             "and path i32 [bs, T]")
    code = _lib.dtype_code(logits)
    dev = _lib.require_cuda(candidates, parents, logits, prefix_lens, verify_lens, *outputs, path)
    lib = _lib.load()
    V = logits.shape[1]
    stride = logits.stride(0) if logits.shape[0] > 1 else V
    wbuf = (workspace or Workspace()).get(lib.dsv_tree_verify_workspace_bytes(bs * T, V), dev)
    _lib.launch("dsv_tree_verify", dev, lib.dsv_tree_verify, logits.data_ptr(), code, bs * T, V, stride, bs, T,
                candidates.data_ptr(), parents.data_ptr(), _lib.ptr(verify_lens), prefix_lens.data_ptr(),
                *(t.data_ptr() for t in outputs), path.data_ptr(), wbuf.data_ptr(), wbuf.numel())
    return outputs, path
