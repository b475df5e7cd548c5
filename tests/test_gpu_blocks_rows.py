"""Scores of blocks where some of a request's rows of q, or all of them, lie outside it: those nodes are not there."""

import math

import blocks_ref as B
import pytest
import torch
import tree_ref as R

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _want(q, bounds, size, *, T, block_table, prefix_lens, row_offsets, verify_lens=None):
    """Each request by itself over its rows that lie inside."""
    H, (bs, L) = bounds.shape[1], block_table.shape
    out = torch.full((bs, H, L), -math.inf, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(bs):
        n = T if verify_lens is None else max(0, min(T, int(verify_lens[b])))
        rows = [r for r in range(int(row_offsets[b]), int(row_offsets[b]) + n) if 0 <= r < q.shape[0]]
        if rows:
            out[b: b + 1], tol[b: b + 1] = B.scores(q[rows], bounds, size, T=len(rows), block_table=block_table[b: b + 1],
                                                    prefix_lens=prefix_lens[b: b + 1])
    return out, tol


@pytest.mark.parametrize("act, offsets", [(BF, torch.int64), (HF, torch.int32)])
@pytest.mark.parametrize("T, H, G, D", [(1, 1, 1, 16), (5, 2, 1, 80), (17, 2, 4, 128), (64, 1, 32, 64)])
def test_rows_outside_are_no_nodes(device, T, H, G, D, act, offsets):
    """Rows before the first and past the last, the ends of the offsets' range; every score is negative, so that a node of
    zeros would be the best."""
    from dspine_amd.kernels.blocks import BlockIndex, score_blocks

    g = torch.Generator().manual_seed(T)
    rows, size, L = T + 3, 16, 9
    ends = torch.iinfo(offsets)
    at = torch.tensor([0, -1, -(T // 2), 4, 3 + T // 2, rows - 1, rows, -T, ends.min, ends.max], dtype=offsets)
    bs = at.numel()
    q = (0.5 + torch.rand(rows, H * G, D, generator=g)).to(act)
    high = -0.5 - torch.rand(bs * L, H, 1, D, generator=g)
    bounds = torch.cat((high - torch.rand(high.shape, generator=g), high), 2).to(act)
    lens = torch.full((bs,), L * size, dtype=torch.int32)
    for nodes in (None, torch.tensor([max(1, T - i % 3) for i in range(bs)], dtype=torch.int32)):
        d = dict(T=T, block_table=torch.arange(bs * L, dtype=torch.int32).view(bs, L), prefix_lens=lens, row_offsets=at,
                 verify_lens=nodes)
        want, tol = _want(q, bounds, size, **d)
        assert bool((want < 0).all()) and bool(torch.isinf(want[-4:]).all())
        got = score_blocks(q.to(device), BlockIndex(bounds.to(device), size),
                           **{k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items()})
        R.close(got, want, tol)


def test_no_rows_at_all(device):
    from dspine_amd.kernels.blocks import new_block_index, score_blocks

    index = new_block_index(8, 2, 32, block_size=16, device=device)
    got = score_blocks(torch.empty(0, 4, 32, dtype=BF, device=device), index, T=3, row_offsets=torch.zeros(2, dtype=torch.int32,
                       device=device), block_table=torch.arange(8, dtype=torch.int32, device=device).view(2, 4),
                       prefix_lens=torch.full((2,), 64, dtype=torch.int32, device=device))
    assert bool((got == -math.inf).all())
