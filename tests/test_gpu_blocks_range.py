"""Finite keys past the index type's range, and bounds that are infinite."""

import math

import blocks_ref as B
import pytest
import torch
import tree_ref as R

pytestmark = pytest.mark.gpu
BF, HF, E4, I8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("act, dtype, unit", [(HF, E4, 400.0), (HF, I8, 2000.0), (HF, BF, 1e38), (BF, E4, 3.4e38 / 448)])
@pytest.mark.parametrize("D, size", [(16, 16), (80, 64), (128, 128)])
def test_finite_keys_past_the_types_range(device, D, size, act, dtype, unit):
    """They count as the type's largest number; a key that is itself infinite or NaN stays what it is."""
    from dspine_amd.kernels.blocks import BlockIndex, index_blocks, score_blocks, select_blocks
    from dspine_amd.kernels.cache import KVCache

    g = torch.Generator().manual_seed(D)
    blocks, H = 6, 2
    slots = blocks * size
    k, scale = torch.randn(slots, H, D, generator=g).clamp(-1, 1).to(BF), None
    big = slice(2 * size + 5, 2 * size + 7)  # two keys of block 2
    if dtype == BF:
        k[big, :, 1], k[big, :, 3] = unit, -unit
    else:
        scale = torch.full((slots, H), 1.0 / R.TOP[dtype])
        k = (k * R.TOP[dtype]).to(dtype) if dtype == E4 else (k.float() * R.TOP[dtype]).round().to(I8)
        scale[big] = unit
        raw = k.float()
        raw[big, :, 1], raw[big, :, 3] = R.TOP[dtype], -R.TOP[dtype]
        k = raw.to(dtype)
    if dtype == BF:
        k[4 * size, 0, 2], k[4 * size + 1, 1, 5] = math.inf, math.nan
    else:
        scale[4 * size, 0], scale[4 * size + 1, 1] = math.inf, math.nan
    bounds = torch.zeros(blocks, H, 2, D, dtype=act)
    args = dict(page_table=torch.arange(slots, dtype=torch.int32).view(1, -1),
                block_table=torch.arange(blocks, dtype=torch.int32).view(1, -1), from_lens=torch.zeros(1, dtype=torch.int32),
                to_lens=torch.tensor([slots], dtype=torch.int32))
    want, _ = B.index(bounds, size, k, scale, **args)
    top = torch.finfo(act).max
    want = torch.where(torch.isfinite(want), want.clamp(-top, top), want)
    tol = want.abs() * (R.half_step(act) + R.U32) * 1.01 + 2.0 ** -25
    assert bool((want[2].abs() == top).any())
    index = BlockIndex(bounds.to(device), size)
    cache = KVCache(*(x if x is None else x.to(device) for x in (k, k, scale, scale)))
    index_blocks(index, cache, **{n: x.to(device) for n, x in args.items()})
    fine = [j for j in range(blocks) if j != 4]
    R.close(index.bounds[fine], want[fine], tol[fine])
    got = index.bounds[4].double().cpu()
    if dtype == BF:
        assert float(got[0, 1, 2]) == math.inf and bool(torch.isnan(got[1, :, 5]).all())
    else:
        assert bool((got[0].abs() == math.inf).any()) and bool(torch.isnan(got[1]).all())
    # a node that such a key attracts finds its block (the one with real infinities left out of the request)
    q = torch.zeros(1, H, D)
    q[:, :, 1], q[:, :, 3], q[:, :, 0] = 0.25, -0.25, -2.0 ** -10
    table = torch.tensor([fine], dtype=torch.int32, device=device)
    pre = torch.tensor([len(fine) * size], dtype=torch.int32, device=device)
    scores = score_blocks(q.to(act).to(device), index, T=1, block_table=table, prefix_lens=pre, scale=2.0 ** -10)
    assert bool(torch.isfinite(scores).all())
    assert select_blocks(scores, 1, prefix_lens=pre, block_size=size).flatten().tolist() == [2, 2]


def _definition(q, bounds, size, *, T, block_table, prefix_lens, scale):
    """(scores, tolerance): the largest over nodes and heads of sum_d max(q_d least_d, q_d largest_d), NaN where a term is."""
    Hq, D = q.shape[1:]
    H, (bs, L) = bounds.shape[1], block_table.shape
    out = torch.full((bs, H, L), -math.inf, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(bs):
        x = q[b * T: (b + 1) * T].double().view(T, H, Hq // H, D)
        for j in range(int(prefix_lens[b]) // size):
            lo, hi = bounds[int(block_table[b, j])].double().view(1, H, 1, 2, D).unbind(3)
            term = torch.maximum(x * lo, x * hi)
            out[b, :, j] = term.sum(-1).amax((0, 2)) * scale
            mag = term.abs().sum(-1)
            tol[b, :, j] = (2 * D + 8) * R.U32 * torch.where(torch.isfinite(mag), mag, 0.0).amax((0, 2)) * scale
    return out, tol


@pytest.mark.parametrize("act", [BF, HF])
@pytest.mark.parametrize("T, H, G, D, L", [(1, 1, 1, 16, 7), (5, 3, 2, 80, 40), (17, 2, 4, 128, 300), (64, 1, 32, 64, 33), (3, 2, 5, 256, 70)])
def test_scores_of_infinite_bounds(device, T, H, G, D, L, act):
    """An element's larger product, where the other one is that of an infinity; zero queries beside one, NaN bounds, and
    infinities of both signs (whose sum is none)."""
    from dspine_amd.kernels.blocks import BlockIndex, score_blocks

    g = torch.Generator().manual_seed(D + L)
    bs, size, scale = 2, 16, 0.25
    q = torch.randn(bs * T, H * G, D, generator=g).to(act)
    q[:, :, 3] = q[:, :, 3].abs() + 0.5
    q[:, :, 4] = -q[:, :, 4].abs() - 0.5
    q[T // 2, :, 5] = 0.0
    low = torch.randn(bs * L + 2, H, D, generator=g)
    high = low + torch.rand(low.shape, generator=g)
    kinds = [  # of block i % 9 + ...: (element, least, largest)
        [], [(3, -math.inf, 1.0)], [(3, 0.5, math.inf)], [(4, -1.0, math.inf)], [(4, -math.inf, 2.0)], [(6, -math.inf, math.inf)],
        [(5, 0.0, math.inf)], [(3, -math.inf, -math.inf), (4, -math.inf, 0.0)], [(7, math.nan, math.nan), (3, -math.inf, 1.0)]]
    for i in range(bs * L):
        for d, l, h in kinds[i % len(kinds)]:
            low[i, :, d], high[i, :, d] = l, h
    low[5 % (bs * L), 0, :], high[5 % (bs * L), 0, :] = math.inf, math.inf
    bounds = torch.stack((low, high), 2).to(act)
    d = dict(T=T, block_table=torch.randperm(bs * L, generator=g).to(torch.int32).view(bs, L),
             prefix_lens=torch.tensor([L * size + 3, (L - 1) * size], dtype=torch.int32), scale=scale)
    want, tol = _definition(q, bounds, size, **d)
    assert bool(torch.isfinite(want).any()) and bool((want == math.inf).any()) and bool(torch.isnan(want).any())
    got = score_blocks(q.to(device), BlockIndex(bounds.to(device), size),
                       **{k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items()})
    R.close(got, want, tol)
