"""Finite keys past the index type's range."""

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
