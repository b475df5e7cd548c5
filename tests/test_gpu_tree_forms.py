"""Attention over slots that hold nothing and values that are not finite, and at dims that fill no power of two, for the
rows of every form of the kernel (one 16-row tile, two, up to eight, more) and every type of cache."""

import math

import pytest
import torch
import tree_ref as R
from test_gpu_tree import BF, E4, HF, I8, _call, _check, _round

pytestmark = pytest.mark.gpu

ROWS = [(3, 2), (7, 4), (17, 4), (40, 4)]  # nodes, query heads a cache head
CACHES = [(BF, BF), (HF, HF), (BF, E4), (HF, E4), (BF, I8), (HF, I8)]


@pytest.mark.parametrize("act, dtype", CACHES)
@pytest.mark.parametrize("T, G", ROWS)
@pytest.mark.parametrize("D", [64, 192])
def test_bad_slots_in_every_place(device, D, T, G, act, dtype):
    """Slots below and past the cache (-1, INT_MIN, num_slots exactly, INT_MAX) beside good ones: in tiles of the context,
    a whole tile of them, at its end and inside the window.  What lies in slot 0 must not be met in their place."""
    d = _round(71, bs=2, T=T, H=1, G=G, D=D, act=act, dtype=dtype, lens=[300, 100], tree=True)
    t, slots = d["page_table"], d["cache"][0].shape[0]
    bad = [-1, -(2 ** 31), slots, 2 ** 31 - 1]
    for i, at in enumerate((0, 5, 31, 32, 63, 64, 100, 127)):
        t[0, at] = bad[i % 4]
    t[0, 192:256] = slots  # a tile of nothing
    t[0, 299], t[0, 301], t[0, 300 + T - 1] = slots, -1, slots
    t[1, 99], t[1, 100], t[1, 102] = -(2 ** 31), slots, 2 ** 31 - 1
    # no page names slot 0; its keys would win every softmax
    moved = int(torch.tensor(sorted(set(range(slots)) - set(t.flatten().tolist())))[-1])
    t[t == 0] = moved
    for x in d["cache"]:
        if x is not None:
            x[moved] = x[0]
    k, v, ks, vs = d["cache"]
    if ks is None:
        k[0], v[0] = math.nan, math.nan
    else:
        ks[0], vs[0] = math.nan, math.nan
    _check(d, *_call(d, device))


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("T, G", ROWS)
def test_a_table_that_ends_in_the_window_or_before_it(device, T, G, dtype):
    d = _round(72, bs=4, T=T, H=2, G=G, D=64, act=BF, dtype=dtype, lens=[70, 69, 300, 0], tree=True)
    d["page_table"] = d["page_table"][:, :71].contiguous()
    _check(d, *_call(d, device))


def _alone(d, T):
    """Each node sees the context, itself and node 0."""
    d["masks"] = torch.tensor([[R.signed(1 | 1 << i) for i in range(T)]] * d["prefix_lens"].numel(), dtype=torch.int64)


def _compare(d, out, lse, hurt):
    """Rows not hurt equal the reference; ``hurt`` [bs, T, ...] names the nodes that see what is not finite."""
    args = {n: x for n, x in d.items() if n not in ("q", "cache")}
    want, wl, otol, ltol = R.attention(d["q"], *d["cache"], **args)
    fine = ~hurt.flatten()
    assert bool(torch.isfinite(out.cpu()[fine]).all()) and bool(torch.isfinite(lse.cpu()[fine]).all())
    R.close(out.cpu()[fine], want[fine], otol[fine])
    R.close(lse.cpu()[fine], wl[fine], ltol[fine])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T, G", [(7, 2), *ROWS[1:]])
@pytest.mark.parametrize("D", [64, 192])
def test_what_is_not_finite_stays_with_the_nodes_that_see_it(device, D, T, G, dtype):
    d = _round(73, bs=2, T=T, H=1, G=G, D=D, act=dtype, dtype=dtype, lens=[150, 61], tree=False)
    _alone(d, T)
    k, v = d["cache"][:2]
    at = d["page_table"].long()
    v[at[0, 150 + 2], 0, 5] = math.nan
    v[at[0, 150 + 3], 0, 6] = math.inf
    v[at[0, 150 + 4], 0, D - 1] = -math.inf
    k[at[0, 150 + 5], 0, 8] = math.nan
    v[at[1, 61 + 6], 0, :] = math.nan
    free = sorted(set(range(k.shape[0])) - set(at.flatten().tolist()))
    k[free], v[free] = math.nan, math.inf
    out, lse = _call(d, device)
    hurt = torch.zeros(2, T, dtype=torch.bool)
    hurt[0, 2:6], hurt[1, 6] = True, True
    _compare(d, out, lse, hurt)
    o = out.cpu().view(2, T, G, D)
    assert bool(torch.isnan(o[0, 2, :, 5]).all()) and bool((o[0, 3, :, 6] == math.inf).all())
    assert bool((o[0, 4, :, D - 1] == -math.inf).all()) and bool(torch.isnan(o[0, 5]).all()) and bool(torch.isnan(o[1, 6]).all())
    rest = torch.arange(D)
    assert bool(torch.isfinite(o[0, 2][:, rest != 5]).all()) and bool(torch.isfinite(o[0, 3][:, rest != 6]).all())


@pytest.mark.parametrize("act, dtype", CACHES[2:])
@pytest.mark.parametrize("T, G", [(7, 2), *ROWS[1:]])
@pytest.mark.parametrize("D", [64, 192])
def test_a_poisoned_row_stays_with_the_nodes_that_see_it(device, D, T, G, act, dtype):
    """Scales of NaN and infinity and an e4m3 code that is NaN, in the window."""
    d = _round(74, bs=2, T=T, H=1, G=G, D=D, act=act, dtype=dtype, lens=[150, 61], tree=False)
    _alone(d, T)
    k, v, ks, vs = d["cache"]
    at = d["page_table"].long()
    vs[at[0, 150 + 2]] = math.nan
    ks[at[0, 150 + 3]] = math.nan
    vs[at[0, 150 + 4]] = math.inf
    hurt = torch.zeros(2, T, dtype=torch.bool)
    hurt[0, 2:5] = True
    if dtype == E4:
        v.view(torch.uint8)[at[1, 61 + 5], 0, 3] = 0x7F
        v.view(torch.uint8)[at[1, 61 + 6], 0, D - 1] = 0xFF
        hurt[1, 5:7] = True
    out, lse = _call(d, device)
    _compare(d, out, lse, hurt)
    o = out.cpu().view(2, T, G, D)
    assert bool(torch.isnan(o[0, 2]).all()) and bool(torch.isnan(o[0, 3]).all()) and not bool(torch.isfinite(o[0, 4]).any())
    if dtype == E4:
        assert bool(torch.isnan(o[1, 5, :, 3]).all()) and bool(torch.isnan(o[1, 6, :, D - 1]).all())
        assert bool(torch.isfinite(o[1, 5, :, 4:]).all()) and bool(torch.isfinite(o[1, 6, :, : D - 1]).all())


@pytest.mark.parametrize("act, dtype", CACHES)
@pytest.mark.parametrize("T, G", ROWS[2:])
@pytest.mark.parametrize("D", [16, 48, 80, 112, 144, 240])
def test_dims_between(device, D, T, G, act, dtype):
    d = _round(75 + D, bs=2, T=T, H=2, G=G, D=D, act=act, dtype=dtype, lens=[200, 37], tree=True)
    _check(d, *_call(d, device))
