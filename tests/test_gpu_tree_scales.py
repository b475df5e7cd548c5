"""Attention over a quantised cache whose value scales lie far apart, against tests/tree_ref.py."""

import pytest
import torch
import tree_ref as R
from test_gpu_tree import BF, E4, I8, _call, _check, _round

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", [(3, 2), (7, 4), (17, 4), (40, 4)])  # rows of every form
@pytest.mark.parametrize("power", [-90, -40, 40, 90])
def test_scales_of_any_size(device, power, T, G, dtype):
    d = _round(31, bs=2, T=T, H=2, G=G, D=64, act=BF, dtype=dtype, lens=[150, 77], tree=True)
    d["cache"][3].mul_(2.0 ** power)
    _check(d, *_call(d, device))


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", [(3, 2), (7, 4), (17, 4), (40, 4)])
@pytest.mark.parametrize("power", [20, 60, 110])
def test_a_large_scale_stays_with_the_nodes_that_see_it(device, power, T, G, dtype):
    """Node 1's values are 2^power above the others': it is a leaf, so no other node's row may lose a bit to it."""
    d = _round(32, bs=2, T=T, H=2, G=G, D=64, act=BF, dtype=dtype, lens=[150, 60], tree=False)
    masks = torch.zeros((2, T), dtype=torch.int64)
    for i in range(T):
        masks[:, i] = R.signed(1 | 1 << i)
    d["masks"] = masks
    for b, n in enumerate((150, 60)):
        d["cache"][3][d["page_table"][b, n + 1].long()] *= 2.0 ** power
    _check(d, *_call(d, device))


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", [(3, 2), (7, 4), (17, 4)])
def test_scales_far_apart_in_a_context(device, T, G, dtype):
    """Positions of scale 2^-90, 1 and 2^90 in one context, in parts of their own and side by side: the sum of the
    weights, and so lse, is whole, the output that of the largest."""
    d = _round(33, bs=2, T=T, H=2, G=G, D=64, act=BF, dtype=dtype, lens=[700, 200], tree=True)
    at = d["page_table"][0].long()
    d["cache"][3][at[:200]] *= 2.0 ** -90
    d["cache"][3][at[400:500]] *= 2.0 ** 90
    at = d["page_table"][1].long()
    d["cache"][3][at[5:200:3]] *= 2.0 ** 90
    _check(d, *_call(d, device))
