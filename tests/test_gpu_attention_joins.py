"""The join of a batch's parts on both sides of the line between its two forms (512 workgroups), and rows whose parts are many."""

import pytest
import torch
from test_gpu_blocks import _block_round, _call as _call_blocks, _check as _check_blocks
from test_gpu_tree import BF, E4, _call, _check, _gen, _round

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("bs, T, H, G, D", [(64, 3, 8, 2, 32), (65, 3, 8, 2, 32), (9, 17, 8, 8, 80), (1, 2, 2, 2, 64)])
def test_joins_on_both_sides(device, bs, T, H, G, D, dtype):
    g = _gen(bs)
    lens = torch.randint(0, 300, (bs,), generator=g).tolist()
    lens[bs // 2] = 2900  # (parts of several ranges)
    d = _round(bs + 1, bs=bs, T=T, H=H, G=G, D=D, act=BF, dtype=dtype, lens=lens, tree=True)
    _check(d, *_call(d, device))
    d = _block_round(bs + 2, count=20, size=16, bs=bs, T=T, H=H, G=G, D=D, act=BF, dtype=dtype, lens=lens, tree=True)
    _check_blocks(d, *_call_blocks(d, device))
