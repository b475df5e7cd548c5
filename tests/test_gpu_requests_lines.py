"""Requests that end on both sides of what one workgroup takes (64 rows, 2048 columns of groups of eight, 8192 entries, 16384
slots), rows named again in every group."""

import blocks_ref as B
import pytest
import torch
from test_gpu_requests import _ids, _pool
from test_gpu_tree import _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [16384, 16385])
@pytest.mark.parametrize("rows, cols", [(64, 128), (64, 129), (65, 100), (1, 2048), (1, 2049), (9, 910), (9, 911), (16, 512), (17, 500)])
def test_ends_on_both_sides(device, rows, cols, slots):
    from dspine_amd.runtime.requests import free_requests

    g = _gen(rows * cols)
    lens = torch.randint(0, cols + 1, (rows,), generator=g).tolist()
    lens[0] = cols
    lend = [(i, i + 1, min(lens[i], lens[i + 1]) // 2) for i in range(0, rows - 1, 2)]
    table, full, shared = _pool(rows, rows=rows + 2, cols=cols, slots=slots, lens=lens, lend=lend)
    t, n, s = (x.to(device) for x in (table, full, shared))
    dead = torch.randint(-1, rows + 3, (rows,), generator=g).tolist()
    for what in (dead, [*range(rows), 0][:rows]):
        got, count = free_requests(t, n, s, _ids(device, what, torch.int64))
        want = B.free(table, full, shared, what)
        assert int(count) == len(want) and got[: len(want)].tolist() == want
        assert torch.equal(n.cpu(), full) and torch.equal(s.cpu(), shared)
    assert not bool(s.any()) and not bool(n.any())
