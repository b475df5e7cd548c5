"""The commit of a path in its own order: slots are moved inside the table in any order, entries that name no node of the
window or a node named before are left out."""

import pytest
import torch
import tree_ref as R

pytestmark = pytest.mark.gpu


def _commit(device, path, accept, lens, prefix, rows, table, ocl):
    from dspine_amd.runtime.worker import commit_accept

    bs, T = path.shape
    d_table, d_seq = table.to(device), torch.zeros(table.shape[0], dtype=torch.int32, device=device)
    outs = (accept.to(device), None, None, torch.empty((bs, T), device=device, dtype=torch.int64), None)
    free, count = commit_accept(outs, prefix_lens=prefix.to(device), req_pool_indices=rows.to(device), req_to_token=d_table,
                                out_cache_loc=None if ocl is None else ocl.to(device), verify_lens=lens.to(device),
                                seq_lens=d_seq, path=path.to(device))
    return free[: int(count.item())].tolist(), d_table.tolist(), d_seq.tolist()


@pytest.mark.parametrize("in_table", [True, False])
@pytest.mark.parametrize("bs, T", [(1, 2), (37, 17), (1300, 64)])
def test_commit_keeps_the_order_of_the_path(device, bs, T, in_table):
    g = torch.Generator().manual_seed(bs)
    lens = torch.randint(1, T + 1, (bs,), generator=g, dtype=torch.int64).to(torch.int32)
    lens[0] = T
    path = torch.full((bs, T), -1, dtype=torch.int32)
    accept = torch.zeros(bs, dtype=torch.int32)
    for b, n in enumerate(lens.tolist()):
        some = torch.randperm(n, generator=g)[: int(torch.randint(1, n + 1, (1,), generator=g))]
        path[b, : some.numel()], accept[b] = some, some.numel() - 1
    path[0, :2], accept[0] = torch.tensor([1, 0], dtype=torch.int32), 1  # (two nodes change places)
    prefix = torch.randint(0, 100, (bs,), generator=g)
    table = torch.randint(0, 1 << 20, (bs + 3, 140), generator=g, dtype=torch.int64).to(torch.int32)
    rows = torch.randperm(bs + 3, generator=g)[:bs]
    ocl = None if in_table else torch.randperm(1 << 20, generator=g)[: bs * T]
    ref, seq = table.tolist(), [0] * (bs + 3)
    freed = R.commit_tree(accept.tolist(), path.tolist(), prefix.tolist(), rows.tolist(), ref, T,
                          out_cache_loc=None if in_table else ocl.tolist(), verify_lens=lens.tolist(), seq_lens=seq)
    assert _commit(device, path, accept, lens, prefix, rows, table, ocl) == (freed, ref, seq)


def test_commit_leaves_out_entries_that_name_nothing_new(device):
    lens, accept = torch.tensor([5, 4], dtype=torch.int32), torch.tensor([4, 2], dtype=torch.int32)
    path = torch.tensor([[0, 3, 0, 5, 1], [-1, 4, 64, 2, 1]], dtype=torch.int32)  # node 5 lies past request 0, 4 past request 1
    table = torch.arange(2 * 12, dtype=torch.int32).view(2, 12) + 100
    got = _commit(device, path, accept, lens, torch.tensor([2, 6]), torch.tensor([1, 0]), table, None)
    ref = table.tolist()
    old = list(ref[1])
    ref[1][2:5] = [old[2], old[5], old[3]]
    assert got == ([old[4], old[6], *ref[0][6:10]], ref, [6, 5])
