"""The long-context and request calls as the user's guide writes them: its own lines are run."""

import pathlib

import pytest
import torch
import tree_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _example(*calls):
    """The guide's Python lines that make all of these calls."""
    texts = [p.read_text() for p in sorted(pathlib.Path(__file__).resolve().parents[1].glob("*.md"))]
    found = [block.split("```")[0] for text in texts for block in text.split("```python\n")[1:]]
    found = [block for block in found if all(f"{c}(" in block for c in calls)]
    assert len(found) == 1
    return found[0]


@pytest.mark.parametrize("lens_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows, pool", [(7, [5, 0, 2]), (3, [2, 0, 1])])
def test_a_long_contexts_round(device, rows, pool, lens_dtype):
    """A forked request among them; the accepted path leaves nodes out and crosses, reaches or misses a block's end.  The
    bounds of what was finished are those of the committed positions' keys."""
    from dspine_amd.kernels.cache import KVCache
    from dspine_amd.runtime.requests import fork_requests

    g = torch.Generator().manual_seed(rows)
    T, H, G, D, size, bs = 6, 2, 3, 64, 64, 3
    lens = [62, 125, 190]
    path = torch.tensor([[0, 2, 5, -1, -1, -1], [0, 1, 4, -1, -1, -1], [0, 3, -1, -1, -1, -1]], dtype=torch.int32)
    accept = torch.tensor([2, 2, 1], dtype=torch.int32)
    cols, slots = 220, 900
    perm = torch.randperm(slots, generator=g).to(torch.int32)
    table = torch.zeros(rows, cols, dtype=torch.int32)
    seq_lens = torch.zeros(rows, dtype=lens_dtype)
    at = 0
    for b, n in enumerate(lens):
        table[pool[b], :n] = perm[at: at + n]
        seq_lens[pool[b]] = n
        at += n
    req_to_token, seq_lens = table.to(device), seq_lens.to(device)
    shared = torch.zeros(slots, dtype=torch.int32, device=device)
    if rows > 3:  # request 1 is forked from row 6
        req_to_token[6, :125] = req_to_token[pool[1], :125]
        seq_lens[6] = 125
        seq_lens[pool[1]] = 0
        fork_requests(req_to_token, seq_lens, shared, torch.tensor([6], device=device), torch.tensor([pool[1]], device=device))
    for b, n in enumerate(lens):  # the window's slots
        req_to_token[pool[b], n: n + T] = perm[at: at + T].to(device)
        at += T
    cache = KVCache(*(torch.randn(slots, H, D, generator=g).to(BF).to(device) for _ in range(2)))
    parents = torch.tensor([[-1, 0, 0, 0, 1, 2]] * bs, dtype=torch.int32)
    masks = torch.tensor([[R.signed(m) for m in row] for row in R.tree_masks(parents)[0]], dtype=torch.int64)
    per = cols // size + 1
    state = dict(torch=torch, num_blocks=bs * per, kv_heads=H, head_dim=D, T=T, cache=cache, req_to_token=req_to_token,
                 seq_lens=seq_lens, pool=torch.tensor(pool, device=device), masks=masks.to(device), path=path.to(device),
                 q=torch.randn(bs * T, H * G, D, generator=g).to(BF).to(device),
                 prefix_lens=torch.tensor(lens, dtype=torch.int32, device=device),
                 block_table=torch.randperm(bs * per, generator=g).view(bs, per).to(torch.int32).to(device),
                 outs=(accept.to(device), None, None, torch.zeros(bs, T, dtype=torch.int64, device=device), None))
    state["page_table"] = req_to_token[state["pool"]]
    before = req_to_token.cpu()
    exec(_example("score_blocks", "select_blocks", "block_attention", "index_blocks"), state)
    bounds, k = state["index"].bounds.cpu(), cache.k.cpu()
    assert bounds.shape[0] == bs * per and not bool(torch.isnan(state["o"]).any())
    done = 0
    for b, n in enumerate(lens):
        committed = before[pool[b], :n].tolist() + [int(before[pool[b], n + i]) for i in path[b].tolist() if i >= 0]
        for j in range(per):
            row = bounds[int(state["block_table"][b, j])]
            if n // size <= j < len(committed) // size:
                keys = k[torch.tensor(committed[j * size: (j + 1) * size])]
                assert torch.equal(row[:, 0], keys.amin(0)) and torch.equal(row[:, 1], keys.amax(0))
                done += 1
            else:
                assert not bool(row.any())
    assert done == 3 and req_to_token[pool[0], 62:65].tolist() == before[pool[0], [62, 64, 67]].tolist()


def test_requests_that_share_slots(device):
    """Forked, ended and compacted; a row of its own holds the slots that no request may be given, and they stay or move
    with what lies in them."""
    from dspine_amd.kernels.cache import KVCache

    g = torch.Generator().manual_seed(5)
    slots, cols, H, D = 300, 90, 2, 32
    perm = 2 + torch.randperm(slots - 3, generator=g).to(torch.int32)
    table = torch.zeros(8, cols, dtype=torch.int32)
    lens = torch.tensor([40, 55, 0, 0, 0, 0, 0, 3], dtype=torch.int32)
    table[0, :40], table[1, :55] = perm[:40], perm[40:95]
    table[7, :3] = torch.tensor([0, 1, slots - 1])  # padding's slots and one that somebody outside reads
    first = [torch.randn(slots, H, D, generator=g).to(BF).to(device) for _ in range(4)]
    caches = [KVCache(first[0].clone(), first[1].clone()), KVCache(first[2].clone(), first[3].clone())]
    state = dict(torch=torch, num_slots=slots, caches=caches, req_to_token=table.to(device), seq_lens=lens.to(device),
                 parents=torch.tensor([0, 0, 1], device=device), children=torch.tensor([2, 3, 4], device=device),
                 rows=torch.tensor([0, 1, 3], device=device), live_rows=torch.tensor([2, 4, 7], device=device))
    exec(_example("fork_requests", "free_requests", "compact_requests"), state)
    t = state["req_to_token"]
    assert state["seq_lens"].tolist() == [0, 0, 40, 0, 55, 0, 0, 3] and int(state["free_count"]) == 0
    assert state["counts"].tolist()[0] == 40 + 55 + 3 and not bool(state["shared"].any())
    held = torch.cat((t[2, :40], t[4, :55], t[7, :3])).long()
    assert sorted(held.tolist()) == list(range(98)) and t[7, :2].tolist() == [0, 1]
    old = torch.cat((perm[:95], table[7, :3])).long().to(device)
    for cache, (k, v) in zip(caches, (first[:2], first[2:])):
        assert torch.equal(cache.k[held], k[old]) and torch.equal(cache.v[held], v[old])
