"""Calls of the block operators as the documentation allows them: a chain's drafts that choose each for itself, a prompt's
queries in groups, another stream, caches with the heads outside, workspaces shared by graphs, the largest head groups."""

import blocks_ref as B
import pytest
import torch
import tree_ref as R
from test_gpu_blocks import _block_round, _call, _check, _score_call, _score_round
from test_gpu_tree import BF, E4, HF, I8, _gen, _round, _to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, I8])
def test_drafts_that_choose_each_for_itself(device, dtype):
    """A chain of drafts as requests of one node over one table row: each sees its own blocks and the drafts before it."""
    from dspine_amd.kernels.blocks import block_attention, index_blocks, new_block_index, score_blocks, select_blocks

    T, H, G, D, size, n = 9, 2, 4, 64, 16, 333
    d = _round(31, bs=1, T=T, H=H, G=G, D=D, act=BF, dtype=dtype, lens=[n], tree=False)
    cache, q = _to(d["cache"], device), d["q"].to(device)
    table = d["page_table"].to(device)
    pre = n + torch.arange(T, dtype=torch.int32, device=device)
    index = new_block_index(30, H, D, block_size=size, device=device)
    rows = torch.arange(30, dtype=torch.int32, device=device).flip(0).view(1, -1)
    # (the longest of them has all the blocks that any has)
    index_blocks(index, cache, page_table=table, block_table=rows, from_lens=pre[:1] * 0, to_lens=pre[-1:])
    pages, blocks_of = table.expand(T, -1), rows.expand(T, -1)
    scores = score_blocks(q, index, T=1, block_table=blocks_of, prefix_lens=pre)
    blocks = select_blocks(scores, 5, prefix_lens=pre, block_size=size, last=1)
    out = block_attention(q, cache, T=1, blocks=blocks, block_size=size, page_table=pages, prefix_lens=pre)
    want, tol = B.scores(d["q"], index.bounds.cpu(), size, T=1, block_table=blocks_of.cpu(), prefix_lens=pre.cpu())
    R.close(scores, want, tol)
    args = dict(T=1, blocks=blocks.cpu(), block_size=size, page_table=pages.cpu(), prefix_lens=pre.cpu())
    assert torch.equal(args["blocks"], B.select(scores.cpu(), 5, prefix_lens=pre.cpu(), block_size=size, last=1))
    assert len({tuple(x) for x in args["blocks"][:, 0].tolist()}) > 1  # (they do choose)
    o, _, otol, _ = B.attention(d["q"], *d["cache"], **args)
    R.close(out, o, otol)


@pytest.mark.parametrize("dtype", [BF, E4])
def test_a_prompt_in_groups_of_queries(device, dtype):
    """64 queries a request over one table row, every finished block selected: causal attention of the whole prompt."""
    from dspine_amd.kernels.blocks import block_attention

    n, T, H, G, D, size = 301, 64, 2, 2, 64, 32
    d = _round(32, bs=1, T=1, H=H, G=G, D=D, act=BF, dtype=dtype, lens=[n - 1], tree=False)
    groups = -(-n // T)
    g = _gen(33)
    q = torch.randn(n, H * G, D, generator=g).to(BF)
    start = torch.arange(groups, dtype=torch.int32) * T
    held = torch.clamp(n - start, max=T)
    count = n // size + 1
    blocks = torch.arange(count, dtype=torch.int32).expand(groups, H, -1).contiguous()
    lse = torch.empty(n, H * G, device=device)
    out = block_attention(q.to(device), _to(d["cache"], device), T=T, blocks=blocks.to(device), block_size=size,
                          page_table=d["page_table"].to(device).expand(groups, -1), prefix_lens=start.to(device),
                          verify_lens=held.to(device), row_offsets=start.to(device), lse=lse)
    k, v, ks, vs = d["cache"]
    for i in (0, 1, 63, 64, 100, 191, 299, 300):
        want, wl, otol, ltol = R.attention(q[i: i + 1], k, v, ks, vs, T=1, page_table=d["page_table"],
                                           prefix_lens=torch.tensor([i], dtype=torch.int32))
        R.close(out[i: i + 1], want, otol)
        R.close(lse[i: i + 1], wl, ltol)


@pytest.mark.parametrize("T, G", [(2, 3), (17, 4)])
@pytest.mark.parametrize("act, dtype", [(BF, BF), (HF, E4), (BF, I8)])
def test_heads_as_the_outer_dimension(device, act, dtype, T, G):
    """Caches whose heads lie far apart, scales too, and a page table that is a slice of a wider one."""
    from dspine_amd.kernels.blocks import block_attention, index_blocks, new_block_index
    from dspine_amd.kernels.cache import KVCache

    d = _block_round(34, count=4, size=16, bs=2, T=T, H=3, G=G, D=48, act=act, dtype=dtype, lens=[200, 70], tree=True)

    def outer(t):
        if t is None:
            return None
        raw = t.view(torch.uint8) if t.dtype == E4 else t
        raw = raw.transpose(0, 1).contiguous().to(device).transpose(0, 1)
        return raw.view(t.dtype) if t.dtype == E4 else raw

    cache = KVCache(*(outer(t) for t in d["cache"]))
    wide = torch.full((2, d["page_table"].shape[1] + 9), -1, dtype=torch.int32, device=device)
    table = wide[:, 5: 5 + d["page_table"].shape[1]]
    table.copy_(d["page_table"])
    lse = torch.full(d["q"].shape[:2], 7.0, device=device)
    args = {k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items() if k not in ("q", "cache", "page_table")}
    out = block_attention(d["q"].to(device), cache, page_table=table, lse=lse, **args)
    _check(d, out, lse)
    index = new_block_index(40, 3, 48, block_size=16, dtype=act, device=device)
    rows = torch.arange(40, dtype=torch.int32).view(2, 20)
    lens = dict(from_lens=torch.zeros(2, dtype=torch.int32), to_lens=d["prefix_lens"])
    want, tol = B.index(index.bounds.cpu(), 16, d["cache"][0], d["cache"][2], page_table=d["page_table"], block_table=rows, **lens)
    index_blocks(index, cache, page_table=table, block_table=rows.to(device), **{k: x.to(device) for k, x in lens.items()})
    R.close(index.bounds, want, tol)


def test_on_another_stream(device):
    """Inputs made on a side stream and used there, while the default stream is busy."""
    d = _block_round(35, count=3, size=16, bs=2, T=5, H=2, G=4, D=64, act=BF, dtype=E4, lens=[130, 60], tree=True)
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device=device)
    for _ in range(3):
        busy = busy @ busy * 1e-2
    with torch.cuda.stream(side):
        out, lse = _call(d, device)
    side.synchronize()
    _check(d, out, lse)


@pytest.mark.parametrize("T, G, D", [(64, 32, 64), (1, 128, 128), (33, 24, 256)])
def test_scores_of_many_heads(device, T, G, D):
    """More query rows than LDS holds at once: they are taken in turns."""
    q, bounds, d = _score_round(36, bs=2, T=T, H=1, G=G, D=D, size=16, act=BF, lens=[700, 3], nodes=[T, 1])
    want, tol = B.scores(q, bounds, 16, **d)
    R.close(_score_call(device, q, bounds, 16, d), want, tol)


def test_graphs_that_share_a_workspace(device):
    """Two captured calls on one workspace, replayed in turn while lists and lengths change, eager calls between them."""
    from dspine_amd.kernels.blocks import block_attention
    from dspine_amd.verify import Workspace

    work, calls = Workspace(), []
    for i, (bs, T, D, dtype) in enumerate([(2, 9, 128, BF), (70, 1, 64, E4)]):
        d = _block_round(37 + i, count=6, size=16, bs=bs, T=T, H=2, G=4, D=D, act=BF, dtype=dtype, lens=[400] * bs, tree=False)
        calls.append({k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items() if k != "cache"}
                     | dict(cache=_to(d["cache"], device)))
    work.get(1 << 26, torch.device(device))
    side, graphs = torch.cuda.Stream(), []
    for a in calls:
        with torch.cuda.stream(side):
            block_attention(**a, workspace=work)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block_attention(**a, workspace=work)
        graphs.append((graph, out, a))
    for turn in range(4):
        for graph, out, a in graphs:
            a["prefix_lens"].copy_((torch.arange(a["prefix_lens"].numel()) * 53 + 131 * turn) % 400)
            a["blocks"].copy_((a["blocks"] + 5 * turn) % 25)
            graph.replay()
            got = out.clone()
            want = block_attention(**a, workspace=work)
            assert torch.equal(got, want) and torch.equal(block_attention(**a), want)
