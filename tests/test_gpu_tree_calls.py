"""Calls of the tree attention as a serving loop makes them: one table row for several requests, graphs that share a
workspace, lengths that change under a captured call, an empty batch of nodes."""

import pytest
import torch
from test_gpu_tree import BF, E4, _call, _check, _round, _to

pytestmark = pytest.mark.gpu


def test_requests_of_one_table_row(device):
    """Forks of one context: the same (expanded) row of the page table, different lengths and trees."""
    d = _round(41, bs=1, T=6, H=2, G=4, D=128, act=BF, dtype=E4, lens=[500], tree=False)
    g = torch.Generator().manual_seed(42)
    d["q"] = torch.randn(3 * 6, 8, 128, generator=g).to(BF)
    d["prefix_lens"] = torch.tensor([500, 130, 0], dtype=torch.int32)
    d["masks"] = torch.randint(0, 64, (3, 6), generator=g)
    d["page_table"] = d["page_table"].expand(3, -1)
    table = d["page_table"][:1].to(device).expand(3, -1)
    assert table.stride(0) == 0
    _check(d, *_call(d, device, page_table=table))


def test_no_request_has_nodes(device):
    d = _round(43, bs=3, T=4, H=1, G=2, D=64, act=BF, dtype=BF, lens=[9, 0, 70], tree=False, nodes=[0, 0, -3])
    out, lse = _call(d, device)
    assert bool((out == 7).all()) and bool((lse == 7).all())


def test_graphs_that_share_a_workspace(device):
    """Two captured calls of different shapes on one workspace, replayed in turn while their lengths change and eager
    calls use it between: each replay equals an eager call of its own."""
    from dspine_amd.kernels.attention import tree_attention
    from dspine_amd.verify import Workspace

    shapes = [dict(bs=2, T=9, H=2, G=4, D=128, lens=[900, 300]), dict(bs=70, T=1, H=2, G=4, D=64, lens=[200] * 70)]
    work, calls = Workspace(), []
    for i, shape in enumerate(shapes):
        d = _round(44 + i, act=BF, dtype=E4, tree=False, **shape)
        a = dict(q=d["q"].to(device), cache=_to(d["cache"], device), T=d["T"], page_table=d["page_table"].to(device),
                 prefix_lens=d["prefix_lens"].to(device))
        calls.append(a)
    work.get(1 << 26, torch.device(device))  # (large enough for both: a graph keeps the address)
    side = torch.cuda.Stream()
    graphs = []
    for a in calls:
        with torch.cuda.stream(side):
            tree_attention(**a, workspace=work)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = tree_attention(**a, workspace=work)
        graphs.append((graph, out, a))
    for turn in range(4):
        for graph, out, a in graphs:
            most = a["page_table"].shape[1] - a["T"]
            a["prefix_lens"].copy_((torch.arange(a["prefix_lens"].numel()) * 37 + 97 * turn) % (most + 1))
            graph.replay()
            got = out.clone()
            want = tree_attention(**a, workspace=work)  # (behind the replay, on its stream)
            assert torch.equal(got, want) and torch.equal(tree_attention(**a), want)
