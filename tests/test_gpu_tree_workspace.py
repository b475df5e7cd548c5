"""Captured calls on one workspace that larger calls outgrow after the capture."""

import pytest
import torch
from test_gpu_tree import BF, E4, _round, _to

pytestmark = pytest.mark.gpu


def _args(device, seed, **shape):
    d = _round(seed, act=BF, dtype=E4, tree=False, **shape)
    return dict(q=d["q"].to(device), cache=_to(d["cache"], device), T=d["T"], page_table=d["page_table"].to(device),
                prefix_lens=d["prefix_lens"].to(device))


def test_a_graph_outlives_its_workspaces_growth(device):
    """A small attention and a small acceptance are captured on a workspace that starts empty, larger calls outgrow it, and
    what is allocated afterwards keeps its values through the replays."""
    from dspine_amd.kernels.attention import tree_attention
    from dspine_amd.verification.tree import accept_greedy_tree
    from dspine_amd.verify import Workspace

    small = _args(device, 61, bs=2, T=3, H=2, G=2, D=64, lens=[900, 300])
    large = _args(device, 62, bs=4, T=40, H=2, G=8, D=128, lens=[700, 80, 9, 300])
    g = torch.Generator(device=device).manual_seed(63)
    tree = dict(candidates=torch.randint(0, 900, (2, 3), generator=g, device=device),
                parents=torch.tensor([[-1, 0, 1]] * 2, dtype=torch.int32, device=device),
                next_token_logits=torch.randn(6, 900, generator=g, device=device),
                prefix_lens=torch.zeros(2, dtype=torch.int32, device=device))

    def both(work):
        outs, path = accept_greedy_tree(workspace=work, **tree)
        return [tree_attention(workspace=work, **small), *outs, path]

    work, side = Workspace(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        both(Workspace())  # (warm-up, on scratch of its own)
    torch.cuda.synchronize()
    want = [t.clone() for t in both(Workspace())]
    held = both(work)  # the buffer that the graph is given: not one of its own pool
    first = work.buf
    at, size = first.data_ptr(), first.numel()
    del first
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(work)
    assert work.buf.data_ptr() == at
    big = tree_attention(workspace=work, **large)
    assert work.buf.data_ptr() != at
    torch.cuda.synchronize()
    fill = [torch.full((size,), 0x5A, dtype=torch.uint8, device=device) for _ in range(8)]
    assert all(t.data_ptr() + size <= at or at + size <= t.data_ptr() for t in fill)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)
        assert all(bool((t == 0x5A).all()) for t in fill)
        assert torch.equal(tree_attention(workspace=work, **large), big)
