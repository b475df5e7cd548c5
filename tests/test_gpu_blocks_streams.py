"""The block and request calls on a side stream: inputs that are made there, late, while the default stream is busy.  A
launch on any other stream would find the inputs of before, or leave the outputs as they were when they are read.  (Outputs
and scratch memory are given: an allocation may wait for the device.)"""

import blocks_ref as B
import pytest
import torch
import tree_ref as R
from test_gpu_blocks import _block_round, _score_round
from test_gpu_requests import _pool
from test_gpu_tree import BF, E4, _gen, _to

pytestmark = pytest.mark.gpu


def _keep_busy(a, out, n):
    """Event at the end of n long kernels on the current stream."""
    for _ in range(n):
        torch.mm(a, a, out=out)
    event = torch.cuda.Event()
    event.record()
    return event


@pytest.fixture(scope="module")
def beside():
    """(a stream whose work ends while the default one's goes on, a matrix whose square takes about a millisecond): streams
    share a few hardware queues, and one that shares the default's would wait for it."""
    a = torch.randn(8192, 8192, device="cuda").to(BF)
    out = torch.empty_like(a)
    _keep_busy(a, out, 1)
    for _ in range(8):
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        busy = _keep_busy(a, out, 30)
        with torch.cuda.stream(side):
            torch.zeros(1, device="cuda").cpu()
        if not busy.query():
            torch.cuda.synchronize()
            return side, a
    pytest.skip("no stream runs beside the default one")


def _run(beside, call, outputs, late):
    """``call()``'s outputs on the host, from a side stream on which the tensors of ``late`` (pairs with their values;
    zeros until then) are filled in behind a long kernel; the default stream works on until the outputs are read."""
    side, a = beside
    late = [(t, x.to(a.device)) for t, x in late]
    out, own = torch.empty_like(a), torch.empty_like(a)
    call()  # (the code is loaded)
    for n in (120, 400, 1200):  # (longer, should the host have been slower)
        for t in (*outputs, *(t for t, _ in late)):
            t.zero_()
        torch.cuda.synchronize()
        busy = _keep_busy(a, out, n)
        with torch.cuda.stream(side):
            _keep_busy(a, own, 8)
            for t, x in late:
                t.copy_(x)
            call()
            got = [x.cpu() for x in outputs]  # (waits for the side stream alone)
            beside_it = not busy.query()
        torch.cuda.synchronize()
        if beside_it:
            return got
    pytest.fail("the call or its outputs waited for the default stream")


def test_index(device, beside):
    from dspine_amd.kernels.blocks import BlockIndex, index_blocks
    from dspine_amd.kernels.cache import new_cache

    slots, H, D, size = 96, 2, 32, 16
    cache = new_cache(slots, H, D, dtype=BF, device=device)
    k = torch.randn(slots, H, D, generator=_gen(1)).to(BF)
    index = BlockIndex(torch.zeros(6, H, 2, D, dtype=BF, device=device), size)
    one = torch.zeros(1, dtype=torch.int32, device=device)
    full = one + slots
    table, rows = (torch.arange(n, dtype=torch.int32, device=device).view(1, -1) for n in (slots, 6))

    got, = _run(beside, lambda: index_blocks(index, cache, page_table=table, block_table=rows, from_lens=one, to_lens=full),
                [index.bounds], [(cache.k, k)])
    k = k.view(6, size, H, D)
    assert torch.equal(got, torch.stack((k.amin(1), k.amax(1)), 2))


def test_scores_and_selection(device, beside):
    from dspine_amd.kernels.blocks import BlockIndex, score_blocks, select_blocks

    q, bounds, d = _score_round(3, bs=2, T=3, H=2, G=2, D=64, size=16, act=BF, lens=[300, 90])
    at = {k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items()}
    gq, index = torch.zeros_like(q, device=device), BlockIndex(bounds.to(device), 16)
    scores = torch.zeros(2, 2, d["block_table"].shape[1], device=device)
    got, = _run(beside, lambda: score_blocks(gq, index, out=scores, **at), [scores], [(gq, q)])
    want, tol = B.scores(q, bounds, 16, **d)
    R.close(got, want, tol)
    args = dict(prefix_lens=d["prefix_lens"], block_size=16, first=1, last=1)
    blocks, late = torch.zeros(2, 2, 6, dtype=torch.int32, device=device), torch.zeros_like(scores)
    picked, = _run(beside, lambda: select_blocks(late, 6, out=blocks, **{**args, "prefix_lens": at["prefix_lens"]}), [blocks],
                   [(late, got)])
    assert torch.equal(picked, B.select(got, 6, **args))


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention(device, beside, dtype):
    from dspine_amd.kernels.blocks import block_attention
    from dspine_amd.verify import Workspace

    d, work = _block_round(35, count=3, size=16, bs=2, T=5, H=2, G=4, D=64, act=BF, dtype=dtype, lens=[530, 60], tree=True), Workspace()
    args = {k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items() if k not in ("q", "cache")}
    q, out, lse = (torch.zeros(s, dtype=t, device=device) for s, t in ((d["q"].shape, BF), (d["q"].shape, BF),
                                                                       (d["q"].shape[:2], torch.float32)))
    cache = _to(d["cache"], device)
    got = _run(beside, lambda: block_attention(q, cache, out=out, lse=lse, workspace=work, **args), [out, lse], [(q, d["q"])])
    want = B.attention(d["q"], *d["cache"], **{k: x for k, x in d.items() if k not in ("q", "cache")})
    R.close(got[0], want[0], want[2])
    R.close(got[1], want[1], want[3])


@pytest.mark.parametrize("slots", [900, 40000])
def test_requests(device, beside, slots):
    """Each call by itself; both paths of the release and of the compaction."""
    from dspine_amd.kernels.cache import copy_kv, new_cache
    from dspine_amd.runtime.requests import compact_requests, fork_requests, free_requests
    from dspine_amd.verify import Workspace

    g, work = _gen(slots), Workspace()
    ids = lambda *x: torch.tensor(x, dtype=torch.int64, device=device)  # noqa: E731
    table, lens, shared = _pool(7, rows=6, cols=260, slots=slots, lens=[200, 150, 90])
    gt, gn, gs = (torch.zeros_like(x, device=device) for x in (table, lens, shared))
    late = [(gt, table), (gn, lens), (gs, shared)]
    one = ids(0, 1), ids(3, 4)

    got = _run(beside, lambda: fork_requests(gt, gn, gs, *one), [gt, gn, gs], late)
    after = [table, lens, shared]
    B.fork(*after, [0, 1], [3, 4])
    assert all(torch.equal(a, b) for a, b in zip(got, after))
    free, count = torch.full((slots,), -7, dtype=torch.int64, device=device), torch.zeros(1, dtype=torch.int32, device=device)
    dead = ids(1, 2, 4)
    got = _run(beside, lambda: free_requests(gt, gn, gs, dead, free_slots=free, free_count=count, workspace=work),
               [gn, gs, free, count], list(zip((gt, gn, gs), after)))
    freed = B.free(*after, [1, 2, 4])
    assert torch.equal(got[0], after[1]) and torch.equal(got[1], after[2])
    assert int(got[3]) == len(freed) and got[2][: len(freed)].tolist() == freed
    cache, k = new_cache(slots, 1, 16, dtype=BF, device=device), torch.randn(slots, 1, 16, generator=g).to(BF)
    moves, counts = torch.full((2, slots // 2), -7, dtype=torch.int64, device=device), torch.zeros(2, dtype=torch.int32, device=device)
    live = ids(0, 3)
    got = _run(beside, lambda: compact_requests(gt, gn, live, cache, shared=gs, moves=moves, counts=counts, workspace=work),
               [gt, gs, cache.k, moves, counts], [*zip((gt, gn, gs), after), (cache.k, k)])
    src, dst, used = B.compact(after[0], after[1], [0, 3], slots, after[2])
    k[dst] = k[src]
    assert torch.equal(got[0], after[0]) and torch.equal(got[1], after[2]) and torch.equal(got[2], k)
    assert got[3][:, : len(src)].tolist() == [src, dst] and got[4].tolist() == [used, len(src)]
    a, b = ids(*range(0, 90)), ids(*range(100, 190))
    got, = _run(beside, lambda: copy_kv(cache, a, b), [cache.k], [(cache.k, k)])
    k[100:190] = k[:90]
    assert torch.equal(got, k)
