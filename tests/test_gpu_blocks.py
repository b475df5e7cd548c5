"""The block index, its scores, the selection and the attention over selected blocks, on the GPU against their
definitions (tests/blocks_ref.py)."""

import math

import blocks_ref as B
import pytest
import torch
import tree_ref as R
from test_gpu_tree import BF, E4, HF, I8, _cache_cpu, _gen, _round, _to

pytestmark = pytest.mark.gpu
CACHES = [(BF, BF), (HF, HF), (BF, E4), (HF, E4), (BF, I8), (HF, I8)]


def _table(g, lens, width, spare=29):
    slots = sum(lens) + spare
    perm = torch.randperm(slots, generator=g)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        table[b, :n] = perm[at: at + n]
        at += n
    return table, slots


def _index_call(device, bounds, size, cache, **tables):
    from dspine_amd.kernels.blocks import BlockIndex, index_blocks

    x = BlockIndex(bounds.to(device), size)
    index_blocks(x, _to(cache, device), **{k: (t.to(device) if isinstance(t, torch.Tensor) else t) for k, t in tables.items()})
    return x.bounds


@pytest.mark.parametrize("act, dtype", CACHES)
@pytest.mark.parametrize("D, H, size", [(16, 1, 16), (64, 3, 32), (80, 2, 64), (128, 8, 64), (192, 1, 128), (256, 2, 16)])
def test_index(device, D, H, size, act, dtype):
    """Growths that finish no block, one, several; from zero; a length of zero; one that shrinks."""
    g = _gen(D + size)
    frm = [0, 0, size - 1, size, 2 * size - 1, 5, 3 * size, 40]
    to = [0, 3 * size + 5, size, 2 * size - 1, 4 * size, 6, 2 * size, 40 + size]
    table, slots = _table(g, [max(t, 1) for t in to], 4 * size + 3)
    cache = _cache_cpu(g, slots, H, D, act, dtype)
    per = 5
    blocks = torch.randperm(8 * per + 3, generator=g)[: 8 * per].view(8, per).to(torch.int32)
    bounds = torch.randn(8 * per + 3, H, 2, D, generator=g).to(act)
    args = dict(page_table=table, block_table=blocks, from_lens=torch.tensor(frm, dtype=torch.int32),
                to_lens=torch.tensor(to, dtype=torch.int32))
    want, tol = B.index(bounds, size, cache[0], cache[2], **args)
    R.close(_index_call(device, bounds, size, cache, **args), want, tol)
    args["longest"] = size + 1  # two blocks of a request at most
    want, tol = B.index(bounds, size, cache[0], cache[2], **args)
    R.close(_index_call(device, bounds, size, cache, **args), want, tol)


@pytest.mark.parametrize("act, dtype", [(BF, BF), (HF, E4), (BF, I8)])
def test_index_of_slots_that_hold_nothing(device, act, dtype):
    """Slots outside the cache, a block of nothing else, a page table that ends inside a block, index rows outside the index,
    a block table that ends early; NaN and infinite keys."""
    g = _gen(3)
    H, D, size = 2, 32, 16
    table, slots = _table(g, [40, 40, 40], 40)
    cache = _cache_cpu(g, slots, H, D, act, dtype)
    table[0, 3], table[0, 4], table[0, 16:32] = -1, slots, 2 ** 31 - 1
    if dtype == BF:
        cache[0][table[1, 5].long(), 0, 7] = math.nan
        cache[0][table[1, 20].long(), 1, 8] = math.inf
    else:
        cache[2][table[1, 5].long(), 0] = math.nan
    blocks = torch.tensor([[3, 0, 9], [1, 8, 2], [-1, 30, 5]], dtype=torch.int32)
    bounds = torch.randn(10, H, 2, D, generator=g).to(act)
    args = dict(page_table=table, block_table=blocks, from_lens=torch.zeros(3, dtype=torch.int32),
                to_lens=torch.tensor([64, 64, 64], dtype=torch.int32))
    want, tol = B.index(bounds, size, cache[0], cache[2], **args)
    got = _index_call(device, bounds, size, cache, **args)
    assert bool(torch.isnan(got[1, 0, :, 7 if dtype == BF else slice(None)]).all())
    nan = torch.isnan(got.cpu())
    want[nan] = math.nan  # (float64's least and largest of NaN are NaN too)
    assert bool((nan.sum() == (2 if dtype == BF else 2 * D)))
    R.close(got, want, torch.nan_to_num(tol, nan=0.0, posinf=0.0))


def _score_round(seed, *, bs, T, H, G, D, size, act, lens, nodes=None, offsets=False):
    g = _gen(seed)
    per = max(1, max(lens) // size) + 1
    rows = bs * per + 5
    mid = torch.randn(rows, H, 1, D, generator=g)
    half = torch.rand(rows, H, 1, D, generator=g)
    d = dict(T=T, block_table=torch.randperm(rows, generator=g)[: bs * per].view(bs, per).to(torch.int32),
             prefix_lens=torch.tensor(lens, dtype=torch.int32),
             verify_lens=None if nodes is None else torch.tensor(nodes, dtype=torch.int32))
    n = bs * T
    if offsets:
        held = torch.tensor(nodes).clamp(0, T)
        d["row_offsets"], n = held.cumsum(0) - held, int(held.sum())
    return torch.randn(n, H * G, D, generator=g).to(act), torch.cat((mid - half, mid + half), 2).to(act), d


def _score_call(device, q, bounds, size, d, **kw):
    from dspine_amd.kernels.blocks import BlockIndex, score_blocks

    return score_blocks(q.to(device), BlockIndex(bounds.to(device), size),
                        **{k: (t.to(device) if isinstance(t, torch.Tensor) else t) for k, t in {**d, **kw}.items()})


SCORES = [  # bs, T, H, G, D, size, lens, nodes
    (1, 1, 1, 1, 16, 16, [15], None),
    (1, 1, 1, 1, 16, 16, [16], None),
    (3, 1, 2, 4, 128, 64, [0, 64, 6500], None),
    (2, 17, 2, 4, 128, 64, [9000, 130], [17, 3]),
    (4, 5, 3, 5, 80, 32, [700, 0, 33, 1100], [5, 2, 0, -1]),
    (2, 33, 1, 7, 96, 16, [2100, 31], None),
    (2, 64, 1, 16, 256, 128, [5000, 700], None),
    (1, 64, 2, 3, 192, 16, [1300], None),
    (2, 64, 1, 8, 64, 16, [4200, 64], [64, 50]),
]


@pytest.mark.parametrize("act", [BF, HF])
@pytest.mark.parametrize("case", range(len(SCORES)))
def test_scores(device, case, act):
    bs, T, H, G, D, size, lens, nodes = SCORES[case]
    q, bounds, d = _score_round(case, bs=bs, T=T, H=H, G=G, D=D, size=size, act=act, lens=lens, nodes=nodes)
    want, tol = B.scores(q, bounds, size, **d)
    R.close(_score_call(device, q, bounds, size, d), want, tol)


def test_scores_of_compact_rows_strided_queries_and_bad_rows(device):
    """Rows by offsets (both widths), queries that are a slice of a fused projection, index rows outside the index, a scale,
    a strided block table; scores of queries that are NaN."""
    q, bounds, d = _score_round(5, bs=4, T=9, H=2, G=3, D=64, size=16, act=BF, lens=[200, 333, 64, 500], nodes=[9, 4, 0, 7],
                                offsets=True)
    d["block_table"][0, 2], d["block_table"][1, 5] = -1, bounds.shape[0]
    want, tol = B.scores(q, bounds, 16, scale=0.3, **d)
    wide = torch.full((q.shape[0], 10, 64), math.nan, dtype=BF)
    wide[:, 2:8] = q
    table = torch.full((4, 40), 7, dtype=torch.int32)
    table[:, : d["block_table"].shape[1]] = d["block_table"]
    from dspine_amd.kernels.blocks import BlockIndex, score_blocks

    for offsets in (torch.int64, torch.int32):
        got = score_blocks(wide.to(device)[:, 2:8], BlockIndex(bounds.to(device), 16), T=9, scale=0.3,
                           block_table=table.to(device)[:, : d["block_table"].shape[1]], prefix_lens=d["prefix_lens"].to(device),
                           verify_lens=d["verify_lens"].to(device), row_offsets=d["row_offsets"].to(offsets).to(device))
        R.close(got, want, tol)
    q[9 + 1, 4] = math.nan  # request 1's second node, cache head 1
    got = _score_call(device, q, bounds, 16, d, scale=0.3).cpu()
    live = torch.isfinite(want)
    assert bool(torch.isnan(got[1, 1][live[1, 1]]).all()) and bool(torch.isfinite(got[1, 0][live[1, 0]]).all())
    assert torch.equal(torch.isfinite(got[[0, 3]]), live[[0, 3]])


def _select_call(device, s, count, **kw):
    from dspine_amd.kernels.blocks import select_blocks

    return select_blocks(s.to(device), count, **{k: (t.to(device) if isinstance(t, torch.Tensor) else t) for k, t in kw.items()})


SELECT = [  # bs, H, L, count, first, last
    (1, 1, 1, 1, 0, 0), (2, 3, 7, 3, 1, 1), (2, 2, 63, 5, 0, 0), (2, 2, 130, 64, 1, 4), (3, 2, 512, 100, 2, 3),
    (2, 2, 513, 511, 0, 2), (2, 4, 2000, 64, 1, 4), (1, 2, 2049, 1000, 0, 0), (1, 2, 8000, 300, 1, 2), (1, 1, 8193, 64, 0, 1),
    (1, 1, 32768, 5000, 3, 0), (2, 1, 300, 299, 150, 149), (1, 1, 9, 20, 0, 0),
]


@pytest.mark.parametrize("kind", ["normal", "few values", "one value", "zeros", "holes", "wide"])
@pytest.mark.parametrize("case", range(len(SELECT)))
def test_selection(device, case, kind):
    bs, H, L, count, first, last = SELECT[case]
    g = _gen(case * 7 + 1)
    s = torch.randn(bs, H, L, generator=g) * 3 + 20
    if kind == "few values":
        s = torch.randint(0, 3, (bs, H, L), generator=g).float()
    elif kind == "one value":
        s = torch.full((bs, H, L), 1.5)
    elif kind == "zeros":
        s = torch.where(torch.rand(bs, H, L, generator=g) < 0.5, 0.0, -0.0)  # one value
        s[..., L // 2:] += (torch.rand(bs, H, L - L // 2, generator=g) < 0.1) * 1e-40
    elif kind == "holes":
        u = torch.rand(bs, H, L, generator=g)
        s = torch.where(u < 0.3, math.nan, torch.where(u < 0.5, -math.inf, torch.where(u < 0.55, math.inf, s)))
    elif kind == "wide":
        s = torch.randn(bs, H, L, generator=g) * torch.exp2(torch.randint(-140, 120, (bs, H, L), generator=g).float())
    size = 32
    lens = torch.tensor([L * size + 5, max(0, L - 2) * size + 31, 0][:bs], dtype=torch.int32)
    args = dict(prefix_lens=lens, block_size=size, first=first, last=last)
    assert torch.equal(_select_call(device, s, count, **args).cpu(), B.select(s, count, **args))


def _block_round(seed, *, count, size, **kw):
    d = _round(seed, **kw)
    g = _gen(seed + 1000)
    bs, H = d["prefix_lens"].numel(), d["cache"][0].shape[1]
    blocks = torch.full((bs, H, count), -1, dtype=torch.int32)
    for b, n in enumerate(d["prefix_lens"].tolist()):
        for h in range(H):
            ids = torch.randperm(max(n, 0) // size, generator=g)[:count]
            blocks[b, h, : ids.numel()] = ids.sort().values
    return dict(d, blocks=blocks, block_size=size)


def _call(d, device, **kw):
    from dspine_amd.kernels.blocks import block_attention

    lse = torch.full(d["q"].shape[:2], 7.0, device=device)
    out = torch.full_like(d["q"], 7.0, device=device)
    args = {k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items() if k not in ("q", "cache")}
    assert block_attention(d["q"].to(device), _to(d["cache"], device), out=out, lse=lse, **{**args, **kw}) is out
    return out, lse


def _check(d, out, lse):
    want, wl, otol, ltol = B.attention(d["q"], *d["cache"], **{k: x for k, x in d.items() if k not in ("q", "cache")})
    none = torch.isnan(wl)
    assert bool((out.cpu()[none] == 7.0).all()) and bool((lse.cpu()[none] == 7.0).all())
    R.close(out.cpu()[~none], want[~none], otol[~none])
    R.close(lse.cpu()[~none], wl[~none], ltol[~none])


SHAPES = [  # T, H, G, D, contexts, tree, size, count
    (1, 1, 1, 16, [1], False, 16, 1),
    (1, 2, 4, 128, [0, 15, 16, 4000], False, 16, 9),
    (1, 8, 8, 64, [700, 33], False, 32, 5),
    (2, 1, 3, 96, [32, 63, 1], True, 16, 2),
    (5, 3, 5, 80, [0, 130, 901], True, 128, 4),
    (16, 2, 1, 128, [47, 1280], False, 64, 12),
    (17, 2, 4, 128, [0, 130, 257, 2900], True, 64, 17),
    (23, 1, 7, 192, [64, 1005], True, 32, 3),
    (33, 1, 2, 256, [95, 650], False, 16, 33),
    (64, 1, 8, 128, [61, 1300], True, 64, 40),
    (64, 2, 1, 256, [429], True, 128, 1),
]


@pytest.mark.parametrize("act, dtype", CACHES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_shapes(device, shape, act, dtype):
    T, H, G, D, lens, tree, size, count = SHAPES[shape]
    d = _block_round(shape * 13 + 1, count=count, size=size, bs=len(lens), T=T, H=H, G=G, D=D, act=act, dtype=dtype, lens=lens,
                     tree=tree)
    _check(d, *_call(d, device))


ROWS = [(3, 2), (7, 4), (17, 4), (40, 4)]  # nodes, query heads a cache head: the forms of the kernel


@pytest.mark.parametrize("act, dtype", CACHES)
@pytest.mark.parametrize("T, G", ROWS)
@pytest.mark.parametrize("size", [16, 128])
def test_attention_lists_as_they_may_come(device, size, T, G, act, dtype):
    """Any order, holes among the entries, entries that name no finished block, a block named twice, entries behind the
    finished blocks' number (not read), bad slots, a page table that ends inside a block and one inside the window."""
    lens = [size * 5 + 3, size * 3, size - 1]
    d = _block_round(91, count=6, size=size, bs=3, T=T, H=2, G=G, D=64, act=act, dtype=dtype, lens=lens, tree=True)
    d["blocks"] = torch.tensor([[[4, -1, 0, 4, 2, 9], [5, 2 ** 31 - 1, -2 ** 31, 3, 1, 1]],
                                [[2, 2, 2, 0, 0, 0], [-1, -1, -1, 0, 1, 2]],
                                [[0, 0, 0, 0, 0, 0], [0, 1, 2, 3, 4, 5]]], dtype=torch.int32)
    slots = d["cache"][0].shape[0]
    t = d["page_table"]
    t[0, 2 * size + 1], t[0, 4 * size + 7], t[0, lens[0] + 1] = -1, slots, 2 ** 31 - 1
    t[1, size: 2 * size] = -1
    _check(d, *_call(d, device))
    d["page_table"] = t[:, : lens[0] + 1].contiguous()
    _check(d, *_call(d, device))
    d["page_table"] = t[:, : 4 * size + 9].contiguous()
    _check(d, *_call(d, device))


@pytest.mark.parametrize("act, dtype", CACHES)
@pytest.mark.parametrize("T, G", ROWS)
def test_what_is_not_finite_stays_with_the_nodes_that_see_it(device, T, G, act, dtype):
    """Values in the window, in the unfinished block and in blocks that are not selected."""
    d = _block_round(92, count=2, size=16, bs=1, T=T, H=1, G=G, D=64, act=act, dtype=dtype, lens=[16 * 9 + 2], tree=False)
    d["masks"] = torch.tensor([[R.signed(1 | 1 << i) for i in range(T)]], dtype=torch.int64)
    k, v, ks, vs = d["cache"]
    at = d["page_table"].long()[0]
    chosen = set(d["blocks"].flatten().tolist())
    out_of = torch.cat([at[16 * j: 16 * j + 16] for j in range(9) if j not in chosen])
    for x in ((k, v) if ks is None else (ks, vs)):
        x[out_of] = math.nan
        x[at[16 * 9 + 2 + 2]] = math.nan  # node 2
    out, lse = _call(d, device)
    want, wl, otol, ltol = B.attention(d["q"], *d["cache"], **{n: x for n, x in d.items() if n not in ("q", "cache")})
    fine = torch.arange(T) != 2
    assert bool(torch.isnan(out.cpu()[2]).all()) and bool(torch.isfinite(out.cpu()[fine]).all())
    R.close(out.cpu()[fine], want[fine], otol[fine])
    R.close(lse.cpu()[fine], wl[fine], ltol[fine])


@pytest.mark.parametrize("dtype", [BF, I8])
def test_attention_of_many_requests(device, dtype):
    """More requests than a wave has lanes, uneven lengths, verify lengths on compact rows in another order."""
    g = _gen(17)
    lens = torch.randint(0, 700, (70,), generator=g).tolist()
    nodes = torch.randint(-1, 6, (70,), generator=g).tolist()
    d = _block_round(93, count=5, size=32, bs=70, T=5, H=2, G=3, D=64, act=BF, dtype=dtype, lens=lens, tree=True, nodes=nodes)
    held = torch.tensor(nodes).clamp(0, 5)
    order = torch.randperm(70, generator=g)
    start = torch.zeros(70, dtype=torch.int64)
    start[order] = held[order].cumsum(0) - held[order]
    rows = int(held.sum()) + 3
    d.update(q=torch.randn(rows, 6, 64, generator=g).to(BF), row_offsets=start)
    _check(d, *_call(d, device))


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("T, G", ROWS)
def test_all_blocks_is_the_whole_context(device, T, G, dtype):
    """Every finished block selected: tree_attention's result, the same bits where neither call cuts a request into parts."""
    from dspine_amd.kernels.attention import tree_attention

    for lens in ([64 * 12, 301, 0], [63 - T]):
        if min(lens) < 0:
            continue
        d = _block_round(94, count=12, size=16, bs=len(lens), T=T, H=2, G=G, D=128, act=BF, dtype=dtype, lens=lens, tree=True)
        d["blocks"] = torch.arange(48, dtype=torch.int32).expand(len(lens), 2, -1).contiguous()
        out, lse = _call(d, device)
        args = {k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items()
                if k not in ("q", "cache", "blocks", "block_size")}
        lse2 = torch.full_like(lse, 7.0)
        want = tree_attention(d["q"].to(device), _to(d["cache"], device), lse=lse2, **args)
        _check(d, out, lse)
        _check(d, want, lse2)
        if len(lens) == 1:  # (one tile)
            assert torch.equal(out, want) and torch.equal(lse, lse2)


def test_a_long_context_of_slots_past_32_bits_of_bytes(device):
    """A cache of more than 4 GiB whose selected blocks lie at its end."""
    slots, H, D, size = 2200000, 8, 128, 64
    g = torch.Generator(device=device).manual_seed(3)
    from dspine_amd.kernels.blocks import BlockIndex, block_attention, index_blocks
    from dspine_amd.kernels.cache import KVCache

    cache = KVCache(*(torch.empty(slots, H, D, dtype=BF, device=device) for _ in range(2)))
    table = torch.arange(slots - 2001, slots, device=device, dtype=torch.int32).flip(0).view(1, -1)
    near = table[0].long()
    small = [torch.randn(2001, H, D, generator=g, device=device).to(BF) for _ in range(2)]
    cache.k[near], cache.v[near] = small[0], small[1]
    blocks = torch.tensor([[[30, 3, 7]] * H], dtype=torch.int32, device=device)
    q = torch.randn(1, H * 4, D, generator=g, device=device).to(BF)
    pre = torch.tensor([2000], dtype=torch.int32, device=device)
    kw = dict(T=1, blocks=blocks, block_size=size, prefix_lens=pre)
    own = KVCache(*small)
    order = torch.arange(2001, device=device, dtype=torch.int32).view(1, -1)
    assert torch.equal(block_attention(q, cache, page_table=table, **kw), block_attention(q, own, page_table=order, **kw))
    bounds = [torch.zeros(31, H, 2, D, dtype=BF, device=device) for _ in range(2)]
    rows = torch.arange(31, device=device, dtype=torch.int32).view(1, -1)
    for x, c, t in zip(bounds, (cache, own), (table, order)):
        index_blocks(BlockIndex(x, size), c, page_table=t, block_table=rows, from_lens=pre * 0, to_lens=pre)
    assert torch.equal(*bounds) and bool((bounds[0][:, :, 0] < bounds[0][:, :, 1]).all())


def test_the_calls_of_a_round_together(device):
    """Prompt indexed, round scored, selected and attended, the round's growth indexed, as a captured graph whose lengths
    change between the replays; each replay equals eager calls, and the score of a block bounds what attention finds in it."""
    from dspine_amd.kernels.blocks import block_attention, index_blocks, new_block_index, score_blocks, select_blocks
    from dspine_amd.kernels.cache import KVCache

    g = _gen(23)
    T, H, G, D, size, lens = 6, 2, 4, 64, 16, [500, 120, 63]
    d = _round(95, bs=3, T=T, H=H, G=G, D=D, act=BF, dtype=BF, lens=[700, 700, 700], tree=True)
    table, q = d["page_table"].to(device), d["q"].to(device)
    cache = KVCache(*(x.to(device) for x in d["cache"][:2]))
    index = new_block_index(3 * 44, H, D, block_size=size, device=device)
    rows = torch.randperm(3 * 44, generator=g).view(3, 44).to(torch.int32).to(device)
    pre, old = torch.zeros(3, dtype=torch.int32, device=device), torch.zeros(3, dtype=torch.int32, device=device)
    masks = d["masks"].to(device)

    def step():
        index_blocks(index, cache, page_table=table, block_table=rows, from_lens=old, to_lens=pre)
        scores = score_blocks(q, index, T=T, block_table=rows, prefix_lens=pre)
        blocks = select_blocks(scores, 7, prefix_lens=pre, block_size=size, first=1, last=2)
        return scores, blocks, block_attention(q, cache, T=T, blocks=blocks, block_size=size, page_table=table,
                                               prefix_lens=pre, masks=masks)

    pre.copy_(torch.tensor(lens))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(4):
        pre.copy_(torch.tensor([n + 17 * turn for n in lens]))
        graph.replay()
        ours = [x.clone() for x in got]
        for x, y in zip(ours, step()):
            assert torch.equal(x, y)
        scores, blocks = ours[0].cpu(), ours[1].cpu()
        now = pre.cpu()
        assert torch.equal(blocks, B.select(scores, 7, prefix_lens=now, block_size=size, first=1, last=2))
        args = dict(T=T, blocks=blocks, block_size=size, page_table=d["page_table"], prefix_lens=now, masks=d["masks"])
        want, _, otol, _ = B.attention(d["q"], *d["cache"], **args)
        R.close(ours[2], want, otol)
        old.copy_(pre)
    for b, n in enumerate(pre.tolist()):
        for j in range(n // size):
            keys = d["cache"][0][d["page_table"][b, j * size: (j + 1) * size].long()].double()
            x = torch.einsum("nhgd,phd->hngp", d["q"][b * T: (b + 1) * T].double().view(T, H, G, D), keys) / math.sqrt(D)
            assert bool((x.amax((1, 2, 3)) <= scores[b, :, j].double() * (1 + 1e-5) + 1e-5).all())
