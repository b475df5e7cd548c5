"""Requests forked, freed and compacted, and slots copied, on the GPU against their definitions (tests/blocks_ref.py):
whole numbers, so every bit."""

import blocks_ref as B
import pytest
import torch
from test_gpu_tree import BF, E4, HF, I8, _cache_cpu, _gen, _to

pytestmark = pytest.mark.gpu


def _pool(seed, *, rows, cols, slots, lens, dtype=torch.int32, lend=()):
    """(table, lens, shared): row r holds lens[r] slots; (a, b, n) in ``lend``: row b's first n slots are row a's."""
    g = _gen(seed)
    perm = torch.randperm(slots, generator=g).to(torch.int32)
    table = torch.full((rows, cols), -1, dtype=torch.int32)
    shared = torch.zeros(slots, dtype=torch.int32)
    at, owner = 0, {b: (a, n) for a, b, n in lend}
    for r, n in enumerate(lens):
        a, k = owner.get(r, (0, 0))
        table[r, :k] = table[a, :k]
        shared[table[a, :k].long()] += 1
        table[r, k:n] = perm[at: at + n - k]
        at += n - k
    full = torch.zeros(rows, dtype=dtype)
    full[: len(lens)] = torch.tensor(lens, dtype=dtype)
    return table, full, shared


def _ids(device, x, dtype):
    return torch.tensor(x, dtype=dtype, device=device)


@pytest.mark.parametrize("lens_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("row_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("cols", [1, 300, 1027])
def test_fork_and_free(device, cols, row_dtype, lens_dtype):
    """Several children of a parent (in a row and apart), rows of no length and past the table's, rows outside the
    table, a row named twice, a request that outlives the others."""
    from dspine_amd.runtime.requests import fork_requests, free_requests

    lens = [cols, 0, min(3, cols), min(257, cols), min(64, cols), cols // 2]
    slots = sum(lens) + 41
    table, full, shared = _pool(1, rows=16, cols=cols, slots=slots, lens=lens, dtype=lens_dtype,
                                lend=[(0, 4, min(30, cols))] if cols > 64 else ())
    full[0], full[1] = cols + 99, -5  # clamped
    parents, children = [0, 0, 3, 0, 4, 1, -1, 5, 2, 17], [6, 7, 8, 9, 10, 11, 12, 5, 99, 13]
    t, n, s = (x.to(device) for x in (table, full, shared))
    fork_requests(t, n, s, _ids(device, parents, row_dtype), _ids(device, children, row_dtype))
    B.fork(table, full, shared, parents, children)
    assert torch.equal(t.cpu(), table) and torch.equal(n.cpu(), full) and torch.equal(s.cpu(), shared)
    for rows in ([0, 3, 0, -4, 9], [], [6, 7, 8, 10, 4, 200], [1, 2, 5, 11, 12, 13]):
        free = torch.full((slots,), -7, dtype=torch.int64, device=device)
        got, count = free_requests(t, n, s, _ids(device, rows, row_dtype), free_slots=free)
        want = B.free(table, full, shared, rows)
        assert got is free and int(count) == len(want)
        assert free.tolist() == want + [-7] * (slots - len(want))
        assert torch.equal(n.cpu(), full) and torch.equal(s.cpu(), shared) and torch.equal(t.cpu(), table)
    assert not bool(s.any())


def test_slots_outside_the_pool_and_too_little_room(device):
    from dspine_amd.runtime.requests import fork_requests, free_requests

    table, full, shared = _pool(2, rows=3, cols=70, slots=90, lens=[60, 10])
    table[0, 5], table[0, 6], table[0, 7] = -1, 90, 2 ** 31 - 1
    t, n, s = (x.to(device) for x in (table, full, shared))
    fork_requests(t, n, s, _ids(device, [0], torch.int64), _ids(device, [2], torch.int64))
    B.fork(table, full, shared, [0], [2])
    assert torch.equal(t.cpu(), table) and torch.equal(s.cpu(), shared)
    free = torch.full((20,), -7, dtype=torch.int64, device=device)
    _, count = free_requests(t, n, s, _ids(device, [0, 2], torch.int64), free_slots=free[:11])
    want = B.free(table, full, shared, [0, 2])
    assert int(count) == 57 and free.tolist() == want[:11] + [-7] * 9 and not bool(s.any())


def test_a_large_pool(device):
    """Many chunks of the pool, most of them without a freed slot; a strided table."""
    from dspine_amd.runtime.requests import fork_requests, free_requests

    rows, cols, slots = 40, 9000, 1000003
    g = _gen(3)
    lens = torch.randint(1, cols, (12,), generator=g).tolist()
    table, full, shared = _pool(4, rows=rows, cols=cols, slots=slots, lens=lens, lend=[(0, 1, min(lens[0], lens[1]) // 2)])
    wide = torch.zeros(rows, cols + 13, dtype=torch.int32, device=device)
    t = wide[:, :cols]
    t.copy_(table)
    n, s = full.to(device), shared.to(device)
    parents, children = [0, 1, 1, 5, 7, 7, 7], list(range(20, 27))
    fork_requests(t, n, s, _ids(device, parents, torch.int64), _ids(device, children, torch.int64))
    B.fork(table, full, shared, parents, children)
    assert torch.equal(t.cpu(), table) and torch.equal(s.cpu(), shared) and not bool(wide[:, cols:].any())
    for dead in ([1, 5, 20], [0, 7, 21, 22, 24], list(range(rows))):
        got, count = free_requests(t, n, s, _ids(device, dead, torch.int64))
        want = B.free(table, full, shared, dead)
        assert got[: int(count)].tolist() == want and torch.equal(s.cpu(), shared) and torch.equal(n.cpu(), full)


LAYERS = [(BF, BF, 2, 64, 1), (HF, HF, 3, 80, 3), (BF, E4, 8, 128, 2), (BF, I8, 1, 16, 5), (BF, I8, 3, 96, 20)]


@pytest.mark.parametrize("act, dtype, H, D, layers", LAYERS)
@pytest.mark.parametrize("slots, lens", [(700, [100, 0, 257, 33]), (9001, [3000, 1, 2500]), (401, [200, 201]), (50, [])])
def test_compact(device, slots, lens, act, dtype, H, D, layers):
    """Used slots anywhere, a full pool, an empty one; shared slots; rows named twice and outside the table; as many
    tensors as need more than one launch."""
    from dspine_amd.runtime.requests import compact_requests

    g = _gen(slots)
    cols = max([*lens, 1]) + 5
    lend = [(0, 2, 50)] if len(lens) > 2 and lens[0] >= 50 else ()
    table, full, shared = _pool(5, rows=9, cols=cols, slots=slots, lens=lens, lend=lend)
    if lens and slots == 700:
        table[0, 60], table[2, 200] = slots + 5, -3  # hold nothing
    caches = [_cache_cpu(g, slots, H, D, act, dtype) for _ in range(layers)]
    rows = [3, 0, 2, 1, 0, -1, 44] if len(lens) > 2 else list(range(len(lens)))
    t, n, s, gpu = table.to(device), full.to(device), shared.to(device), [_to(c, device) for c in caches]
    moves = torch.full((2, slots // 2 + 3), -7, dtype=torch.int64, device=device)
    got, counts = compact_requests(t, n, _ids(device, rows, torch.int32), gpu, shared=s, moves=moves)
    src, dst, used = B.compact(table, full, rows, slots, shared)
    assert got is moves and counts.tolist() == [used, len(src)]
    assert moves[0].tolist() == src + [-7] * (moves.shape[1] - len(src))
    assert moves[1].tolist() == dst + [-7] * (moves.shape[1] - len(src))
    assert torch.equal(t.cpu(), table) and torch.equal(s.cpu(), shared) and torch.equal(n.cpu(), full)
    for c, x in zip(caches, gpu):
        for want, have in zip(c, (x.k, x.v, x.k_scale, x.v_scale)):
            if want is not None:
                want = want.view(torch.uint8) if want.dtype == E4 else want
                have = have.view(torch.uint8) if have.dtype == E4 else have
                want[dst] = want[src]
                assert torch.equal(have.cpu(), want)
    _, counts = compact_requests(t, n, _ids(device, rows, torch.int32), gpu, shared=s)
    assert counts.tolist() == [used, 0] and torch.equal(t.cpu(), table) and torch.equal(s.cpu(), shared)


def test_compact_a_block_table(device):
    """A block index follows its own table."""
    from dspine_amd.kernels.blocks import new_block_index
    from dspine_amd.runtime.requests import compact_requests

    g = _gen(8)
    table, full, _ = _pool(6, rows=4, cols=20, slots=60, lens=[7, 20, 3])
    index = new_block_index(60, 3, 48, block_size=16, device=device)
    index.bounds.copy_(torch.randn(index.bounds.shape, generator=g))
    before, t = index.bounds.clone(), table.to(device)
    moves, counts = compact_requests(t, full.to(device), _ids(device, [0, 1, 2], torch.int64), index)
    src, dst, used = B.compact(table, full, [0, 1, 2], 60)
    assert counts.tolist() == [30, len(src)] and torch.equal(t.cpu(), table)
    before[dst] = before[src]
    assert torch.equal(index.bounds, before)


@pytest.mark.parametrize("dtype", [BF, E4])
def test_copy_of_strided_caches(device, dtype):
    """Keys and values as two halves of one tensor, heads apart, scales in one table; pairs outside the pool; a count on
    the device; both widths of slots."""
    from dspine_amd.kernels.cache import KVCache, copy_kv

    slots, H, D, g = 333, 3, 32, _gen(9)
    both = torch.randint(0, 120, (slots, 2, H, 2, D), generator=g, dtype=torch.uint8).to(device)
    if dtype == BF:
        both = both.to(torch.int16)
    scales = torch.randn(2, H, slots, generator=g).to(device)
    view = both.view(dtype)
    cache = KVCache(view[:, 0, :, 0], view[:, 1, :, 0], *((scales[0].t(), scales[1].t()) if dtype == E4 else (None, None)))
    perm = torch.randperm(slots, generator=g)
    src, dst = perm[:100].clone(), perm[100:200].clone()
    src[3], dst[4], src[5] = -1, slots, 2 ** 40
    for count, i64 in ((None, False), (7, True), (-3, True), (1000, False)):
        n = 100 if count is None else max(0, min(count, 100))
        want, wants = both.clone(), scales.clone()
        for a, b in list(zip(src.tolist(), dst.tolist()))[:n]:
            if 0 <= a < slots and 0 <= b < slots:
                want[b, :, :, 0] = want[a, :, :, 0]
                wants[:, :, b] = wants[:, :, a] if dtype == E4 else wants[:, :, b]
        kw = {} if count is None else dict(count=torch.tensor([count], dtype=torch.int32, device=device))
        a = src if i64 else src.clamp(max=2 ** 31 - 1).to(torch.int32)
        copy_kv(cache, a.to(device), dst.to(device), **kw)
        assert torch.equal(both, want) and torch.equal(scales, wants)


def test_a_round_of_samples(device):
    """As they are used: a prompt forked, samples that grow by slots of their own, losers freed, the pool compacted, what a
    request reads unchanged; captured, and replayed from the same beginning."""
    from dspine_amd.kernels.cache import new_cache, read_kv, write_kv
    from dspine_amd.runtime.requests import compact_requests, fork_requests, free_requests
    from dspine_amd.verify import Workspace

    g = _gen(11)
    slots, cols = 900, 300
    cache = new_cache(slots, 2, 64, dtype=BF, device=device)
    first = [torch.randn(slots, 2, 64, generator=g).to(BF).to(device) for _ in range(2)]
    every = torch.arange(slots, device=device)
    perm = torch.randperm(slots, generator=g).to(torch.int32).to(device)
    table, lens = torch.zeros(8, cols, dtype=torch.int32, device=device), torch.zeros(8, dtype=torch.int32, device=device)
    shared, work = torch.zeros(slots, dtype=torch.int32, device=device), Workspace()
    work.get(1 << 20, device)
    kids, dead = _ids(device, [1, 2, 3], torch.int64), _ids(device, [0, 2], torch.int64)
    live, zero = _ids(device, [1, 3], torch.int64), _ids(device, [0, 0, 0], torch.int64)
    free_slots = torch.empty(slots, dtype=torch.int64, device=device)
    free_count = torch.empty(1, dtype=torch.int32, device=device)

    def begin():
        write_kv(cache, *first, every)
        table.zero_(), lens.zero_(), shared.zero_()
        table[0, :200] = perm[:200]
        lens[:1] = 200

    def step():
        fork_requests(table, lens, shared, zero, kids)
        for r in (1, 2, 3):
            table[r, 200: 200 + 30 * r] = perm[200 + 100 * r: 200 + 130 * r]
            lens[r: r + 1] += 30 * r
        free_requests(table, lens, shared, dead, free_slots=free_slots, free_count=free_count, workspace=work)
        before = [read_kv(cache, table[r, :n].contiguous(), dtype=BF) for r, n in ((1, 230), (3, 290))]
        moves, counts = compact_requests(table, lens, live, cache, shared=shared, workspace=work)
        after = [read_kv(cache, table[r, :n].contiguous(), dtype=BF) for r, n in ((1, 230), (3, 290))]
        return before, after, moves, counts

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        begin()
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    begin()
    with torch.cuda.graph(graph):
        before, after, moves, counts = step()
    for _ in range(3):
        begin()
        graph.replay()
        assert lens.tolist() == [0, 230, 0, 290, 0, 0, 0, 0]
        # the prompt is held by two, row 2's own sixty are free
        assert int(free_count) == 60 and counts.tolist()[0] == 200 + 30 + 90
        assert int(shared.sum()) == 200 and int(table[1, :230].max()) < 320 and int(table[3, :290].max()) < 320
        assert sorted(free_slots[:60].tolist()) == free_slots[:60].tolist() == sorted(perm[400:460].tolist())
        for a, b in zip(before, after):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("rows, cols", [(40, 60), (75, 320), (75, 330), (1030, 7), (1, 8000), (9, 4096), (9, 4097)])
def test_many_short_rows_and_few_long_ones(device, rows, cols):
    """On both sides of what one workgroup takes: rows that share, rows named again in another group of eight, all of them
    ended in two calls, and the rest compacted between."""
    from dspine_amd.runtime.requests import compact_requests, free_requests

    g = _gen(rows + cols)
    lens = torch.randint(0, min(cols, 16000 // rows) + 1, (rows,), generator=g).tolist()
    lend = [(i, i + 1, min(lens[i], lens[i + 1]) // 2) for i in range(0, rows - 1, 2)]
    slots = max(1, min(16384, sum(lens) + 50))
    table, full, shared = _pool(rows, rows=rows, cols=cols, slots=slots, lens=lens, lend=lend)
    t, n, s = (x.to(device) for x in (table, full, shared))
    dead = torch.randint(-1, rows + 1, (rows,), generator=g).tolist() + [0, 0]
    for what in (dead, list(range(rows))):
        got, count = free_requests(t, n, s, _ids(device, what, torch.int32))
        want = B.free(table, full, shared, what)
        assert got[: int(count)].tolist() == want
        assert torch.equal(n.cpu(), full) and torch.equal(s.cpu(), shared)
        cache = _cache_cpu(g, slots, 1, 16, BF, BF)
        gpu = _to(cache, device)
        live = list(range(rows - 1, -1, -1)) + [0]
        moves, counts = compact_requests(t, n, _ids(device, live, torch.int64), gpu, shared=s)
        src, dst, used = B.compact(table, full, live, slots, shared)
        assert counts.tolist() == [used, len(src)] and moves[0, : len(src)].tolist() == src
        assert torch.equal(t.cpu(), table) and torch.equal(s.cpu(), shared)
        cache[0][dst] = cache[0][src]
        assert torch.equal(gpu.k.cpu(), cache[0])
    assert not bool(n.any())
