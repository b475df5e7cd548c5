"""The KV cache's write and read, the attention of drafted trees over it, and the greedy acceptance
and commit of a tree, on the GPU against their definitions in float64 (tests/tree_ref.py)."""

import math

import pytest
import torch
import tree_ref as R

pytestmark = pytest.mark.gpu

BF, HF, E4, I8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _to(cache, device):
    from dspine_amd.kernels.cache import KVCache

    return KVCache(*(None if t is None else t.to(device) for t in cache))


def _cache_cpu(g, slots, H, D, act, dtype):
    """(k, v, k_scale, v_scale) on the CPU; 8-bit codes of random rows with scales over a wide range."""
    if dtype not in R.TOP:
        return tuple(torch.randn(slots, H, D, generator=g).to(dtype) for _ in range(2)) + (None, None)
    kv = []
    for _ in range(2):
        x = torch.randn(slots, H, D, generator=g)
        scale, y = R.quantise(x, dtype)
        kv.append((y.float().to(dtype) if dtype == E4 else y.round().to(I8), scale.float()))
    kv[1] = (kv[1][0], kv[1][1] * torch.exp2(torch.randint(-6, 5, (slots, H), generator=g)))
    return kv[0][0], kv[1][0], kv[0][1], kv[1][1]


def _tree(g, bs, T):
    i = torch.arange(T)
    p = (i - 1 - (torch.rand(bs, T, generator=g) * torch.clamp(i, max=5)).long()).clamp(min=0)
    p[:, 0] = -1
    masks, _ = R.tree_masks(p)
    return p.to(torch.int32), torch.tensor([[R.signed(m) for m in row] for row in masks], dtype=torch.int64)


def _round(seed, *, bs, T, H, G, D, act, dtype, lens, tree, nodes=None, spare=37):
    """A batch's inputs on the CPU: contexts ``lens``, nodes per request (default T) on dense rows."""
    g = _gen(seed)
    lens = list(lens)
    width = max(lens) + T
    slots = sum(n + T for n in lens) + spare
    perm = torch.randperm(slots, generator=g)
    table = torch.full((bs, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        table[b, : n + T] = perm[at: at + n + T]
        at += n + T
    k, v, ks, vs = _cache_cpu(g, slots, H, D, act, dtype)
    return dict(q=torch.randn(bs * T, H * G, D, generator=g).to(act), cache=(k, v, ks, vs),
                T=T, page_table=table, prefix_lens=torch.tensor(lens, dtype=torch.int32),
                verify_lens=None if nodes is None else torch.tensor(nodes, dtype=torch.int32),
                masks=_tree(g, bs, T)[1] if tree else None)


def _call(d, device, **kw):
    from dspine_amd.kernels.attention import tree_attention

    lse = torch.full(d["q"].shape[:2], 7.0, device=device)
    out = torch.full_like(d["q"], 7.0, device=device)
    args = {k: (x.to(device) if isinstance(x, torch.Tensor) else x) for k, x in d.items() if k not in ("q", "cache")}
    got = tree_attention(d["q"].to(device), _to(d["cache"], device), out=out, lse=lse, **{**args, **kw})
    assert got is out
    return out, lse


def _check(d, out, lse, touched=None):
    args = {k: x for k, x in d.items() if k not in ("q", "cache")}
    want, wl, otol, ltol = R.attention(d["q"], *d["cache"], **args)
    none = torch.isnan(wl) if touched is None else ~touched  # rows of no node: left as they were
    assert bool((out.cpu()[none] == 7.0).all()) and bool((lse.cpu()[none] == 7.0).all())
    R.close(out.cpu()[~none], want[~none], otol[~none])
    R.close(lse.cpu()[~none], wl[~none], ltol[~none])


SHAPES = [  # T, H, G, D, contexts, tree
    (1, 1, 1, 16, [1], False),
    (1, 2, 4, 128, [0, 15, 16, 31], False),
    (1, 8, 8, 64, [700, 33], False),
    (2, 1, 3, 96, [32, 63, 1], True),
    (5, 3, 5, 80, [0, 30, 301], True),
    (16, 2, 1, 128, [47, 128], False),
    (17, 2, 4, 128, [0, 130, 257, 900], True),
    (23, 1, 7, 192, [64, 5], True),
    (33, 1, 2, 256, [95, 250], False),
    (64, 1, 8, 128, [61, 300], True),
    (64, 2, 1, 256, [129], True),
]


@pytest.mark.parametrize("act, dtype", [(BF, BF), (HF, HF), (BF, E4), (HF, E4), (BF, I8), (HF, I8)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_shapes(device, shape, act, dtype):
    T, H, G, D, lens, tree = SHAPES[shape]
    d = _round(shape * 11 + 1, bs=len(lens), T=T, H=H, G=G, D=D, act=act, dtype=dtype, lens=lens, tree=tree)
    _check(d, *_call(d, device))


@pytest.mark.parametrize("dtype", [BF, I8])
def test_attention_many_requests_of_uneven_length(device, dtype):
    g = _gen(5)
    lens = torch.randint(0, 400, (70,), generator=g).tolist()
    lens[3], lens[41] = 5000, 2311
    d = _round(6, bs=70, T=4, H=2, G=2, D=64, act=BF, dtype=dtype, lens=lens, tree=True)
    _check(d, *_call(d, device))


@pytest.mark.parametrize("dtype", [HF, E4])
def test_attention_long_context(device, dtype):
    d = _round(8, bs=2, T=3, H=1, G=4, D=128, act=HF, dtype=dtype, lens=[40001, 77], tree=True)
    _check(d, *_call(d, device))


@pytest.mark.parametrize("offsets", ["i32", "i64", "dense"])
def test_attention_ragged_nodes_leave_other_rows(device, offsets):
    """Per-request node counts (zero among them), on dense or compact rows with gaps."""
    nodes = [4, 0, 17, 1, 9]
    d = _round(9, bs=5, T=17, H=2, G=3, D=64, act=BF, dtype=BF, lens=[40, 12, 0, 333, 64], tree=True, nodes=nodes)
    if offsets != "dense":
        at, o = 2, []
        for n in nodes:
            o.append(at)
            at += n + 1
        d["row_offsets"] = torch.tensor(o, dtype=torch.int32 if offsets == "i32" else torch.int64)
        d["q"] = torch.randn(at + 3, 6, 64, generator=_gen(3)).to(BF)
    _check(d, *_call(d, device))


def test_attention_rows_outside_q_are_left_out(device):
    """Row offsets that point outside q: those nodes are dropped, the others computed."""
    d = _round(9, bs=3, T=4, H=1, G=2, D=64, act=BF, dtype=BF, lens=[10, 11, 12], tree=False)
    d["row_offsets"] = torch.tensor([0, -3, 6], dtype=torch.int64)
    d["q"] = d["q"][:8].contiguous()
    out, lse = _call(d, device)
    ref = dict(d, row_offsets=torch.tensor([0, 20, 8], dtype=torch.int64), q=torch.zeros(24, 2, 64, dtype=BF))
    ref["q"][0:4] = d["q"][0:4]
    ref["q"][23] = d["q"][0]  # request 1's last node is row 0, as request 0's first: either may be written last
    ref["q"][8:10] = d["q"][6:8]
    args = {k: x for k, x in ref.items() if k not in ("q", "cache")}
    want, wl, otol, ltol = R.attention(ref["q"], *ref["cache"], **args)
    R.close(out.cpu()[1:4], want[1:4], otol[1:4])
    R.close(out.cpu()[6:8], want[8:10], otol[8:10])
    assert bool((out.cpu()[4:6] == 7.0).all()) and bool((lse.cpu()[4:6] == 7.0).all())


@pytest.mark.parametrize("dtype", [BF, HF, E4, I8])
def test_attention_masks_that_leave_rows_empty(device, dtype):
    """No context and masks without the node's own bit: zeros and -inf; bits past the window do nothing."""
    act = HF if dtype == HF else BF
    d = _round(12, bs=3, T=64, H=1, G=2, D=128, act=act, dtype=dtype, lens=[0, 0, 5], tree=True, nodes=[64, 40, 64])
    d["masks"][0, ::3] = 0
    d["masks"][1, 7] = -(2 ** 63)  # node 63 only, which request 1 does not have
    d["masks"][2, 11] = 0  # its context remains
    d["masks"][0, 1] = -1
    out, lse = _call(d, device)
    _check(d, out, lse)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all()) and bool((lse[64 + 7] == -math.inf).all())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_nan_and_infinity_stay_with_the_nodes_that_see_them(device, dtype):
    """Window nodes whose keys or values are not finite: only the nodes that see them are touched."""
    d = _round(13, bs=2, T=20, H=1, G=2, D=64, act=dtype, dtype=dtype, lens=[50, 0], tree=False)
    k, v = d["cache"][:2]
    masks = torch.tensor([[1 << i for i in range(20)]] * 2, dtype=torch.int64)  # each sees itself alone
    d["masks"] = masks | 1
    at = d["page_table"].long()
    v[at[0, 50 + 3], 0, 5] = math.nan
    v[at[0, 50 + 4], 0, 6] = math.inf
    v[at[0, 50 + 5], 0, 7] = -math.inf
    k[at[0, 50 + 6], 0, 8] = math.nan
    v[at[1, 9], 0, :] = math.nan
    # slots that no request's window or context holds, and one that a page names past the end
    free = sorted(set(range(k.shape[0])) - set(at.flatten().tolist()))
    k[free], v[free] = math.nan, math.inf
    out, lse = _call(d, device)
    o = out.cpu().view(2, 20, 2, 64)
    assert bool(torch.isnan(o[0, 3, :, 5]).all()) and bool((o[0, 4, :, 6] == math.inf).all())
    assert bool((o[0, 5, :, 7] == -math.inf).all()) and bool(torch.isnan(o[0, 6]).all())
    assert bool(torch.isnan(o[1, 9]).all())
    hurt = torch.zeros(2, 20, dtype=torch.bool)
    hurt[0, 3:7] = True
    hurt[1, 9] = True
    args = {n: x for n, x in d.items() if n not in ("q", "cache")}
    want, wl, otol, ltol = R.attention(d["q"], *d["cache"], **args)
    fine = ~hurt.flatten()
    assert bool(torch.isfinite(out.cpu()[fine]).all())
    R.close(out.cpu()[fine], want[fine], otol[fine])
    R.close(lse.cpu()[fine], wl[fine], ltol[fine])
    rest = torch.ones(64, dtype=torch.bool)
    rest[5] = False
    R.close(o[0, 3][:, rest], want.view(2, 20, 2, 64)[0, 3][:, rest], otol.view(2, 20, 2, 64)[0, 3][:, rest])


@pytest.mark.parametrize("dtype", [E4, I8])
def test_attention_a_poisoned_row_of_a_quantised_cache(device, dtype):
    """A scale of NaN (a row that was not finite when it was written) reaches only the nodes that see it, and an
    e4m3 code that is NaN likewise."""
    d = _round(14, bs=1, T=9, H=1, G=1, D=64, act=BF, dtype=dtype, lens=[20], tree=False)
    d["masks"] = torch.tensor([[1 << i for i in range(9)]], dtype=torch.int64)
    k, v, ks, vs = d["cache"]
    at = d["page_table"][0].long()
    vs[at[20 + 2]] = math.nan
    ks[at[20 + 4]] = math.nan
    if dtype == E4:
        v.view(torch.uint8)[at[20 + 6], 0, 3] = 0x7F
    out, lse = _call(d, device)
    bad = torch.isnan(out.cpu().float())[:, 0]
    assert bool(bad[2].all()) and bool(bad[4].all()) and bool(bad[6, 3]) == (dtype == E4)
    want, wl, otol, ltol = R.attention(d["q"], k, v, ks, vs, **{n: x for n, x in d.items() if n not in ("q", "cache")})
    fine = [0, 1, 3, 5, 7, 8]
    R.close(out.cpu()[fine], want[fine], otol[fine])
    R.close(lse.cpu()[fine], wl[fine], ltol[fine])


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_bad_slots_hold_nothing(device, dtype):
    """Slots outside the cache, in the context and in the window, and a table that ends before the window."""
    d = _round(15, bs=3, T=6, H=2, G=2, D=128, act=BF, dtype=dtype, lens=[100, 70, 0], tree=False)
    t = d["page_table"]
    t[0, 3], t[0, 40], t[0, 99], t[0, 102] = -1, 1 << 30, -(2 ** 31), d["cache"][0].shape[0]
    t[2, :] = -1
    d["page_table"] = t[:, :73].contiguous()
    _check(d, *_call(d, device))


def test_attention_strides(device):
    """Keys and values interleaved in one tensor, heads before slots, q and out as slices of wider rows, a page
    table with wide rows, scales in the other order."""
    from dspine_amd.kernels.attention import tree_attention
    from dspine_amd.kernels.cache import KVCache

    for dtype in (BF, I8):
        d = _round(16, bs=2, T=5, H=3, G=2, D=64, act=BF, dtype=dtype, lens=[65, 190], tree=True)
        k, v, ks, vs = (None if x is None else x.to(device) for x in d["cache"])
        n = k.shape[0]
        both = torch.zeros((n, 3, 2, 64), dtype=dtype, device=device)
        both.view(torch.uint8)[:] = 0x7F
        both[:, :, 0], both[:, :, 1] = k, v
        heads_first = torch.empty((3, n, 64), dtype=dtype, device=device)
        heads_first.copy_(v.transpose(0, 1))
        if ks is not None:
            ks, vs = ks.t().contiguous().t(), torch.stack((vs, vs), -1)[..., 0]
        table = torch.full((2, 400), -7, dtype=torch.int32, device=device)
        table[:, 1: 1 + d["page_table"].shape[1]] = d["page_table"].to(device)
        q = torch.full((10, 10, 64), math.nan, dtype=BF, device=device)
        q[:, 2:8] = d["q"].to(device)
        args = dict(T=5, prefix_lens=d["prefix_lens"].to(device), masks=d["masks"].to(device),
                    page_table=table[:, 1: 1 + d["page_table"].shape[1]])
        for vv in (both[:, :, 1], heads_first.transpose(0, 1)):
            out = torch.full((10, 8, 64), 7.0, dtype=BF, device=device)
            lse = torch.empty((10, 6), device=device)
            tree_attention(q[:, 2:8], KVCache(both[:, :, 0], vv, ks, vs), out=out[:, 1:7], lse=lse, **args)
            assert bool((out[:, 0] == 7).all()) and bool((out[:, 7] == 7).all())
            _check(d, out[:, 1:7], lse)


def test_attention_scale_and_large_scores(device):
    """A caller's scale (negative, zero), and scores far beyond exp's range."""
    for scale in (-0.3, 0.0, 1.0, 40.0):
        d = _round(17, bs=2, T=7, H=1, G=4, D=128, act=BF, dtype=BF, lens=[90, 333], tree=True)
        d["scale"] = scale
        _check(d, *_call(d, device))


def test_attention_rising_and_falling_scores(device):
    """Scores that grow (the running maximum moves at every step) or shrink along the context."""
    for sign in (1.0, -1.0):
        d = _round(18, bs=1, T=3, H=2, G=2, D=64, act=HF, dtype=HF, lens=[1500], tree=False)
        k = d["cache"][0]
        d["q"][..., 0] = 8.0
        p = torch.arange(1503)
        k[d["page_table"][0].long(), :, 0] = (sign * p / 100.0).to(HF).unsqueeze(-1)
        _check(d, *_call(d, device))


def test_attention_offsets_past_32_bits(device):
    """A cache of more than 2^31 elements whose last slots are used."""
    slots, H, D = (1 << 21) + 64, 8, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB of free device memory")
    from dspine_amd.kernels.attention import tree_attention
    from dspine_amd.kernels.cache import KVCache, read_kv, write_kv

    g = _gen(19)
    k, v = (torch.zeros((slots, H, D), dtype=I8, device=device) for _ in range(2))
    ks, vs = (torch.zeros((slots, H), device=device) for _ in range(2))
    cache = KVCache(k, v, ks, vs)
    n = 40
    at = torch.cat((torch.arange(slots - 30, slots), torch.arange(10)))[torch.randperm(n, generator=g)]
    x, y = (torch.randn(n, H, D, generator=g).to(BF) for _ in range(2))
    write_kv(cache, x.to(device), y.to(device), at.to(device))
    small = tuple(t[at.to(device)].cpu() for t in (k, v, ks, vs))
    assert bool((small[2] > 0).all())
    back = read_kv(cache, at.to(device), dtype=torch.float32)[0].cpu()
    R.close(back, R.values(small[0], small[2]), R.values(small[0], small[2]).abs() * R.U32)
    d = dict(q=torch.randn(2, 8, D, generator=g).to(BF), cache=small, T=2,
             page_table=torch.arange(n, dtype=torch.int32).unsqueeze(0), prefix_lens=torch.tensor([n - 2], dtype=torch.int32))
    lse = torch.empty((2, 8), device=device)
    out = tree_attention(d["q"].to(device), cache, T=2, page_table=at.to(torch.int32).unsqueeze(0).to(device),
                         prefix_lens=d["prefix_lens"].to(device), lse=lse)
    _check(d, out, lse)


def test_attention_is_the_same_each_time_and_on_any_stream(device):
    d = _round(20, bs=4, T=17, H=2, G=4, D=128, act=BF, dtype=E4, lens=[2000, 31, 640, 5], tree=True)
    first = _call(d, device)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    runs = []
    for s in streams * 3:  # calls that may run at once
        with torch.cuda.stream(s):
            runs.append(_call(d, device))
    torch.cuda.synchronize()
    for r in runs:
        assert torch.equal(r[0], first[0]) and torch.equal(r[1], first[1])


def test_round_in_a_graph(device):
    """A whole round (masks, write, attention, acceptance, commit) captured once and replayed on changing inputs with
    eager work between: every replay equals the eager round."""
    from dspine_amd.kernels.attention import tree_attention
    from dspine_amd.kernels.cache import KVCache, new_cache, read_kv, write_kv
    from dspine_amd.runtime.worker import commit_accept
    from dspine_amd.verification.tree import accept_greedy_tree, tree_masks

    bs, T, H, G, D, V, L = 3, 9, 2, 2, 64, 500, 300
    g = torch.Generator(device=device).manual_seed(3)
    cache = new_cache(1000, H, D, dtype=E4, device=device)
    write_kv(cache, *(torch.randn(1000, H, D, generator=g, device=device).to(BF) for _ in range(2)),
             torch.arange(1000, device=device))
    s = dict(q=torch.zeros(bs * T, H * G, D, dtype=BF, device=device),
             k=torch.zeros(bs * T, H, D, dtype=BF, device=device), v=torch.zeros(bs * T, H, D, dtype=BF, device=device),
             parents=torch.zeros(bs, T, dtype=torch.int32, device=device),
             prefix=torch.zeros(bs, dtype=torch.int32, device=device),
             logits=torch.zeros(bs * T, V, device=device), tokens=torch.zeros(bs, T, dtype=torch.int64, device=device),
             table=torch.zeros(bs, L, dtype=torch.int32, device=device),
             loc=torch.zeros(bs * T, dtype=torch.int64, device=device))

    def one_round(c, s):
        masks, depths = tree_masks(s["parents"])
        write_kv(c, s["k"], s["v"], s["loc"])
        lse = torch.empty(bs * T, H * G, device=device)
        out = tree_attention(s["q"], c, T=T, page_table=s["table"], prefix_lens=s["prefix"], masks=masks, lse=lse)
        outs, path = accept_greedy_tree(candidates=s["tokens"], parents=s["parents"], next_token_logits=s["logits"],
                                        prefix_lens=s["prefix"])
        seq = torch.zeros(bs, dtype=torch.int64, device=device)
        free, count = commit_accept(outs, prefix_lens=s["prefix"], req_pool_indices=torch.arange(bs, device=device),
                                    req_to_token=s["table"], seq_lens=seq, path=path,
                                    free_slots=torch.zeros(bs * T, dtype=torch.int64, device=device))
        back = read_kv(c, s["loc"])
        return [masks, depths, out, lse, *outs, path, seq, free, count, s["table"], *back]

    def fill(seed):
        c = _gen(seed)
        i = torch.arange(T)
        p = (i - 1 - (torch.rand(bs, T, generator=c) * torch.clamp(i, max=3)).long()).clamp(min=0)
        p[:, 0] = -1
        perm = torch.randperm(1000, generator=c)[: bs * L].view(bs, L)
        prefix = torch.randint(0, L - T, (bs,), generator=c)
        logits = torch.randn(bs * T, V, generator=c)
        top = logits.argmax(-1).view(bs, T)
        new = dict(parents=p.to(torch.int32), prefix=prefix.to(torch.int32), logits=logits,
                   tokens=torch.gather(top, 1, p.clamp(min=0)), table=perm.to(torch.int32),
                   loc=torch.stack([perm[b, prefix[b]: prefix[b] + T] for b in range(bs)]).flatten(),
                   q=torch.randn(bs * T, H * G, D, generator=c).to(BF), k=torch.randn(bs * T, H, D, generator=c).to(BF),
                   v=torch.randn(bs * T, H, D, generator=c).to(BF))
        return {n: x.to(device) for n, x in new.items()}

    for n, x in fill(100).items():
        s[n].copy_(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        one_round(cache, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = one_round(cache, s)
    for seed in range(4):
        new = fill(seed)
        twin = KVCache(*(t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
        want = [t.clone() for t in one_round(twin, {n: x.clone() for n, x in new.items()})]
        for n, x in new.items():
            s[n].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)
        assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8))


# ---------------------------------------------------------------------------------------------
# write and read
# ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("act", [BF, HF])
@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("n, H, D", [(1, 1, 16), (7, 3, 80), (40, 2, 128), (129, 5, 192), (33, 8, 256), (1000, 1, 64)])
def test_write_quantises(device, n, H, D, dtype, act):
    from dspine_amd.kernels.cache import new_cache, read_kv, write_kv

    g = _gen(n + H + D)
    x, y = (torch.randn(n, H, D, generator=g).mul(torch.exp2(torch.randint(-9, 9, (n, H, 1), generator=g))).to(act)
            for _ in range(2))
    x[0, 0] = 0
    y[n - 1, H - 1, D - 1] = 700.0
    cache = new_cache(n + 9, H, D, dtype=dtype, device=device)
    slots = torch.randperm(n + 9, generator=g)[:n]
    write_kv(cache, x.to(device), y.to(device), slots.to(device))
    rest = torch.ones(n + 9, dtype=torch.bool)
    rest[slots] = False
    for src, codes, scale in ((x, cache.k.cpu(), cache.k_scale.cpu()), (y, cache.v.cpu(), cache.v_scale.cpu())):
        assert bool((codes[rest].float() == 0).all()) and bool((scale[rest] == 0).all())
        want, ratio = R.quantise(src, dtype)
        zero = want == 0
        got = scale[slots].double()
        assert bool((got[zero] == 0).all()) and bool((codes[slots].float()[zero] == 0).all())
        # 1 / top and the product: two roundings
        assert bool(((got - want).abs() <= 2 * R.U32 * 1.01 * want).all())
        c = codes[slots].float().double()[~zero]
        r = ratio[~zero]
        slack = 4 * R.U32 * r.abs()  # the reciprocal, its product and x's product
        if dtype == I8:
            assert bool(((c - r).abs() <= 0.5 + slack).all())
        else:  # half a step: 2^-4 of a normal value, half of 2^-9 below 2^-6
            assert bool(((c - r).abs() <= torch.clamp(r.abs() * 2.0 ** -4, min=2.0 ** -10) + slack).all())
        assert c.numel() == 0 or float(c.abs().max()) == R.TOP[dtype]
    for to in (torch.float32, BF, HF):
        k, v = read_kv(cache, slots.to(device), dtype=to)
        for got, codes, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
            want = codes.cpu()[slots].float() * scale.cpu()[slots].unsqueeze(-1)
            assert got.dtype == to and torch.equal(got.cpu(), want.to(to))


def test_write_follows_the_formula_exactly(device):
    """The codes and scales bit for bit as the documented float32 steps give them."""
    from dspine_amd.kernels.cache import new_cache, write_kv

    x = (torch.randn(500, 4, 128, generator=_gen(2)) * 3).to(BF)
    for dtype in (E4, I8):
        cache = new_cache(500, 4, 128, dtype=dtype, device=device)
        write_kv(cache, x.to(device), x.to(device), torch.arange(500, device=device, dtype=torch.int32))
        amax = x.float().abs().amax(-1)
        top = torch.tensor(R.TOP[dtype])
        y = x.float() * ((torch.ones(()) / amax) * top).unsqueeze(-1)
        codes = y.to(E4) if dtype == E4 else y.round().to(I8)
        assert torch.equal(cache.k_scale.cpu(), amax * (torch.ones(()) / top))
        assert torch.equal(cache.k.cpu().view(torch.uint8), codes.view(torch.uint8))
        assert torch.equal(cache.v.view(torch.uint8), cache.k.view(torch.uint8))


@pytest.mark.parametrize("dtype", [E4, I8])
def test_write_of_rows_that_are_not_finite_or_tiny(device, dtype):
    from dspine_amd.kernels.cache import new_cache, read_kv, write_kv

    x = torch.ones(6, 1, 32, dtype=BF)
    x[0, 0, 3], x[1, 0, 31], x[2, 0, 0] = math.nan, math.inf, -math.inf
    x[3] = 1e-38
    x[4] = 2.0 ** -100
    cache = new_cache(6, 1, 32, dtype=dtype, device=device)
    slots = torch.arange(6, device=device)
    write_kv(cache, x.to(device), x.to(device), slots)
    k, v = (t.cpu() for t in read_kv(cache, slots, dtype=torch.float32))
    assert bool(torch.isnan(k[:3]).all()) and bool((cache.k.cpu()[:4].float() == 0).all())
    assert bool((k[3] == 0).all()) and torch.allclose(k[4], torch.tensor(2.0 ** -100), rtol=1e-6) and torch.equal(k[4:], v[4:])
    assert bool((k[5] - 1).abs().max() <= 4 * R.U32)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_write_and_read_of_a_16_bit_cache(device, dtype):
    """A copy of the bits (NaN payloads among them), and reads rounded once to the other types."""
    from dspine_amd.kernels.cache import KVCache, read_kv, write_kv

    bits = torch.randint(-(1 << 15), 1 << 15, (50, 3, 48), generator=_gen(4), dtype=torch.int16)
    x = bits.view(dtype)
    cache = KVCache(*(torch.zeros(60, 3, 48, dtype=dtype, device=device) for _ in range(2)))
    slots = torch.randperm(60, generator=_gen(5))[:50].to(device)
    write_kv(cache, x.to(device), x.flip(0).to(device), slots)
    assert torch.equal(cache.k[slots].cpu().view(torch.int16), bits)
    assert torch.equal(cache.v[slots].cpu().view(torch.int16), bits.flip(0))
    for to in (torch.float32, BF, HF):
        k, _ = read_kv(cache, slots, dtype=to)
        want = x.float().to(to)
        same = (k.cpu() == want) | (torch.isnan(k.cpu()) & torch.isnan(want))
        assert bool(same.all())


def test_write_and_read_skip_bad_slots_and_read_repeats(device):
    from dspine_amd.kernels.cache import new_cache, read_kv, write_kv

    for dtype in (BF, I8):
        cache = new_cache(5, 2, 64, dtype=dtype, device=device)
        x = torch.randn(6, 2, 64, generator=_gen(6)).to(BF).to(device)
        for index in (torch.int32, torch.int64):
            write_kv(cache, x, x, torch.tensor([-1, 3, 5, 1 << 30, 0, -(1 << 31)], dtype=index, device=device))
            k, v = read_kv(cache, torch.tensor([3, 0, 3, -1, 5, 1, 3], dtype=index, device=device), dtype=torch.float32)
            assert torch.equal(k, v) and torch.equal(k[0], k[2]) and torch.equal(k[0], k[6])
            assert bool((k[3:6] == 0).all()) and bool((k[:2] != 0).any(-1).all())
            step = 0.5 / 127 * x.float().abs().amax(-1, keepdim=True) * 1.001 if dtype == I8 else 0.0
            assert bool(((k[0] - x[1].float()).abs() <= (step[1] if dtype == I8 else 0.0)).all())
            assert bool(((k[1] - x[4].float()).abs() <= (step[4] if dtype == I8 else 0.0)).all())
    empty = torch.zeros(0, dtype=torch.int64, device=device)
    write_kv(cache, x[:0], x[:0], empty)
    assert read_kv(cache, empty)[0].shape == (0, 2, 64)


def test_write_of_strided_rows_into_a_strided_cache(device):
    """Slices of a fused projection into an interleaved cache with its scales in the other order."""
    from dspine_amd.kernels.cache import KVCache, new_cache, write_kv

    n, H, D = 37, 3, 96
    qkv = torch.randn(n, 4 * H, D, generator=_gen(7)).to(HF).to(device)
    k, v = qkv[:, H: 2 * H], qkv[:, 3 * H:]
    slots = torch.randperm(n, generator=_gen(8)).to(device)
    for dtype in (HF, E4, I8):
        plain = new_cache(n, H, D, dtype=dtype, device=device)
        write_kv(plain, k.contiguous(), v.contiguous(), slots)
        both = torch.zeros((H, n, 2, D), dtype=dtype, device=device)
        scales = None if dtype == HF else torch.zeros((H, 2, n), device=device)
        odd = KVCache(both[:, :, 0].transpose(0, 1), both[:, :, 1].transpose(0, 1),
                      *(() if dtype == HF else (scales[:, 0].t(), scales[:, 1].t())))
        write_kv(odd, k, v, slots)
        for a, b in zip((plain.k, plain.v, plain.k_scale, plain.v_scale), (odd.k, odd.v, odd.k_scale, odd.v_scale)):
            assert a is None or torch.equal(a.float(), b.float())


# ---------------------------------------------------------------------------------------------
# trees
# ---------------------------------------------------------------------------------------------


def _random_parents(g, bs, T):
    i = torch.arange(T)
    p = (i - 1 - (torch.rand(bs, T, generator=g) * torch.clamp(i, max=8)).long()).clamp(min=0)
    p[:, 0] = -1
    return p.to(torch.int32)


@pytest.mark.parametrize("bs, T", [(1, 1), (5, 2), (9, 17), (3, 63), (130, 64)])
def test_tree_masks(device, bs, T):
    from dspine_amd.verification.tree import tree_masks

    p = _random_parents(_gen(bs), bs, T)
    p[0] = torch.arange(T) - 1  # a chain
    if bs > 2:
        p[1, 1:] = 0  # a star
        p[2, T // 2] = -1  # a second root
        p[2, T - 1] = T + 5  # not an earlier node
    masks, depths = tree_masks(p.to(device))
    want, deep = R.tree_masks(p)
    assert masks.tolist() == [[R.signed(m) for m in row] for row in want]
    assert depths.tolist() == deep


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("bs, T, V, ragged", [(1, 1, 7, False), (3, 2, 16385, True), (4, 17, 4099, True),
                                              (64, 17, 1000, False), (2, 64, 40003, True), (1, 25, 151936, False)])
def test_accept_greedy_tree(device, bs, T, V, ragged, dtype):
    from dspine_amd.verification.tree import accept_greedy_tree

    g = _gen(bs * 100 + T)
    # few distinct values: the row's largest is met several times
    logits = torch.randint(-40, 40, (bs * T, V), generator=g).to(dtype)
    logits[0] = -math.inf
    logits[-1] = 0.0
    logits[-1, V // 2:] = -0.0
    top1 = torch.stack([row.double().eq(row.double().max()).nonzero()[0, 0] for row in logits]).view(bs, T)
    p = _random_parents(g, bs, T)
    tokens = torch.gather(top1, 1, p.long().clamp(min=0))
    miss = torch.rand(bs, T, generator=g) < 0.3
    tokens[miss] = torch.randint(0, V, (bs, T), generator=g)[miss]
    if T > 3:
        p[0, 3] = -1  # a second root, never accepted
    prefix = torch.randint(0, 5000, (bs,), generator=g, dtype=torch.int64).to(torch.int32)
    lens = torch.randint(0, T + 2, (bs,), generator=g, dtype=torch.int64).to(torch.int32) if ragged else None
    # rows apart by more than their length
    wide = torch.full((bs * T, V + 3), math.nan, dtype=dtype)
    wide[:, :V] = logits
    outs, path = accept_greedy_tree(candidates=tokens.to(device), parents=p.to(device),
                                    next_token_logits=wide.to(device)[:, :V], prefix_lens=prefix.to(device),
                                    verify_lens=None if lens is None else lens.to(device))
    got = list(zip(*(t.tolist() for t in (*outs, path))))
    assert got == [tuple(r) for r in R.accept_tree(tokens, p, top1, prefix, lens)]


def test_accept_greedy_tree_of_a_chain_is_accept_greedy(device):
    from dspine_amd.verification.caps import accept_greedy
    from dspine_amd.verification.tree import accept_greedy_tree

    bs, T, V = 40, 17, 33000
    g = torch.Generator(device=device).manual_seed(1)
    logits = torch.randn(bs * T, V, generator=g, device=device).to(BF)
    top1 = torch.empty((bs, T), dtype=torch.int64, device=device)
    chain = (torch.arange(T, device=device, dtype=torch.int32) - 1).expand(bs, -1).contiguous()
    zero = torch.zeros(bs, T, dtype=torch.int64, device=device)
    prefix = torch.arange(bs, dtype=torch.int32, device=device)
    accept_greedy(candidates=zero, next_token_logits=logits, prefix_lens=prefix, top1=top1)
    tokens = torch.cat((zero[:, :1], top1[:, :-1]), 1)
    for b in range(bs):
        tokens[b, 1 + b % (T - 1)] += b % 3
    want = accept_greedy(candidates=tokens, next_token_logits=logits, prefix_lens=prefix)
    got, path = accept_greedy_tree(candidates=tokens, parents=chain, next_token_logits=logits, prefix_lens=prefix)
    for k in (0, 1, 2, 4):
        assert torch.equal(got[k], want[k])
    for b, a in enumerate(got[0].tolist()):
        assert got[3][b, : a + 1].tolist() == want[3][b, : a + 1].tolist() and not bool(got[3][b, a + 1:].any())
        assert path[b].tolist() == list(range(a + 1)) + [-1] * (T - a - 1)


@pytest.mark.parametrize("mode", ["window_slots", "in_table", "compact_slots"])
@pytest.mark.parametrize("bs, T", [(1, 1), (37, 17), (1500, 64)])
def test_commit_of_a_path(device, bs, T, mode):
    from dspine_amd.runtime.worker import commit_accept

    g = _gen(bs + T)
    lens = torch.randint(1, T + 1, (bs,), generator=g, dtype=torch.int64).to(torch.int32)
    path = torch.full((bs, T), -1, dtype=torch.int32)
    accept = torch.zeros(bs, dtype=torch.int32)
    for b in range(bs):
        n = int(lens[b])
        rest = (torch.randperm(n - 1, generator=g)[: int(torch.randint(0, n, (1,), generator=g))] + 1).sort()[0]
        accept[b] = rest.numel()
        path[b, 0] = 0
        path[b, 1: 1 + rest.numel()] = rest
    prefix = torch.randint(0, 200, (bs,), generator=g, dtype=torch.int64)
    prefix[0] = 222  # positions past the table's columns are not written
    cols, pool = 230, bs + 5
    rows = torch.randperm(pool, generator=g)[:bs]
    ocl = torch.randperm(1 << 20, generator=g)[: bs * T].to(torch.int64)
    table = torch.randint(0, 1 << 20, (pool, cols), generator=g, dtype=torch.int64).to(torch.int32)
    offs = None
    if mode == "compact_slots":
        offs = lens.to(torch.int64).cumsum(0) - lens
        ocl = ocl[: int(lens.sum())].contiguous()
    ref, seq = table.tolist(), [0] * pool
    freed = R.commit_tree(accept.tolist(), path.tolist(), prefix.tolist(), rows.tolist(), ref, T,
                          out_cache_loc=None if mode == "in_table" else ocl.tolist(), verify_lens=lens.tolist(),
                          slot_offsets=None if offs is None else offs.tolist(), seq_lens=seq)
    d_table, d_seq = table.to(device), torch.zeros(pool, dtype=torch.int32, device=device)
    outs = (accept.to(device), None, None, torch.empty((bs, T), device=device, dtype=torch.int64), None)
    free, count = commit_accept(outs, prefix_lens=prefix.to(device), req_pool_indices=rows.to(device),
                                req_to_token=d_table, out_cache_loc=None if mode == "in_table" else ocl.to(device),
                                verify_lens=lens.to(device), slot_offsets=None if offs is None else offs.to(device),
                                seq_lens=d_seq, path=path.to(device))
    n = int(count.item())
    assert free[:n].tolist() == freed
    assert d_table.tolist() == ref and d_seq.tolist() == seq
