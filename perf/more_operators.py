"""What the performance of the long-context operators is measured on: attention over the blocks of
a cache that a cheap score selects, and the life of the cache's pages around it, each through its
public entry points, with inputs made on the GPU from a seed.

A case's ``kind`` names the calls of a pass:

  index    index_blocks: the least and largest key elements of the blocks that a round or a prompt completed
  score    score_blocks: an upper bound of every block's attention scores from its index and the queries
  select   select_blocks: the best blocks of each (request, cache head), in ascending order
  attend   block_attention: drafted nodes over the selected blocks, the unfinished block and the window
  branch   fork_requests, then free_requests: winning samples forked into new rows, losing ones freed
  compact  compact_requests: the used slots of a fragmented pool moved to its front, in every layer's cache

``run`` computes them in elementary torch operations, in 32 bits, or (``own``) through the
package's entry points.
"""

from __future__ import annotations

import math

import torch

DEV = "cuda"
own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
BYTES = {"bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}
TOP_CODE = {"e4m3": 448.0, "int8": 127.0}  # the largest magnitude of a code

# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------


def listed():
    return [
        # after a round: 64 requests grew by up to 17 tokens, about one in seven completed a block
        dict(name="index_round_64x17", kind="index", bs=64, grow=17, Hkv=8, D=128, B=64, lo=500, hi=4000, dtype="bf16",
             cache="bf16"),
        # four prompts just written into an 8-bit float cache
        dict(name="index_prompt_4x32k_e4m3", kind="index", bs=4, grow=0, Hkv=8, D=128, B=64, lo=8000, hi=32000,
             dtype="bf16", cache="e4m3"),
        # one interactive user, a single token over a long document: launch bound
        dict(name="score_1x1_32k", kind="score", bs=1, T=1, Hkv=8, G=4, D=128, B=64, lo=32000, hi=32000, dtype="bf16",
             ragged=False),
        # a busy server's round of drafts (4 to 17 on compact rows) over long contexts
        dict(name="score_64x17_64k", kind="score", bs=64, T=17, Hkv=8, G=4, D=128, B=64, lo=8000, hi=64000,
             dtype="bf16", ragged=True),
        # one request's heads, 500 blocks each
        dict(name="select_1x8_500", kind="select", bs=1, Hkv=8, B=64, NB=500, lo=32000, hi=32000, count=32, first=1,
             last=2),
        # a busy server's heads over very long contexts
        dict(name="select_64x8_2000", kind="select", bs=64, Hkv=8, B=64, NB=2000, lo=8000, hi=128000, count=64, first=1,
             last=4),
        # one interactive user, a single token over 32 blocks of a long document
        dict(name="attend_1x1_32k", kind="attend", bs=1, T=1, Hkv=8, G=4, D=128, B=64, count=32, lo=32000, hi=32000,
             dtype="bf16", cache="bf16", tree=False, ragged=False),
        # a busy server's round of drafted trees over 64 blocks a head
        dict(name="attend_64x17_32k", kind="attend", bs=64, T=17, Hkv=8, G=4, D=128, B=64, count=64, lo=8000, hi=32000,
             dtype="bf16", cache="bf16", tree=True, ragged=True),
        # one question's four samples, two of them pruned
        dict(name="branch_1x4_700", kind="branch", groups=1, wide=4, kids=1, lo=700, hi=700, tail=40),
        # 64 questions' samples over long prompts
        dict(name="branch_64x4_20k", kind="branch", groups=64, wide=4, kids=1, lo=8000, hi=30000, tail=900),
        # a small server's pool before it is shrunk: odd counts, an 8-bit integer cache of two layers
        dict(name="compact_7x1500_int8", kind="compact", bs=7, Hkv=3, D=96, layers=2, slots=14001, lo=300, hi=2701,
             dtype="bf16", cache="int8"),
        # a large pool, 16-bit caches of four layers
        dict(name="compact_64x2k_bf16", kind="compact", bs=64, Hkv=8, D=128, layers=4, slots=200000, lo=1000, hi=3000,
             dtype="bf16", cache="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["index", "score", "select", "attend", "attend", "branch", "compact"])
    c = dict(kind=kind)
    if kind in ("index", "score", "attend"):
        dtype = rng.choice(["bf16", "bf16", "f16"])
        c.update(bs=_log(rng, 1, 64), Hkv=rng.choice([1, 2, 3, 4, 8, 8]), D=rng.choice([64, 80, 96, 128, 128, 192, 256]),
                 B=rng.choice([16, 32, 64, 64, 128]), dtype=dtype)
        if kind != "score":
            c.update(cache=rng.choice([dtype, dtype, "e4m3", "int8"]))
        if kind != "index":
            c.update(T=rng.choice([1, rng.randint(2, 64), rng.randint(2, 32), 17]), G=rng.choice([1, 2, 3, 4, 4, 5, 8, 16]),
                     ragged=rng.random() < 0.4)
    if kind == "index":
        c.update(grow=rng.choice([0, 1, 17, rng.randint(2, 64)]))
        hi = _log(rng, 64, 32000)
        while c["bs"] > 1 and c["bs"] * hi * c["Hkv"] * c["D"] > 8e7:
            c["bs"] = (c["bs"] + 1) // 2
        hi = min(hi, int(8e7 / (c["bs"] * c["Hkv"] * c["D"])))
        c.update(lo=rng.choice([hi, hi // 2, hi // 8, 0]), hi=hi)
        while work(c)["bytes"] == 0:  # (lengths at which no block was completed)
            c.update(lo=c["lo"] + 1, hi=c["hi"] + 1)
    elif kind == "score":
        hi = _log(rng, 64, 64000)
        while c["bs"] > 1 and c["bs"] * (hi // c["B"] + 1) * c["Hkv"] * c["D"] * max(1.0, c["T"] * c["G"] / 68) > 3.5e7:
            c["bs"] = (c["bs"] + 1) // 2
        most = 3.5e7 / (c["bs"] * c["Hkv"] * c["D"] * max(1.0, c["T"] * c["G"] / 68)) * c["B"]
        hi = max(64, min(hi, int(most)))
        c.update(lo=rng.choice([hi, hi // 2, hi // 8, 0]), hi=hi)
    elif kind == "select":
        B = rng.choice([16, 32, 64, 64, 128])
        NB = _log(rng, 2, 8000)
        count = min(NB, _log(rng, 1, 512))
        first = rng.choice([0, min(1, count)])
        c.update(bs=_log(rng, 1, 64), Hkv=rng.choice([1, 2, 3, 4, 8, 8]), B=B, NB=NB, count=count, first=first,
                 last=rng.randint(0, min(4, count - first)))
        while c["bs"] > 1 and c["bs"] * c["Hkv"] * NB > 1e6:
            c["bs"] //= 2
        c.update(lo=rng.choice([NB * B, NB * B // 2, 0]), hi=NB * B)
    elif kind == "attend":
        c.update(tree=rng.random() < 0.6)
        hi = _log(rng, 64, 32000)
        count = max(1, min(_log(rng, 1, 8192) // c["B"], hi // c["B"]))

        def costs(bs, seen):
            heads = bs * c["Hkv"]
            return max(heads * seen * c["D"] / 2.7e8, heads * c["G"] * c["T"] * seen / 1.4e8,
                       heads * c["G"] * c["T"] * seen * c["D"] / 1.8e10, bs * hi * c["Hkv"] * c["D"] / 1.3e9)

        while c["bs"] > 1 and costs(c["bs"], count * c["B"] + c["B"] + c["T"]) > 1:
            c["bs"] = (c["bs"] + 1) // 2
        while count > 1 and costs(c["bs"], count * c["B"] + c["B"] + c["T"]) > 1:
            count //= 2
        c.update(count=count, lo=rng.choice([hi, hi // 2, hi // 8, 0]), hi=hi)
    elif kind == "branch":
        groups, wide, kids, hi = _log(rng, 1, 64), rng.randint(2, 8), rng.randint(1, 3), _log(rng, 16, 30000)
        while groups > 1 and groups * (wide + kids * wide) * hi > 1.4e7:
            groups = (groups + 1) // 2
        c.update(groups=groups, wide=wide, kids=kids, lo=rng.choice([hi, hi // 2, 0]), hi=hi, tail=_log(rng, 1, 1000))
    else:
        dtype = rng.choice(["bf16", "f16"])
        bs, hi = _log(rng, 1, 64), _log(rng, 16, 20000)
        while bs > 1 and bs * hi > 120000:
            bs = (bs + 1) // 2
        c.update(bs=bs, Hkv=rng.choice([1, 2, 3, 4, 8]), D=rng.choice([64, 80, 96, 128, 192]), layers=rng.randint(1, 4),
                 lo=rng.choice([hi, hi // 2, 0]), hi=hi, dtype=dtype, cache=rng.choice([dtype, "e4m3", "int8"]))
        c.update(slots=int(bs * hi * rng.uniform(1.02, 2.5)) + 64)
        while c["layers"] > 1 and c["slots"] * c["layers"] * c["Hkv"] * c["D"] > 8e8:
            c["layers"] -= 1
    return c


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 41)


def _spread(lo, hi, n):
    """n lengths spread evenly over [lo, hi]."""
    return [int(lo + (hi - lo) * (i + 0.5) / n) for i in range(n)]


def _mixed(values):
    """The same values in another order, so that two spreads do not rise together."""
    n = len(values)
    step = next(s for s in (5, 7, 11, 13) if math.gcd(s, n) == 1)
    return [values[i * step % n] for i in range(n)]


def _lengths(c):
    """(context, nodes) of each request, before the seed's order."""
    bs, T = c["bs"], c.get("T", 1)
    nodes = _spread(max(1, T // 4), T + 1, bs) if c.get("ragged") else [T] * bs
    return list(zip(_spread(c["lo"], c["hi"], bs), _mixed(nodes)))


def _grown(c):
    """(length before, length after) of each request whose blocks are indexed."""
    to = _spread(c["lo"], c["hi"], c["bs"])
    if c["grow"] == 0:  # a prompt
        return [(0, t) for t in to]
    step = _mixed(_spread(1, c["grow"] + 1, c["bs"]))
    return [(max(0, t - g), t) for t, g in zip(to, step)]


def _activations(g, n, heads, dim, dtype):
    """Keys or values as a projection leaves them: a few channels of a head much larger than the rest."""
    gain = torch.ones(heads, dim, device=DEV)
    gain[:, torch.randint(0, dim, (max(1, dim // 32),), generator=g, device=DEV)] = 4.0
    return (torch.randn(n, heads, dim, generator=g, device=DEV) * gain).to(TYPES[dtype])


def _quantise(x, cache):
    """x [n, heads, dim] as (codes, scales), a scale for each (slot, head)."""
    x = x.float()
    scale = x.abs().amax(-1).clamp_(min=1e-20) / TOP_CODE[cache]
    codes = x / scale.unsqueeze(-1)
    return (codes.to(TYPES["e4m3"]) if cache == "e4m3" else codes.round().to(torch.int8)), scale


def _cache(g, slots, c):
    s = dict(k_scale=None, v_scale=None)
    for name in ("k", "v"):
        s[name] = _activations(g, slots, c["Hkv"], c["D"], c["dtype"])
        if c["cache"] in TOP_CODE:
            s[name], s[name + "_scale"] = _quantise(s[name], c["cache"])
    return s


def _table(g, lengths, width, extra):
    """(a page table whose rows hold ``lengths`` slots, the pool's size): three quarters of a request in one run of
    slots, what came later wherever slots were free."""
    total = torch.tensor(lengths, device=DEV)
    used = int(sum(lengths))
    slots = used + used // 8 + extra
    head = total * 3 // 4
    free = torch.randperm(slots - int(head.sum()), generator=g, device=DEV) + head.sum()
    pos = torch.arange(width, device=DEV).expand(len(lengths), -1)
    run = (head.cumsum(0) - head).unsqueeze(1) + pos
    tail = (total - head).cumsum(0) - (total - head)
    late = free[(tail.unsqueeze(1) + pos - head.unsqueeze(1)).clamp_(0, free.numel() - 1)]
    table = torch.where(pos < head.unsqueeze(1), run, late)
    return torch.where(pos < total.unsqueeze(1), table, torch.zeros_like(table)).to(torch.int32), slots


def _masks(g, bs, T):
    """Drafted trees as bits, a node seeing itself and its ancestors; its parent is one of the few nodes before it."""
    i = torch.arange(T, device=DEV)
    back = 1 + (torch.rand(bs, T, generator=g, device=DEV).square() * torch.clamp(i, max=6)).long()
    parents = (i - back).clamp_(min=0)
    masks = torch.ones(bs, T, dtype=torch.int64, device=DEV)
    for k in range(1, T):
        masks[:, k] = torch.gather(masks, 1, parents[:, k: k + 1])[:, 0] | (1 << k if k < 63 else -2 ** 63)
    return masks


def _round(g, c):
    """The seed's order of a round's lengths, and its compact rows."""
    lengths = _lengths(c)
    lengths = [lengths[i] for i in torch.randperm(c["bs"], generator=g, device=DEV).tolist()]
    ctx, nodes = [a for a, _ in lengths], [b for _, b in lengths]
    rows = sum(nodes) if c["ragged"] else c["bs"] * c["T"]
    held = torch.tensor(nodes, device=DEV)
    s = dict(prefix_lens=torch.tensor(ctx, device=DEV, dtype=torch.int32),
             verify_lens=held.to(torch.int32) if c["ragged"] else None,
             row_offsets=held.cumsum(0) - held if c["ragged"] else None,
             q=(1.5 * torch.randn(rows, c["Hkv"] * c["G"], c["D"], generator=g, device=DEV)).to(TYPES[c["dtype"]]))
    return s, ctx, nodes


def _family(c):
    """(prompt, tail) of each sample of a branch case, group after group."""
    prompts = _spread(c["lo"], c["hi"], c["groups"])
    tails = _mixed(_spread(0, c["tail"], c["groups"] * c["wide"]))
    return [(prompts[i // c["wide"]], tails[i]) for i in range(c["groups"] * c["wide"])]


def _winners(c):
    return max(1, c["wide"] // 2)


def _owned(c):
    """(slots of its own, slots it shares with the request before) of each request of a compact case."""
    lens = _mixed(_spread(c["lo"], c["hi"], c["bs"]))
    owned = []
    for i, n in enumerate(lens):
        lent = min(n // 4, lens[i - 1]) if i % 2 else 0
        owned.append((n - lent, lent))
    return owned


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=dict(c))
    if c["kind"] == "index":
        pairs = _grown(c)
        pairs = [pairs[i] for i in torch.randperm(c["bs"], generator=g, device=DEV).tolist()]
        table, slots = _table(g, [t for _, t in pairs], c["hi"] + 1, 64)
        per = c["hi"] // c["B"] + 1  # blocks of a table row
        rows = torch.randperm(c["bs"] * per + 7, generator=g, device=DEV)[: c["bs"] * per]
        s.update(cache=_cache(g, slots, c), page_table=table, block_table=rows.view(c["bs"], per).to(torch.int32),
                 from_lens=torch.tensor([a for a, _ in pairs], device=DEV, dtype=torch.int32),
                 to_lens=torch.tensor([b for _, b in pairs], device=DEV, dtype=torch.int32),
                 bounds=torch.zeros(c["bs"] * per + 7, c["Hkv"], 2, c["D"], device=DEV, dtype=TYPES[c["dtype"]]))
    elif c["kind"] == "score":
        more, ctx, _ = _round(g, c)
        per = max(1, c["hi"] // c["B"])
        rows = c["bs"] * per + 7
        # the elements of a block's keys lie around a value of the block's own
        mid = torch.randn(rows, c["Hkv"], 1, c["D"], generator=g, device=DEV)
        half = 1.0 + torch.rand(rows, c["Hkv"], 1, c["D"], generator=g, device=DEV)
        s.update(more, bounds=torch.cat((mid - half, mid + half), 2).to(TYPES[c["dtype"]]),
                 block_table=torch.randperm(rows, generator=g, device=DEV)[: c["bs"] * per].view(c["bs"], per).to(torch.int32))
    elif c["kind"] == "select":
        ctx = _spread(c["lo"], c["hi"], c["bs"])
        ctx = torch.tensor(ctx, device=DEV)[torch.randperm(c["bs"], generator=g, device=DEV)]
        scores = torch.randn(c["bs"], c["Hkv"], c["NB"], generator=g, device=DEV) * 3.0 + 20.0
        live = torch.arange(c["NB"], device=DEV) < (ctx // c["B"]).view(-1, 1, 1)
        s.update(scores=torch.where(live, scores, torch.full_like(scores, -math.inf)), prefix_lens=ctx.to(torch.int32))
    elif c["kind"] == "attend":
        more, ctx, nodes = _round(g, c)
        table, slots = _table(g, [a + b for a, b in zip(ctx, nodes)], c["hi"] + c["T"] + 32, 64)
        # each head's own blocks, the last ones among them
        full = more["prefix_lens"].long() // c["B"]
        per = max(1, c["hi"] // c["B"])
        j = torch.arange(per, device=DEV)
        want = torch.rand(c["bs"], c["Hkv"], per, generator=g, device=DEV) + (j >= full.view(-1, 1, 1) - 2)
        want = torch.where(j < full.view(-1, 1, 1), want, torch.full_like(want, -1.0))
        ids = want.argsort(-1, descending=True)[..., : c["count"]]
        ids = torch.where(torch.gather(want, -1, ids) >= 0, ids, per).sort(-1).values
        blocks = torch.full((c["bs"], c["Hkv"], c["count"]), -1, device=DEV)
        blocks[..., : ids.shape[-1]] = torch.where(ids < per, ids, -1)
        s.update(more, cache=_cache(g, slots, c), page_table=table, blocks=blocks.to(torch.int32),
                 masks=_masks(g, c["bs"], c["T"]) if c["tree"] else None)
    elif c["kind"] == "branch":
        family, wide, win = _family(c), c["wide"], _winners(c)
        n, kids = len(family), c["groups"] * win * c["kids"]
        cols = c["hi"] + c["tail"] + 8
        fresh = sum(p for p, _ in family[::wide]) + sum(t for _, t in family)
        pool = torch.randperm(fresh + fresh // 4 + 64, generator=g, device=DEV)
        prompt = torch.tensor([p for p, _ in family], device=DEV)
        tail = torch.tensor([t for _, t in family], device=DEV)
        lead = prompt[::wide]
        start = (lead.cumsum(0) - lead).repeat_interleave(wide)  # of the group's prompt
        late = lead.sum() + tail.cumsum(0) - tail
        pos = torch.arange(cols, device=DEV).expand(n, -1)
        at = torch.where(pos < prompt.unsqueeze(1), start.unsqueeze(1) + pos,
                         late.unsqueeze(1) + pos - prompt.unsqueeze(1))
        held = pos < (prompt + tail).unsqueeze(1)
        entries = pool[torch.where(held, at, torch.zeros_like(at))]
        row = torch.randperm(n + kids, generator=g, device=DEV)  # rows of the request pool
        table = torch.zeros(n + kids, cols, device=DEV, dtype=torch.int32)
        table[row[:n]] = torch.where(held, entries, torch.zeros_like(entries)).to(torch.int32)
        lens = torch.zeros(n + kids, device=DEV, dtype=torch.int32)
        lens[row[:n]] = (prompt + tail).to(torch.int32)
        shared = torch.zeros(pool.numel(), device=DEV, dtype=torch.int32)
        shared[pool[: int(lead.sum())]] = wide - 1
        rank = torch.rand(c["groups"], wide, generator=g, device=DEV).argsort(-1)
        best = (rank < win).flatten()
        s.update(req_to_token=table, seq_lens=lens, shared=shared, rows=row[:n][~best].contiguous(),
                 parents=row[:n][best].repeat_interleave(c["kids"]), children=row[n:].contiguous(),
                 free_slots=torch.full((pool.numel(),), -1, device=DEV, dtype=torch.int64))
    else:
        owned = _owned(c)
        n, cols = c["bs"], c["hi"] + 9
        pool = torch.randperm(c["slots"], generator=g, device=DEV)
        mine = torch.tensor([a for a, _ in owned], device=DEV)
        theirs = torch.tensor([b for _, b in owned], device=DEV)
        start = mine.cumsum(0) - mine
        pos = torch.arange(cols, device=DEV).expand(n, -1)
        before = torch.roll(start, 1)
        at = torch.where(pos < theirs.unsqueeze(1), before.unsqueeze(1) + pos, start.unsqueeze(1) + pos - theirs.unsqueeze(1))
        held = pos < (mine + theirs).unsqueeze(1)
        entries = pool[torch.where(held, at, torch.zeros_like(at))]
        row = torch.randperm(n + 3, generator=g, device=DEV)
        table = torch.zeros(n + 3, cols, device=DEV, dtype=torch.int32)
        table[row[:n]] = torch.where(held, entries, torch.zeros_like(entries)).to(torch.int32)
        lens = torch.zeros(n + 3, device=DEV, dtype=torch.int32)
        lens[row[:n]] = (mine + theirs).to(torch.int32)
        shared = torch.zeros(c["slots"], device=DEV, dtype=torch.int32)
        lent = (pos < theirs.unsqueeze(1)) & held
        shared.index_add_(0, entries.flatten(), lent.flatten().to(torch.int32))
        s.update(req_to_token=table, seq_lens=lens, shared=shared, rows=row[:n].contiguous(),
                 moves=torch.full((2, c["slots"] // 2), -1, device=DEV, dtype=torch.int64),
                 caches=[_cache(g, c["slots"], c) for _ in range(c["layers"])])
    return s


def work(case):
    c = case
    if c["kind"] == "index":
        blocks = sum(b // c["B"] - a // c["B"] for a, b in _grown(c))
        keys = blocks * c["B"] * c["Hkv"]
        return {"bytes": keys * c["D"] * BYTES[c["cache"]] + (4 * keys if c["cache"] in TOP_CODE else 0)
                + blocks * (4 * c["B"] + c["Hkv"] * 2 * c["D"] * 2 + 4), "flops": 2 * keys * c["D"]}
    if c["kind"] == "score":
        lengths = _lengths(c)
        blocks, rows = sum(a // c["B"] for a, _ in lengths), sum(b for _, b in lengths)
        return {"bytes": blocks * (c["Hkv"] * (2 * c["D"] * 2 + 4) + 4) + rows * c["Hkv"] * c["G"] * c["D"] * 2,
                "flops": sum(4.0 * (a // c["B"]) * b for a, b in lengths) * c["Hkv"] * c["G"] * c["D"]}
    if c["kind"] == "select":
        scores = sum(min(a // c["B"], c["NB"]) for a in _spread(c["lo"], c["hi"], c["bs"])) * c["Hkv"]
        return {"bytes": 4 * scores + 4 * c["bs"] * c["Hkv"] * c["count"], "flops": scores}
    if c["kind"] == "attend":
        seen = [(min(c["count"], a // c["B"]) * c["B"] + a % c["B"], b) for a, b in _lengths(c)]
        positions, rows = sum(a + b for a, b in seen), sum(b for _, b in seen)
        per = 2 * c["D"] * BYTES[c["cache"]] + (8 if c["cache"] in TOP_CODE else 0) + 4
        return {"bytes": positions * c["Hkv"] * per + rows * c["Hkv"] * c["G"] * (2 * c["D"] * 2 + 4),
                "flops": 4.0 * c["D"] * c["Hkv"] * c["G"] * sum((a + 1) * b for a, b in seen)}
    if c["kind"] == "branch":
        family, wide, win = _family(c), c["wide"], _winners(c)
        prompts, tails = sum(p for p, _ in family[::wide]), sum(t for _, t in family)
        forked = c["kids"] * (win * prompts + tails * win // wide)
        freed = (wide - win) * prompts + tails * (wide - win) // wide
        # entries read and written, the counts of the slots that change, the freed slots
        return {"bytes": 8 * forked + 4 * freed + 8 * 2 * (prompts + tails) + 8 * tails * (wide - win) // wide,
                "flops": forked + freed}
    owned = _owned(c)
    used, entries = sum(a for a, _ in owned), sum(a + b for a, b in owned)
    moved = used * (c["slots"] - used) // c["slots"]  # slots in use lie anywhere
    row = c["Hkv"] * (2 * c["D"] * BYTES[c["cache"]] + (8 if c["cache"] in TOP_CODE else 0)) * c["layers"]
    return {"bytes": moved * (2 * row + 24) + 8 * entries, "flops": entries}


# ---------------------------------------------------------------------------------------------
# the passes
# ---------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _own(state)
    return {"index": _index, "score": _score, "select": _select, "attend": _attend, "branch": _branch,
            "compact": _compact}[state["case"]["kind"]](state)


def _own(s):
    c = s["case"]
    if c["kind"] in ("branch", "compact"):
        from dspine_amd.kernels.cache import KVCache
        from dspine_amd.runtime.requests import compact_requests, fork_requests, free_requests

        # (the counts and the lengths begin as they were in every pass)
        shared, lens = s["shared"].clone(), s["seq_lens"].clone()
        if c["kind"] == "branch":
            fork_requests(s["req_to_token"], lens, shared, s["parents"], s["children"])
            slots, count = free_requests(s["req_to_token"], lens, shared, s["rows"], free_slots=s["free_slots"])
            return dict(table=s["req_to_token"], lens=lens, shared=shared, free_slots=slots, free_count=count)
        table = s["req_to_token"].clone()
        moves, counts = compact_requests(table, lens, s["rows"], [KVCache(**x) for x in s["caches"]], shared=shared,
                                         moves=s["moves"])
        return dict(table=table, shared=shared, moves=moves, counts=counts,
                    caches=[{k: v for k, v in x.items() if v is not None} for x in s["caches"]])
    from dspine_amd.kernels.blocks import BlockIndex, block_attention, index_blocks, score_blocks, select_blocks
    from dspine_amd.kernels.cache import KVCache

    if c["kind"] == "index":
        index_blocks(BlockIndex(s["bounds"], c["B"]), KVCache(**s["cache"]), page_table=s["page_table"],
                     block_table=s["block_table"], from_lens=s["from_lens"], to_lens=s["to_lens"],
                     longest=c["grow"] or c["hi"])
        return dict(bounds=s["bounds"])
    if c["kind"] == "score":
        return dict(scores=score_blocks(s["q"], BlockIndex(s["bounds"], c["B"]), T=c["T"], block_table=s["block_table"],
                                        prefix_lens=s["prefix_lens"], verify_lens=s["verify_lens"],
                                        row_offsets=s["row_offsets"]))
    if c["kind"] == "select":
        return dict(blocks=select_blocks(s["scores"], c["count"], prefix_lens=s["prefix_lens"], block_size=c["B"],
                                         first=c["first"], last=c["last"]))
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=DEV)
    out = block_attention(s["q"], KVCache(**s["cache"]), T=c["T"], blocks=s["blocks"], block_size=c["B"],
                          page_table=s["page_table"], prefix_lens=s["prefix_lens"], verify_lens=s["verify_lens"],
                          row_offsets=s["row_offsets"], masks=s["masks"], lse=lse)
    return dict(out=out, lse=lse)


def _index(s):
    c = s["case"]
    B, H, D, cache = c["B"], c["Hkv"], c["D"], s["cache"]
    # the blocks that may have been completed: as many of each request as its growth can hold
    grow = c["grow"] or c["hi"]
    j = (s["from_lens"].long() // B).unsqueeze(1) + torch.arange((grow + B - 1) // B, device=DEV)
    done = j < (s["to_lens"].long() // B).unsqueeze(1)
    p = j.clamp(max=s["page_table"].shape[1] // B - 1).clamp(min=0).unsqueeze(-1) * B + torch.arange(B, device=DEV)
    p = p.clamp(max=s["page_table"].shape[1] - 1)
    at = torch.gather(s["page_table"].long(), 1, p.flatten(1)).view(*p.shape)
    keys = cache["k"][at].float()  # [bs, blocks, B, H, D]
    if cache["k_scale"] is not None:
        keys = keys * cache["k_scale"][at].unsqueeze(-1)
    bounds = torch.stack((keys.amin(2), keys.amax(2)), 3).to(TYPES[c["dtype"]])
    rows = torch.gather(s["block_table"].long(), 1, j.clamp(max=s["block_table"].shape[1] - 1))
    s["bounds"][rows[done]] = bounds[done]
    return dict(bounds=s["bounds"])


def _rows(s):
    """The nodes' rows [bs, T] and which of them are there."""
    c = s["case"]
    node = torch.arange(c["T"], device=DEV)
    nodes = torch.full((c["bs"],), c["T"], device=DEV) if s["verify_lens"] is None else s["verify_lens"].long()
    start = torch.arange(c["bs"], device=DEV) * c["T"] if s["row_offsets"] is None else s["row_offsets"]
    real = node < nodes.unsqueeze(1)
    return torch.where(real, start.unsqueeze(1) + node, torch.zeros_like(start).unsqueeze(1)), real, nodes


def _score(s):
    c = s["case"]
    bs, T, H, G, D = c["bs"], c["T"], c["Hkv"], c["G"], c["D"]
    rows, real, _ = _rows(s)
    q = s["q"].float()[rows].view(bs, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(bs, H, T * G, D)
    bounds = s["bounds"].float()[s["block_table"].long()]  # [bs, NB, H, 2, D]
    low = bounds[:, :, :, 0].permute(0, 2, 3, 1).contiguous()
    high = bounds[:, :, :, 1].permute(0, 2, 3, 1).contiguous()
    # an element adds the larger of its two products: with the largest key where the query is positive, else the least
    x = torch.matmul(q.clamp(min=0), high) + torch.matmul(q.clamp(max=0), low)
    x = x.view(bs, H, T, G, -1).masked_fill_(~real.view(bs, 1, T, 1, 1), -math.inf).amax((2, 3)) * (1.0 / math.sqrt(D))
    live = torch.arange(x.shape[-1], device=DEV) < (s["prefix_lens"].long() // c["B"]).view(-1, 1, 1)
    return dict(scores=x.masked_fill_(~live, -math.inf))


def _select(s):
    c = s["case"]
    NB = c["NB"]
    full = (s["prefix_lens"].long() // c["B"]).clamp(max=NB).view(-1, 1, 1)
    j = torch.arange(NB, device=DEV)
    live = j < full
    must = live & ((j < c["first"]) | (j >= full - c["last"]))
    x = torch.where(must, math.inf, torch.where(live, s["scores"], -math.inf))
    ids = x.sort(stable=True, dim=-1, descending=True).indices[..., : c["count"]]
    ids = torch.where(ids < full, ids, NB).sort(-1).values
    return dict(blocks=torch.where(ids < NB, ids, -1).to(torch.int32))


def _attend(s):
    c, cache = s["case"], s["cache"]
    bs, T, H, G, D, B = c["bs"], c["T"], c["Hkv"], c["G"], c["D"], c["B"]
    rows, real, nodes = _rows(s)
    prefix = s["prefix_lens"].long()
    blocks = s["blocks"].long()  # [bs, H, S]
    # the positions each head reads: its blocks', then those from the unfinished block on
    p = (blocks.clamp(min=0).unsqueeze(-1) * B + torch.arange(B, device=DEV)).flatten(2)
    there = (blocks >= 0).unsqueeze(-1).expand(*blocks.shape, B).flatten(2)
    late = (prefix // B * B).unsqueeze(1) + torch.arange(B + T, device=DEV)  # [bs, B + T]
    p = torch.cat((p, late.unsqueeze(1).expand(bs, H, -1)), 2)
    window = p - prefix.view(-1, 1, 1)  # the node at a position
    there = torch.cat((there, (late < (prefix + nodes).unsqueeze(1)).unsqueeze(1).expand(bs, H, -1)), 2)
    at = torch.gather(s["page_table"].long().unsqueeze(1).expand(bs, H, -1), 2,
                      p.clamp(max=s["page_table"].shape[1] - 1))
    head = torch.arange(H, device=DEV).view(1, H, 1)

    def values(name):
        x = cache[name][at, head].float()
        return x if cache[name + "_scale"] is None else x * cache[name + "_scale"][at, head].unsqueeze(-1)

    q = s["q"].float()[rows].view(bs, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(bs, H, T * G, D)
    scores = torch.matmul(q, values("k").transpose(2, 3).contiguous()).view(bs, H, T, G, -1) * (1.0 / math.sqrt(D))
    node = torch.arange(T, device=DEV)
    if s["masks"] is None:
        sees = window.unsqueeze(2) <= node.view(1, 1, T, 1)
    else:
        sees = (s["masks"].view(bs, 1, T, 1) >> window.clamp(0, 63).unsqueeze(2)) & 1 == 1
    sees = ((window < 0).unsqueeze(2) | sees) & there.unsqueeze(2)  # [bs, H, T, L]
    scores = scores.masked_fill_(~sees.unsqueeze(3), -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    del scores
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(bs, H, T * G, -1), values("v")).view(bs, H, T, G, D) / total
    lse = (top + torch.log(total))[..., 0]
    out = out.permute(0, 2, 1, 3, 4).reshape(bs, T, H * G, D)[real].to(s["q"].dtype)
    return dict(out=out, lse=lse.permute(0, 2, 1, 3).reshape(bs, T, H * G)[real])


def _held(table, lens, rows):
    """The entries [n, cols] of rows of a table, and which of them a request holds."""
    return table[rows], torch.arange(table.shape[1], device=DEV) < lens[rows].unsqueeze(1)


def _branch(s):
    table, shared, lens = s["req_to_token"], s["shared"].clone(), s["seq_lens"].clone()
    entries, held = _held(table, lens, s["parents"])
    table[s["children"]] = torch.where(held, entries, table[s["children"]])
    lens[s["children"]] = lens[s["parents"]]
    shared.index_add_(0, entries.flatten(), held.flatten().to(torch.int32))
    entries, held = _held(table, lens, s["rows"])
    lens[s["rows"]] = 0
    shared.index_add_(0, entries.flatten(), -held.flatten().to(torch.int32))
    freed = shared < 0
    slots = torch.arange(shared.numel(), device=DEV)[freed]
    s["free_slots"][: slots.numel()] = slots
    return dict(table=table, lens=lens, shared=shared.clamp_(min=0), free_slots=s["free_slots"],
                free_count=freed.sum().to(torch.int32).view(1))


def _compact(s):
    c = s["case"]
    table, shared, lens, n = s["req_to_token"].clone(), s["shared"].clone(), s["seq_lens"], c["slots"]
    entries, held = _held(table, lens, s["rows"])
    slot = torch.arange(n, device=DEV)
    hits = torch.zeros(n, device=DEV, dtype=torch.int32).index_add_(0, entries.flatten(), held.flatten().to(torch.int32))
    used = hits > 0
    count = used.sum()
    late, hole = used & (slot >= count), ~used & (slot < count)
    src, dst = slot[late], slot[hole]  # in ascending order, the k-th to the k-th
    s["moves"][0, : src.numel()], s["moves"][1, : dst.numel()] = src, dst
    to = slot.clone()
    to[src] = dst
    table[s["rows"]] = torch.where(held, to[entries.long()].to(torch.int32), entries)
    shared[dst] = shared[src]
    shared[src] = 0
    for x in s["caches"]:
        for t in x.values():
            if t is not None:
                raw = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
                raw[dst] = raw[src]
    return dict(table=table, shared=shared, moves=s["moves"], counts=torch.stack((count, late.sum())).to(torch.int32),
                caches=[{k: v for k, v in x.items() if v is not None} for x in s["caches"]])


# ---------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------


def exact(case, seed):
    c = case
    if c["kind"] not in ("index", "score", "attend"):
        return None
    s = prepare(case, seed)
    cache = s.get("cache")

    def real(name, slots, h):
        x = cache[name][slots, h].double()
        return x if cache[name + "_scale"] is None else x * cache[name + "_scale"][slots, h].double()[:, None]

    if c["kind"] == "index":
        bounds = s["bounds"].double()
        for b, (old, new) in enumerate(zip(s["from_lens"].tolist(), s["to_lens"].tolist())):
            for j in range(old // c["B"], new // c["B"]):
                slots = s["page_table"][b, j * c["B"]: (j + 1) * c["B"]].long()
                row = int(s["block_table"][b, j])
                for h in range(c["Hkv"]):
                    keys = real("k", slots, h)
                    bounds[row, h, 0], bounds[row, h, 1] = keys.min(0).values, keys.max(0).values
        return dict(bounds=bounds)
    H, G, D, at = c["Hkv"], c["G"], c["D"], 0
    if c["kind"] == "score":
        scores = torch.full((c["bs"], H, s["block_table"].shape[1]), -math.inf, dtype=torch.float64, device=DEV)
        for b, ctx in enumerate(s["prefix_lens"].tolist()):
            n = c["T"] if s["verify_lens"] is None else int(s["verify_lens"][b])
            q = s["q"][at: at + n].double()
            at += n
            full = ctx // c["B"]
            rows = s["block_table"][b, :full].long()
            for h in range(H):
                qs = q[:, h * G: (h + 1) * G].reshape(-1, D)
                low, high = s["bounds"][rows, h, 0].double(), s["bounds"][rows, h, 1].double()
                # (a chunk of queries at a time)
                best = torch.full((full,), -math.inf, dtype=torch.float64, device=DEV)
                for part in qs.split(max(1, int(3e8 / (max(1, full) * D * 8)))):
                    x = torch.maximum(part[:, None] * low, part[:, None] * high).sum(-1) / D ** 0.5
                    best = torch.maximum(best, x.max(0).values)
                scores[b, h, :full] = best
        return dict(scores=scores)
    outs, lses = [], []
    for b, ctx in enumerate(s["prefix_lens"].tolist()):
        n = c["T"] if s["verify_lens"] is None else int(s["verify_lens"][b])
        q = s["q"][at: at + n].double()
        at += n
        window = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        if s["masks"] is not None:
            window = (s["masks"][b, :n, None] >> torch.arange(n, device=DEV)) & 1 == 1
        out = torch.empty(n, H * G, D, dtype=torch.float64, device=DEV)
        lse = torch.empty(n, H * G, dtype=torch.float64, device=DEV)
        for h in range(H):
            mine = s["blocks"][b, h]
            mine = mine[mine >= 0].long()
            p = (mine[:, None] * c["B"] + torch.arange(c["B"], device=DEV)).flatten()
            p = torch.cat((p, torch.arange(ctx // c["B"] * c["B"], ctx + n, device=DEV)))
            slots = s["page_table"][b, p].long()
            seen = torch.ones(n, p.numel(), dtype=torch.bool, device=DEV)
            seen[:, p.numel() - n:] = window
            k, v = real("k", slots, h).t().contiguous(), real("v", slots, h)
            for a in range(h * G, (h + 1) * G):
                x = (q[:, a] @ k / D ** 0.5).masked_fill(~seen, -math.inf)
                lse[:, a] = torch.logsumexp(x, -1)
                out[:, a] = torch.exp(x - lse[:, a, None]) @ v
        outs.append(out)
        lses.append(lse)
    return dict(out=torch.cat(outs), lse=torch.cat(lses))
