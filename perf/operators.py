"""What the performance of the cache and tree operators is measured on: the calls a server makes
around the target forward of a drafted tree, each through its public entry point, with inputs
made on the GPU from a seed.

A case's ``kind`` names the call:

  attend   tree_attention: attention of each request's drafted nodes over its paged KV cache
  write    write_kv: new keys and values into cache slots, quantised where the cache is
  read     read_kv: slots of a cache gathered and brought back to activations
  accept   accept_greedy_tree: the path of a drafted tree that the target's argmaxes take

``run`` computes them in elementary torch operations, in 32 bits, or (``own``) through the
package's entry points.
"""

from __future__ import annotations

import math

import torch

DEV = "cuda"
own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn,
         "int8": torch.int8}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1, "int8": 1}
TOP_CODE = {"e4m3": 448.0, "int8": 127.0}  # the largest magnitude of a code
TINY = 2.0 ** -100  # a (token, head) whose largest magnitude is below it is stored as zeros

# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------


def listed():
    return [
        # one interactive user without drafts: a single token over a short context, launch bound
        dict(name="attend_1x1_640", kind="attend", bs=1, T=1, Hkv=8, G=4, D=128, lo=640, hi=640, dtype="bf16",
             cache="bf16", tree=False, ragged=False),
        # four users, a drafted tree of 25 nodes each over a few thousand tokens
        dict(name="attend_4x25_tree_3k", kind="attend", bs=4, T=25, Hkv=8, G=4, D=128, lo=1500, hi=4700,
             dtype="bf16", cache="bf16", tree=True, ragged=False),
        # a busy server's round: a planner's verify lengths (4 to 17) on compact rows, chains of drafts
        dict(name="attend_64x17_ragged_8k", kind="attend", bs=64, T=17, Hkv=8, G=4, D=128, lo=1000, hi=8000,
             dtype="bf16", cache="bf16", tree=False, ragged=True),
        # wide trees of 64 nodes, eight query heads a KV head, an 8-bit float cache: the most arithmetic a byte
        dict(name="attend_16x64_tree_e4m3", kind="attend", bs=16, T=64, Hkv=8, G=8, D=128, lo=4000, hi=12000,
             dtype="bf16", cache="e4m3", tree=True, ragged=False),
        # single tokens over long documents, an 8-bit integer cache
        dict(name="attend_8x1_64k_int8", kind="attend", bs=8, T=1, Hkv=8, G=4, D=128, lo=16000, hi=64000,
             dtype="bf16", cache="int8", tree=False, ragged=False),
        # a small float16 model with odd counts: five query heads a KV head, heads of 96, new conversations among
        # the requests
        dict(name="attend_13x23_odd_f16", kind="attend", bs=13, T=23, Hkv=3, G=5, D=96, lo=0, hi=3001, dtype="f16",
             cache="f16", tree=True, ragged=False),
        # one request's drafted block into an 8-bit float cache: launch bound
        dict(name="write_17_e4m3", kind="write", n=17, Hkv=8, D=128, Hq=32, dtype="bf16", cache="e4m3"),
        # a prompt's chunk into an 8-bit integer cache
        dict(name="write_16384_int8", kind="write", n=16384, Hkv=8, D=128, Hq=32, dtype="bf16", cache="int8"),
        # a short shared prefix brought back from an 8-bit float cache
        dict(name="read_777_e4m3", kind="read", n=777, Hkv=8, D=128, dtype="f16", cache="e4m3"),
        # a long document brought back from an 8-bit integer cache, to be moved or computed on
        dict(name="read_50000_int8", kind="read", n=50000, Hkv=8, D=128, dtype="bf16", cache="int8"),
        # an interactive user's tree of 25 nodes, float32 logits
        dict(name="accept_1x25_f32", kind="accept", bs=1, T=25, V=151936, dtype="f32", ragged=False),
        # a busy server's trees
        dict(name="accept_64x17_bf16", kind="accept", bs=64, T=17, V=151936, dtype="bf16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "read", "accept"])
    c = dict(kind=kind)
    if kind == "attend":
        dtype = rng.choice(["bf16", "bf16", "f16"])
        c.update(bs=_log(rng, 1, 64), T=rng.choice([1, rng.randint(2, 64), rng.randint(2, 32), 17]),
                 Hkv=rng.choice([1, 2, 3, 4, 8, 8]), G=rng.choice([1, 2, 3, 4, 4, 5, 8, 16]),
                 D=rng.choice([64, 80, 96, 128, 128, 192, 256]), dtype=dtype,
                 cache=rng.choice([dtype, dtype, "e4m3", "int8"]), tree=rng.random() < 0.6,
                 ragged=rng.random() < 0.4)
        hi = _log(rng, 16, 64000)
        # no more than the largest listed case gathers, scores or multiplies
        while c["bs"] > 1 and (c["bs"] * hi * c["Hkv"] * c["D"] > 5e8 or
                               c["bs"] * hi * c["Hkv"] * c["G"] * c["T"] > 7e8 or
                               c["bs"] * hi * c["Hkv"] * c["G"] * c["T"] * c["D"] > 6e10):
            c["bs"] = (c["bs"] + 1) // 2
        most = min(5e8 / (c["Hkv"] * c["D"]), 7e8 / (c["Hkv"] * c["G"] * c["T"]),
                   6e10 / (c["Hkv"] * c["G"] * c["T"] * c["D"])) / c["bs"]
        hi = max(1, min(hi, int(most)))
        c.update(lo=rng.choice([hi, hi // 2, hi // 8, 0]), hi=hi)
    elif kind in ("write", "read"):
        c.update(n=_log(rng, 1, 16384 if kind == "write" else 50000), Hkv=rng.choice([1, 2, 3, 4, 8]),
                 D=rng.choice([64, 80, 96, 128, 128, 192, 256]), dtype=rng.choice(["bf16", "f16"]))
        while c["n"] * c["Hkv"] * c["D"] > (16384 if kind == "write" else 50000) * 1024:
            c["n"] //= 2
        c.update(cache=rng.choice([c["dtype"], "e4m3", "int8", "e4m3", "int8"]))
        if kind == "write":
            c.update(Hq=c["Hkv"] * rng.choice([1, 4, 8]))
    else:
        dtype = rng.choice(["bf16", "bf16", "f32"])
        c.update(bs=_log(rng, 1, 64), T=rng.randint(2, 64), V=_log(rng, 8192, 262144), dtype=dtype,
                 ragged=rng.random() < 0.4)
        if rng.random() < 0.7:
            c["V"] = c["V"] // 64 * 64
        while c["bs"] > 1 and c["bs"] * c["T"] * c["V"] * BYTES[dtype] > 64 * 17 * 151936 * 2:
            c["bs"] //= 2
    return c


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 6151 + 29)


def _spread(lo, hi, n):
    """n lengths spread evenly over [lo, hi]."""
    return [int(lo + (hi - lo) * (i + 0.5) / n) for i in range(n)]


def _lengths(c):
    """(context, nodes) of each request, before the seed's order."""
    bs, T = c["bs"], c["T"]
    nodes = _spread(max(1, T // 4), T + 1, bs) if c["ragged"] else [T] * bs
    ctx = _spread(c["lo"], c["hi"], bs) if c["kind"] == "attend" else [0] * bs
    step = next(s for s in (5, 7, 11, 13) if math.gcd(s, bs) == 1)
    return [(ctx[i], nodes[i * step % bs]) for i in range(bs)]


def _activations(g, n, heads, dim, dtype):
    """Keys or values as a projection leaves them: a few channels of a head much larger than the rest."""
    gain = torch.ones(heads, dim, device=DEV)
    gain[:, torch.randint(0, dim, (max(1, dim // 32),), generator=g, device=DEV)] = 4.0
    return (torch.randn(n, heads, dim, generator=g, device=DEV) * gain).to(TYPES[dtype])


def _quantise(x, cache):
    """x [n, heads, dim] as (codes, scales): a scale for each (token, head), its largest magnitude at the largest
    code; rounding to nearest even."""
    top = TOP_CODE[cache]
    x = x.float()
    amax = x.abs().amax(-1)
    live = amax >= TINY
    inverse = torch.where(live, torch.reciprocal(amax) * top, torch.zeros_like(amax))
    scale = torch.where(live, amax * torch.full_like(amax, 1.0 / top), torch.zeros_like(amax))
    codes = x * inverse.unsqueeze(-1)
    codes = codes.to(TYPES["e4m3"]) if cache == "e4m3" else codes.round().to(torch.int8)
    return codes, scale


def _cache(g, slots, c, dtype):
    x, scale = [], []
    for _ in range(2):
        a = _activations(g, slots, c["Hkv"], c["D"], dtype)
        s = None
        if c["cache"] in TOP_CODE:
            a, s = _quantise(a, c["cache"])
        x.append(a)
        scale.append(s)
    return dict(k=x[0], v=x[1], k_scale=scale[0], v_scale=scale[1])


def _parents(g, bs, T):
    """Drafted trees: node 0 is the last accepted token, a node's parent one of the few nodes before it."""
    i = torch.arange(T, device=DEV)
    back = 1 + (torch.rand(bs, T, generator=g, device=DEV).square() * torch.clamp(i, max=6)).long()
    parents = (i - back).clamp_(min=0)
    parents[:, 0] = -1
    return parents.to(torch.int32)


def _masks(parents):
    """The nodes each node sees: itself and its ancestors, as bits."""
    bs, T = parents.shape
    masks = torch.ones(bs, T, dtype=torch.int64, device=DEV)
    for i in range(1, T):
        up = torch.gather(masks, 1, parents[:, i: i + 1].long())[:, 0]
        masks[:, i] = up | (1 << i if i < 63 else -2 ** 63)
    return masks


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=dict(c))
    if c["kind"] == "attend":
        lengths = _lengths(c)
        order = torch.randperm(c["bs"], generator=g, device=DEV).tolist()
        lengths = [lengths[i] for i in order]
        ctx = torch.tensor([a for a, _ in lengths], device=DEV)
        nodes = torch.tensor([b for _, b in lengths], device=DEV)
        total = ctx + nodes
        width = max(c["hi"], 1) + c["T"] + 32
        used = int(total.sum())
        slots = used + used // 8 + 64
        # a request's prompt (three quarters) lies in one run of slots, what came later wherever slots were free
        head = total * 3 // 4
        free = torch.randperm(slots - int(head.sum()), generator=g, device=DEV) + head.sum()
        pos = torch.arange(width, device=DEV).expand(c["bs"], -1)
        run = (head.cumsum(0) - head).unsqueeze(1) + pos
        tail = (total - head).cumsum(0) - (total - head)
        late = free[(tail.unsqueeze(1) + pos - head.unsqueeze(1)).clamp_(0, free.numel() - 1)]
        table = torch.where(pos < head.unsqueeze(1), run, late)
        table = torch.where(pos < total.unsqueeze(1), table, torch.zeros_like(table))
        parents = _parents(g, c["bs"], c["T"])
        rows = int(nodes.sum()) if c["ragged"] else c["bs"] * c["T"]
        s.update(cache=_cache(g, slots, c, c["dtype"]), page_table=table.to(torch.int32),
                 prefix_lens=ctx.to(torch.int32), masks=_masks(parents) if c["tree"] else None,
                 verify_lens=nodes.to(torch.int32) if c["ragged"] else None,
                 row_offsets=nodes.cumsum(0) - nodes if c["ragged"] else None,
                 q=(1.5 * torch.randn(rows, c["Hkv"] * c["G"], c["D"], generator=g, device=DEV)).to(TYPES[c["dtype"]]),
                 longest=max(a + b for a, b in lengths))
    elif c["kind"] == "write":
        n, H, D = c["n"], c["Hkv"], c["D"]
        # keys and values are slices of the fused projection's output
        qkv = _activations(g, n, c["Hq"] + 2 * H, D, c["dtype"])
        slots = n + n // 4 + 16
        s.update(new_k=qkv[:, c["Hq"]: c["Hq"] + H], new_v=qkv[:, c["Hq"] + H:],
                 cache=_cache(g, slots, c, c["dtype"]),
                 slots=torch.randperm(slots, generator=g, device=DEV)[:n])
    elif c["kind"] == "read":
        slots = c["n"] + c["n"] // 4 + 16
        s.update(cache=_cache(g, slots, c, c["dtype"]), slots=torch.randperm(slots, generator=g, device=DEV)[: c["n"]])
    else:
        bs, T, V = c["bs"], c["T"], c["V"]
        logits = (torch.randn(bs * T, V, generator=g, device=DEV) * 2.5).to(TYPES[c["dtype"]])
        parents = _parents(g, bs, T)
        # most nodes carry their parent's likeliest token, the siblings after it others
        best = logits.argmax(-1).view(bs, T)
        takes = torch.gather(best, 1, parents.clamp(min=0).long())
        takes = torch.where(torch.rand(bs, T, generator=g, device=DEV) < 0.6, takes,
                            torch.randint(0, V, (bs, T), generator=g, device=DEV))
        lens = torch.tensor([b for _, b in _lengths(c)], device=DEV, dtype=torch.int32)
        s.update(logits=logits, candidates=takes, parents=parents,
                 prefix_lens=torch.randint(64, 4096, (bs,), generator=g, device=DEV).to(torch.int32),
                 verify_lens=lens[torch.randperm(bs, generator=g, device=DEV)] if c["ragged"] else None,
                 masks=_masks(parents))
    return s


def work(case):
    c = case
    if c["kind"] == "attend":
        lengths = _lengths(c)
        heads, quant = c["Hkv"], c["cache"] in TOP_CODE
        positions, rows = sum(a + b for a, b in lengths), sum(b for _, b in lengths)
        per = heads * (2 * c["D"] * BYTES[c["cache"]] + (8 if quant else 0)) + 4
        return {"bytes": positions * per + rows * heads * c["G"] * (2 * c["D"] * BYTES[c["dtype"]] + 4),
                "flops": 4.0 * c["D"] * heads * c["G"] * sum((a + 1) * b for a, b in lengths)}
    if c["kind"] in ("write", "read"):
        elements = 2 * c["n"] * c["Hkv"] * c["D"]
        scales = 8 * c["n"] * c["Hkv"] if c["cache"] in TOP_CODE else 0
        return {"bytes": elements * (BYTES[c["dtype"]] + BYTES[c["cache"]]) + scales + 8 * c["n"], "flops": elements}
    elements = sum(n for _, n in _lengths(c)) * c["V"]
    return {"bytes": elements * BYTES[c["dtype"]], "flops": elements}


# ---------------------------------------------------------------------------------------------
# the passes
# ---------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _own(state)
    return {"attend": _attend, "write": _write, "read": _read, "accept": _accept}[state["case"]["kind"]](state)


def _own(s):
    from dspine_amd.kernels.attention import tree_attention
    from dspine_amd.kernels.cache import KVCache, read_kv, write_kv
    from dspine_amd.verification.tree import accept_greedy_tree

    c = s["case"]
    if c["kind"] == "accept":
        outputs, path = accept_greedy_tree(candidates=s["candidates"], parents=s["parents"],
                                           next_token_logits=s["logits"], prefix_lens=s["prefix_lens"],
                                           verify_lens=s["verify_lens"])
        return dict(zip(("accept", "commit", "bonus", "output", "new_seq"), outputs), path=path)
    cache = KVCache(**s["cache"])
    if c["kind"] == "attend":
        lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=DEV)
        out = tree_attention(s["q"], cache, T=c["T"], page_table=s["page_table"], prefix_lens=s["prefix_lens"],
                             verify_lens=s["verify_lens"], row_offsets=s["row_offsets"], masks=s["masks"], lse=lse)
        return dict(out=out, lse=lse)
    if c["kind"] == "write":
        write_kv(cache, s["new_k"], s["new_v"], s["slots"])
        return {k: v for k, v in s["cache"].items() if v is not None}
    k, v = read_kv(cache, s["slots"], dtype=TYPES[c["dtype"]])
    return dict(k=k, v=v)


def _values(cache, name, at):
    """The values that the slots ``at`` of a cache stand for, in 32 bits."""
    x = cache[name][at].float()
    scale = cache[name + "_scale"]
    return x if scale is None else x * scale[at].unsqueeze(-1)


def _attend(s):
    c = s["case"]
    bs, T, H, G, D = c["bs"], c["T"], c["Hkv"], c["G"], c["D"]
    prefix, L = s["prefix_lens"].long(), s["longest"]
    node, pos = torch.arange(T, device=DEV), torch.arange(L, device=DEV)
    nodes = torch.full_like(prefix, T) if s["verify_lens"] is None else s["verify_lens"].long()
    start = torch.arange(bs, device=DEV) * T if s["row_offsets"] is None else s["row_offsets"]
    real = node < nodes.unsqueeze(1)  # [bs, T]
    rows = torch.where(real, start.unsqueeze(1) + node, torch.zeros_like(start).unsqueeze(1))
    q = s["q"].float()[rows].view(bs, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(bs, H, T * G, D)
    at = s["page_table"][:, :L].long()
    k = _values(s["cache"], "k", at).permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(q, k).view(bs, H, T, G, L) * (1.0 / math.sqrt(D))
    del k
    j = pos - prefix.unsqueeze(1)  # the window's node at a position, [bs, L]
    if s["masks"] is None:
        sees = j.unsqueeze(1) <= node.unsqueeze(1)
    else:
        sees = (s["masks"].unsqueeze(-1) >> j.clamp(0, 63).unsqueeze(1)) & 1 == 1
    sees = (j < 0).unsqueeze(1) | (sees & (j < nodes.unsqueeze(1)).unsqueeze(1))  # [bs, T, L]
    scores = scores.masked_fill_(~sees.view(bs, 1, T, 1, L), -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    v = _values(s["cache"], "v", at).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(p.view(bs, H, T * G, L), v).view(bs, H, T, G, D) / total
    lse = (top + torch.log(total))[..., 0]
    out = out.permute(0, 2, 1, 3, 4).reshape(bs, T, H * G, D)[real].to(s["q"].dtype)
    lse = lse.permute(0, 2, 1, 3).reshape(bs, T, H * G)[real]
    return dict(out=out, lse=lse)


def _write(s):
    c, cache, at = s["case"], s["cache"], s["slots"]
    if c["cache"] in TOP_CODE:
        k, k_scale = _quantise(s["new_k"], c["cache"])
        v, v_scale = _quantise(s["new_v"], c["cache"])
        cache["k_scale"][at], cache["v_scale"][at] = k_scale, v_scale
    else:
        k, v = s["new_k"], s["new_v"]
    # (8-bit floats are moved as bytes)
    raw = torch.uint8 if c["cache"] == "e4m3" else cache["k"].dtype
    cache["k"].view(raw)[at], cache["v"].view(raw)[at] = k.view(raw), v.view(raw)
    return {name: x for name, x in cache.items() if x is not None}


def _read(s):
    to = TYPES[s["case"]["dtype"]]
    return dict(k=_values(s["cache"], "k", s["slots"]).to(to), v=_values(s["cache"], "v", s["slots"]).to(to))


def _accept(s):
    c = s["case"]
    bs, T, V = c["bs"], c["T"], c["V"]
    logits, tokens, parents, masks = s["logits"], s["candidates"], s["parents"].long(), s["masks"]
    ids = torch.arange(V, device=DEV, dtype=torch.int32)
    best = torch.where(logits == logits.amax(-1, keepdim=True), ids, V).amin(-1).long().view(bs, T)
    node = torch.arange(T, device=DEV)
    lens = torch.full((bs,), T, device=DEV) if s["verify_lens"] is None else s["verify_lens"].long()
    fits = (tokens == torch.gather(best, 1, parents.clamp(min=0))) & (node < lens.unsqueeze(1))
    # of siblings with one token the first is taken
    twin = (tokens.unsqueeze(2) == tokens.unsqueeze(1)) & (parents.unsqueeze(2) == parents.unsqueeze(1))
    fits &= ~(twin & (node.unsqueeze(0) < node.unsqueeze(1))).any(-1)
    fits[:, 0] = True
    sees = (masks.unsqueeze(-1) >> node) & 1 == 1  # [bs, T, T]: itself and its ancestors
    on = (fits.unsqueeze(1) | ~sees).all(-1)  # the nodes of the accepted path
    count = on.sum(-1)
    place = torch.where(on, on.cumsum(-1) - 1, T)
    path = torch.full((bs, T + 1), -1, device=DEV, dtype=torch.int64).scatter_(1, place, node.expand(bs, -1))[:, :T]
    last = torch.gather(path, 1, (count - 1).unsqueeze(1))
    bonus = torch.gather(best, 1, last)
    follow = torch.cat((path[:, 1:], path[:, :1] * 0 - 1), 1)
    output = torch.where(follow >= 0, torch.gather(tokens, 1, follow.clamp(min=0)), torch.zeros_like(tokens))
    output = output.scatter(1, (count - 1).unsqueeze(1), bonus)
    accept = (count - 1).to(torch.int32)
    return dict(accept=accept, commit=accept + 1, bonus=bonus[:, 0], output=output,
                new_seq=s["prefix_lens"] + accept + 1, path=path.to(torch.int32))


# ---------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    c, cache = case, s.get("cache")

    def real(name, rows):
        x = cache[name][rows].double()
        return x if cache[name + "_scale"] is None else x * cache[name + "_scale"][rows].double()[..., None]

    if c["kind"] == "attend":
        outs, lses = [], []
        at = 0
        for b, (ctx, table) in enumerate(zip(s["prefix_lens"].tolist(), s["page_table"].long())):
            n = c["T"] if s["verify_lens"] is None else int(s["verify_lens"][b])
            q = s["q"][at: at + n].double()
            at += n
            rows = table[: ctx + n]
            seen = torch.ones(n, ctx + n, dtype=torch.bool, device=DEV)
            for i in range(n):
                bits = (1 << (i + 1)) - 1 if s["masks"] is None else int(s["masks"][b, i])
                seen[i, ctx:] = torch.tensor([bool(bits >> j & 1) for j in range(n)], device=DEV)
            out = torch.empty(n, c["Hkv"] * c["G"], c["D"], dtype=torch.float64, device=DEV)
            lse = torch.empty(n, c["Hkv"] * c["G"], dtype=torch.float64, device=DEV)
            keys, values = real("k", rows), real("v", rows)
            for h in range(c["Hkv"]):
                k, v = keys[:, h].t().contiguous(), values[:, h].contiguous()
                for a in range(h * c["G"], (h + 1) * c["G"]):
                    x = (q[:, a] @ k / c["D"] ** 0.5).masked_fill(~seen, -math.inf)
                    lse[:, a] = torch.logsumexp(x, -1)
                    out[:, a] = torch.exp(x - lse[:, a, None]) @ v
            outs.append(out)
            lses.append(lse)
        return dict(out=torch.cat(outs), lse=torch.cat(lses))
    if c["kind"] == "read":
        return dict(k=real("k", s["slots"]), v=real("v", s["slots"]))
    if c["kind"] == "write" and c["cache"] in TOP_CODE:
        # codes are whole or 8-bit numbers: their values depend on the rounding's rule, the scales do not
        done = {}
        for name in ("k", "v"):
            amax = s["new_" + name].double().abs().amax(-1)
            scale = cache[name + "_scale"].double()
            scale[s["slots"]] = amax / TOP_CODE[c["cache"]]
            done[name + "_scale"] = scale
        return dict(done, k=None, v=None)
    return None
