"""The block operators and the life of the cache's pages from their definitions, on the CPU: floats in float64 with
how far a kernel may be off by counting its roundings (tests/tree_ref.py), whole numbers as they have to be."""

import math

import torch
import tree_ref as R


def keys_of(k, k_scale, slots):
    """The keys [n, H, D] of slots, float64; an 8-bit cache's product is float32."""
    return R.values(k[slots], None if k_scale is None else k_scale[slots])


def index(bounds, block_size, k, k_scale, *, page_table, block_table, from_lens, to_lens, longest=None):
    """(bounds, tolerance) float64 after the call."""
    want, tol = bounds.double(), torch.zeros(bounds.shape, dtype=torch.float64)
    cols = page_table.shape[1]
    most = -(-(cols if longest is None else longest) // block_size)
    u = 0.0 if k_scale is None else R.U32
    step = 0.0 if k_scale is None and k.dtype == bounds.dtype else R.half_step(bounds.dtype)
    for b in range(from_lens.numel()):
        first, past = max(0, int(from_lens[b])) // block_size, int(to_lens[b]) // block_size
        for j in range(first, min(past, first + most, block_table.shape[1])):
            row = int(block_table[b, j])
            if not 0 <= row < bounds.shape[0]:
                continue
            slots = [int(s) for s in page_table[b, j * block_size: min((j + 1) * block_size, cols)]]
            slots = [s for s in slots if 0 <= s < k.shape[0]]
            want[row], tol[row] = 0.0, 0.0
            if slots:
                x = keys_of(k, k_scale, torch.tensor(slots))
                want[row, :, 0], want[row, :, 1] = x.amin(0), x.amax(0)
                tol[row] = want[row].abs() * (u + step) * 1.01
                if bounds.dtype == torch.float16 and step:
                    tol[row] += 2.0 ** -25  # below float16's normal range
    return want, tol


def scores(q, bounds, block_size, *, T, block_table, prefix_lens, verify_lens=None, row_offsets=None, scale=None):
    """(scores, tolerance) float64 [bs, H, L]: 2 D products and sums, the scale."""
    rows, Hq, D = q.shape
    n_rows, H = bounds.shape[:2]
    G, (bs, L) = Hq // H, block_table.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.full((bs, H, L), -math.inf, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(bs):
        n = T if verify_lens is None else max(0, min(T, int(verify_lens[b])))
        at = b * T if row_offsets is None else int(row_offsets[b])
        if n == 0:
            continue
        x = q[at: at + n].double().view(n, H, G, D)
        for j in range(min(L, max(0, int(prefix_lens[b])) // block_size)):
            r = int(block_table[b, j])
            if not 0 <= r < n_rows:
                continue
            lo, hi = bounds[r, :, 0].double().view(1, H, 1, D), bounds[r, :, 1].double().view(1, H, 1, D)
            parts = x.clamp(max=0) * lo + x.clamp(min=0) * hi
            mag = (x.clamp(max=0) * lo).abs() + (x.clamp(min=0) * hi).abs()
            out[b, :, j] = parts.sum(-1).amax((0, 2)) * scale
            tol[b, :, j] = ((2 * D + 8) * R.U32 * mag.sum(-1)).amax((0, 2)) * scale
    return out, tol


def select(scores, count, *, prefix_lens, block_size, first=0, last=0):
    bs, H, L = scores.shape
    out = torch.full((bs, H, count), -1, dtype=torch.int32)
    for b in range(bs):
        n = min(L, max(0, int(prefix_lens[b])) // block_size)
        for h in range(H):
            row = [(-math.inf if math.isnan(v) else v) for v in scores[b, h, :n].tolist()]
            must = [j for j in range(n) if j < first or j >= n - last]
            rest = sorted((j for j in range(n) if j not in set(must)), key=lambda j: (-row[j], j))
            ids = sorted(must + rest[: max(0, count - len(must))])[:count]
            out[b, h, : len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return out


def attention(q, k, v, k_scale, v_scale, *, T, blocks, block_size, page_table, prefix_lens, verify_lens=None,
              row_offsets=None, masks=None, scale=None):
    """(out, lse, out tolerance, lse tolerance): each cache head's attention over a page table of its own."""
    rows, Hq, D = q.shape
    H, bs = k.shape[1], prefix_lens.numel()
    G, cols = Hq // H, page_table.shape[1]
    outs = []
    for h in range(H):
        tables, pres = [], []
        for b in range(bs):
            pre = max(0, int(prefix_lens[b]))
            full = pre // block_size
            at = []
            for i in blocks[b, h, : min(blocks.shape[2], full)].tolist():
                at += range(i * block_size, (i + 1) * block_size) if 0 <= i < full else [cols] * block_size
            at += range(full * block_size, pre + T)
            tables.append([int(page_table[b, p]) if p < cols else -1 for p in at])
            pres.append(len(at) - T)
        width = max(len(t) for t in tables)
        table = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32)
        mine = slice(h, h + 1)
        outs.append(R.attention(q[:, h * G: (h + 1) * G], k[:, mine], v[:, mine],
                                None if k_scale is None else k_scale[:, mine], None if v_scale is None else v_scale[:, mine],
                                T=T, page_table=table, prefix_lens=torch.tensor(pres, dtype=torch.int32),
                                verify_lens=verify_lens, row_offsets=row_offsets, masks=masks, scale=scale))
    return tuple(torch.cat(x, 1) for x in zip(*outs))


def _held(table, lens, row):
    return min(max(int(lens[row]), 0), table.shape[1])


def fork(table, lens, shared, parents, children):
    """In place."""
    for p, c in zip(parents, children):
        if not (0 <= p < table.shape[0] and 0 <= c < table.shape[0]) or p == c:
            continue
        n = _held(table, lens, p)
        table[c, :n] = table[p, :n]
        lens[c] = n
        for s in table[p, :n].tolist():
            if 0 <= s < shared.numel():
                shared[s] += 1


def free(table, lens, shared, rows):
    """In place; returns the freed slots."""
    for r in dict.fromkeys(rows):
        if 0 <= r < table.shape[0]:
            for s in table[r, : _held(table, lens, r)].tolist():
                if 0 <= s < shared.numel():
                    shared[s] -= 1
            lens[r] = 0
    freed = [s for s in range(shared.numel()) if shared[s] < 0]
    shared[freed] = 0
    return freed


def compact(table, lens, rows, slots, shared=None):
    """In place on table and shared; returns (from, to, used)."""
    rows = [r for r in dict.fromkeys(rows) if 0 <= r < table.shape[0]]
    used = {s for r in rows for s in table[r, : _held(table, lens, r)].tolist() if 0 <= s < slots}
    U = len(used)
    src, dst = sorted(s for s in used if s >= U), [s for s in range(U) if s not in used]
    to = dict(zip(src, dst))
    for r in rows:
        for p in range(_held(table, lens, r)):
            table[r, p] = to.get(int(table[r, p]), int(table[r, p]))
    if shared is not None:
        for s, d in to.items():
            shared[d], shared[s] = int(shared[s]), 0
    return src, dst, U
