"""The cache's and the trees' operators from their definitions, in float64 on the CPU, and how far a
kernel may be off by counting its roundings (a rounding to type t is off by at most
``torch.finfo(t).eps / 2`` of the value; U32 = 2^-24 for each float32 operation)."""

import math

import torch

U32 = 2.0 ** -24
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def values(x, scale):
    """What a cache's entries stand for."""
    x = x.float().double()
    return x if scale is None else x * scale.double().unsqueeze(-1)


def chain_mask(i):
    return (1 << (i + 1)) - 1


def seen_positions(b, i, *, prefix, nodes, cols, table, slots, masks):
    """The slots that node i of request b sees, in order of their positions."""
    bits = chain_mask(i) if masks is None else int(masks[b, i]) & (2 ** 64 - 1)
    got = []
    for p in range(min(prefix + nodes, cols)):
        if p >= prefix and not bits >> (p - prefix) & 1:
            continue
        s = int(table[b, p])
        if 0 <= s < slots:
            got.append(s)
    return got


def attention(q, k, v, k_scale, v_scale, *, T, page_table, prefix_lens, verify_lens=None, row_offsets=None,
              masks=None, scale=None):
    """(out, lse, out tolerance, lse tolerance) float64; rows of no node are NaN.  All inputs on the CPU."""
    rows, Hq, D = q.shape
    slots, H, _ = k.shape
    G = Hq // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.full((rows, Hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((rows, Hq), math.nan, dtype=torch.float64)
    otol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    cols = page_table.shape[1]
    u_out = half_step(q.dtype)
    # the weights meet the values in the values' 16-bit type, 8-bit codes in float16
    u_p = half_step(k.dtype if k.dtype == torch.bfloat16 else torch.float16)
    for b in range(prefix_lens.numel()):
        n = T if verify_lens is None else max(0, min(T, int(verify_lens[b])))
        pre = max(0, int(prefix_lens[b]))
        for i in range(n):
            r = (b * T if row_offsets is None else int(row_offsets[b])) + i
            at = torch.tensor(seen_positions(b, i, prefix=pre, nodes=n, cols=cols, table=page_table, slots=slots,
                                             masks=masks), dtype=torch.long)
            if at.numel() == 0:
                out[r], lse[r] = 0.0, -math.inf
                continue
            kk = values(k[at], None if k_scale is None else k_scale[at])  # [n, H, D]
            vv = values(v[at], None if v_scale is None else v_scale[at])
            qq = q[r].double().view(H, G, D)
            s = torch.einsum("hgd,nhd->hgn", qq, kk) * scale
            mag = torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()) * abs(scale)
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - l.unsqueeze(-1))
            o = torch.einsum("hgn,nhd->hgd", p, vv)
            pv = torch.einsum("hgn,nhd->hgd", p, vv.abs())
            # a score: D products and sums, the scales and the base-2 exponent's own product and difference
            score = (D + 8) * U32 * mag + 8 * U32 * s.abs()
            # a weight: its score's error (and the reference score's), exp2's 2 U32, its value scale's 2 U32, and its rounding
            # into 16 bits; float16 below its normal range: half of 2^-24 under a largest weight of at least 2^7,
            # times codes whose scale may be the largest (taken as a power of two)
            weight = 2 * score.amax(-1, keepdim=True) + (4 + at.numel()) * U32
            largest = torch.where(torch.isfinite(vv), vv.abs(), torch.zeros_like(vv))
            deep = 0.0 if k.dtype == torch.bfloat16 else 2.0 ** -31 * at.numel() * largest.amax((0, 2)).view(H, 1, 1)
            t = (weight + u_p) * pv * 1.01 + (weight + (2 + at.numel()) * U32) * o.abs() + u_out * o.abs() * 1.01 + deep
            if q.dtype == torch.float16:
                t = t + 2.0 ** -25  # below float16's normal range
            out[r], otol[r] = o.reshape(Hq, D), t.reshape(Hq, D)
            lse[r] = l.reshape(Hq)
            ltol[r] = (score.amax(-1) + (8 + at.numel()) * U32 + 4 * U32 * l.abs()).reshape(Hq)
    return out, lse, otol, ltol


def close(got, want, tol):
    """Elementwise |got - want| <= tol, NaN and infinities in the same places; NaN in ``want`` skips nothing."""
    got = got.double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)])
    bad = (got - want).abs()[finite] - tol[finite]
    assert bad.numel() == 0 or float(bad.max()) <= 0, (float(bad.max()), float(tol[finite].max()))


def quantise(x, dtype):
    """(scales float32, exact ratios x / scale float64) of rows x [n, heads, dim]."""
    amax = x.double().abs().amax(-1)
    return amax / TOP[dtype], x.double() * (TOP[dtype] / amax).unsqueeze(-1)


def tree_masks(parents):
    """masks (Python ints) and depths from parents, by climbing."""
    masks, depths = [], []
    for row in parents.tolist():
        m, d = [], []
        for i, p in enumerate(row):
            if i == 0 or not 0 <= p < i:
                m.append(1 << i)
                d.append(0)
            else:
                m.append(m[p] | 1 << i)
                d.append(d[p] + 1)
        masks.append(m)
        depths.append(d)
    return masks, depths


def signed(bits):
    return bits - 2 ** 64 if bits >> 63 else bits


def accept_tree(candidates, parents, top1, prefix, lens):
    """The walk: (accept, commit, bonus, output, new_seq, path) lists."""
    bs, T = candidates.shape
    res = []
    for b in range(bs):
        n = T if lens is None else max(1, min(T, int(lens[b])))
        path = [0]
        while True:
            here = path[-1]
            step = [i for i in range(here + 1, n) if int(parents[b, i]) == here
                    and int(candidates[b, i]) == int(top1[b, here])]
            if not step:
                break
            path.append(step[0])
        a = len(path) - 1
        bonus = int(top1[b, path[-1]])
        output = [int(candidates[b, i]) for i in path[1:]] + [bonus] + [0] * (T - a - 1)
        res.append((a, a + 1, bonus, output, int(prefix[b]) + a + 1, path + [-1] * (T - a - 1)))
    return res


def commit_tree(accept, path, prefix, rows, table, T, *, out_cache_loc=None, verify_lens=None, slot_offsets=None,
                seq_lens=None):
    """In place on table / seq_lens (numpy-like); returns the freed slots in order."""
    freed = []
    for b in range(len(accept)):
        n = T if verify_lens is None else max(1, min(T, int(verify_lens[b])))
        c = max(1, min(n, int(accept[b]) + 1))
        nodes = [int(x) for x in path[b][:c]]
        pre, r = int(prefix[b]), int(rows[b])
        base = b * T if slot_offsets is None else int(slot_offsets[b])

        def slot(i):
            if out_cache_loc is not None:
                return int(out_cache_loc[base + i])
            return int(table[r][pre + i]) if 0 <= pre + i < len(table[r]) else -1

        slots = [slot(i) for i in range(n)]
        freed += [slots[i] for i in range(n) if i not in nodes]
        for k, i in enumerate(nodes):
            if 0 <= pre + k < len(table[r]):
                table[r][pre + k] = slots[i]
        if seq_lens is not None:
            seq_lens[r] = pre + len(nodes)
    return freed
