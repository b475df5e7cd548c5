"""Attention over a quantised cache in which positions of large value scales have next to no weight: what counts in the
sum is a position's weight times its scale, and the others must keep their bits whatever a single scale is."""

import math

import pytest
import torch
import tree_ref as R
from test_gpu_tree import BF, E4, I8, _call, _round

pytestmark = pytest.mark.gpu

FORMS = [(3, 2), (7, 4), (17, 4), (40, 4)]  # nodes, query heads a cache head: rows of every form


def _reference(d):
    """(out, lse, out tolerance, lse tolerance) float64 as tree_ref.attention counts them, but for float16's lower end: a
    position's weight times scale, whose largest of the row is held at 2^10 or more, is off by at most half of float16's
    lowest step there, 2^-25, so by 2^-35 of that largest; a score that is held against a reference up to 128 away in powers
    of two is rounded by 2^-18, and so is its weight, by less than 2^-18 of it (twice, for the reference's own)."""
    q, (k, v, ks, vs) = d["q"], d["cache"]
    rows, heads, D = q.shape
    slots, H, _ = k.shape
    G, T = heads // H, d["T"]
    out, lse = torch.zeros(rows, heads, D, dtype=torch.float64), torch.zeros(rows, heads, dtype=torch.float64)
    otol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    u_out, u_p = R.half_step(q.dtype), R.half_step(torch.float16)
    for b in range(d["prefix_lens"].numel()):
        for i in range(T):
            at = torch.tensor(R.seen_positions(b, i, prefix=int(d["prefix_lens"][b]), nodes=T, cols=d["page_table"].shape[1],
                                               table=d["page_table"], slots=slots, masks=d["masks"]))
            kk, vv = R.values(k[at], ks[at]).permute(1, 2, 0), R.values(v[at], vs[at]).transpose(0, 1)
            qq = q[b * T + i].double().view(H, G, D)
            s, mag = qq @ kk / math.sqrt(D), qq.abs() @ kk.abs() / math.sqrt(D)
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - l.unsqueeze(-1))
            o, pv = p @ vv, p @ vv.abs()
            most = (p * vs[at].double().t().unsqueeze(1)).amax(-1, keepdim=True) * R.TOP[v.dtype]
            score = (D + 8) * R.U32 * mag + 8 * R.U32 * s.abs()
            weight = 2 * score.amax(-1, keepdim=True) + (4 + at.numel()) * R.U32 + 2.0 ** -17
            t = ((weight + u_p) * pv * 1.01 + (weight + (2 + at.numel()) * R.U32) * o.abs() + u_out * o.abs() * 1.01
                 + at.numel() * 2.0 ** -35 * most)
            r = b * T + i
            out[r], otol[r], lse[r] = o.reshape(heads, D), t.reshape(heads, D), l.reshape(heads)
            ltol[r] = (score.amax(-1) + (8 + at.numel()) * R.U32 + 4 * R.U32 * l.abs() + 2.0 ** -17).reshape(heads)
    return out, lse, otol, ltol


def _lower(d, positions, down, power):
    """Scores of request 0's ``positions`` about ``down`` below the others', their value scales 2^power above."""
    k, v, ks, vs = d["cache"]
    d["q"][..., 0] = round(math.sqrt(k.shape[2]))  # a key's first element adds (about) itself to the score
    at = d["page_table"][0].long()[positions]
    k[at] = torch.zeros_like(k[at])
    k[at, :, 0] = torch.full(k[at, :, 0].shape, -R.TOP[k.dtype]).to(k.dtype)
    ks[at] = down / R.TOP[k.dtype]
    vs[at] *= 2.0 ** power


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", FORMS)
@pytest.mark.parametrize("power", [20, 30, 36, 80, 100])
@pytest.mark.parametrize("place", ["first", "inside", "last", "every"])
def test_a_large_scale_without_weight(device, place, power, T, G, dtype):
    """Weights of e^-60 (2^-87): up to scales 2^80 apart those positions hardly count, at 2^100 they are the output."""
    d = _round(51, bs=2, T=T, H=2, G=G, D=64, act=BF, dtype=dtype, lens=[700, 90], tree=True)
    _lower(d, {"first": [0], "inside": [333], "last": [699], "every": list(range(5, 700, 9))}[place], 60.0, power)
    out, lse = _call(d, device)
    want, wl, otol, ltol = _reference(d)
    R.close(out.cpu(), want, otol)
    R.close(lse.cpu(), wl, ltol)


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", FORMS)
@pytest.mark.parametrize("D", [96, 128, 192, 256])
def test_a_large_scale_without_weight_at_other_dims(device, D, T, G, dtype):
    d = _round(57, bs=2, T=T, H=1, G=G, D=D, act=BF, dtype=dtype, lens=[400, 90], tree=True)
    _lower(d, list(range(5, 400, 9)), 60.0, 36)
    out, lse = _call(d, device)
    want, wl, otol, ltol = _reference(d)
    R.close(out.cpu(), want, otol)
    R.close(lse.cpu(), wl, ltol)


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", FORMS)
def test_scales_that_fall_as_scores_rise(device, T, G, dtype):
    """Along the context scores rise by 100 in all while scales fall by 2^120: either reference moves all the time."""
    d = _round(52, bs=1, T=T, H=1, G=G, D=64, act=BF, dtype=dtype, lens=[800], tree=True)
    k, v, ks, vs = d["cache"]
    d["q"][..., 0] = 8.0
    at = d["page_table"][0].long()
    for turn in (1.0, -1.0):
        step = torch.arange(len(at)) / len(at) if turn > 0 else torch.arange(len(at), 0, -1) / len(at)
        k[at] = torch.zeros_like(k[at])
        k[at, :, 0] = torch.full((len(at), 1), -R.TOP[k.dtype]).to(k.dtype)
        ks[at] = (100.0 * (1 - step) / R.TOP[k.dtype]).float().unsqueeze(1)
        vs[at] = torch.exp2(60 - 120 * step).float().unsqueeze(1)
        out, lse = _call(d, device)
        want, wl, otol, ltol = _reference(d)
        R.close(out.cpu(), want, otol)
        R.close(lse.cpu(), wl, ltol)


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", FORMS)
def test_a_context_of_zero_scales(device, T, G, dtype):
    """Values of nothing but zeros (scale 0) in the context: lse is whole, the output the window's share."""
    d = _round(53, bs=2, T=T, H=2, G=G, D=64, act=BF, dtype=dtype, lens=[300, 40], tree=True)
    for b, n in enumerate((300, 40)):
        d["cache"][3][d["page_table"][b, :n].long()] = 0.0
    out, lse = _call(d, device)
    want, wl, otol, ltol = _reference(d)
    R.close(out.cpu(), want, otol)
    R.close(lse.cpu(), wl, ltol)


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", FORMS)
def test_values_up_to_the_largest_of_their_type(device, T, G, dtype):
    """Rows that write_kv takes near bfloat16's largest: outputs are finite and right, as the rows read back are."""
    from dspine_amd.kernels.cache import new_cache, read_kv, write_kv

    d = _round(54, bs=2, T=T, H=2, G=G, D=64, act=BF, dtype=dtype, lens=[300, 40], tree=True)
    n = d["cache"][0].shape[0]
    x = torch.randn(n, 2, 64, generator=torch.Generator().manual_seed(55))
    x = (x * (3e38 / x.abs().amax(-1, keepdim=True))).to(BF)
    cache, slots = new_cache(n, 2, 64, dtype=dtype, device=device), torch.arange(n, device=device)
    write_kv(cache, x.to(device), x.to(device), slots)
    assert bool(torch.isfinite(read_kv(cache, slots, dtype=torch.float32)[1]).all())
    d["cache"] = (*d["cache"][:1], cache.v.cpu(), d["cache"][2], cache.v_scale.cpu())
    out, lse = _call(d, device)
    want, wl, otol, ltol = _reference(d)
    assert bool(torch.isfinite(out).all())
    R.close(out.cpu(), want, otol)
    R.close(lse.cpu(), wl, ltol)


@pytest.mark.parametrize("dtype", [E4, I8])
@pytest.mark.parametrize("T, G", FORMS)
@pytest.mark.parametrize("power", [119, -108])
def test_small_weights_count_whatever_the_scales(device, power, T, G, dtype):
    """4096 weights of e^-13.5 beside one of 1, every scale near the end of write_kv's range: they are half a percent of
    the sum, and all of it is there."""
    d = _round(56, bs=1, T=T, H=1, G=G, D=64, act=BF, dtype=dtype, lens=[4097], tree=True)
    k, v, ks, vs = d["cache"]
    _lower(d, list(range(4096)), 13.5, 0)
    at = d["page_table"][0].long()
    k[at[4096:]] = torch.zeros_like(k[at[4096:]])
    d["masks"][:] = 0  # (the context alone)
    vs[:] = 2.0 ** power
    out, lse = _call(d, device)
    want, wl, otol, ltol = _reference(d)
    R.close(out.cpu(), want, otol)
    R.close(lse.cpu(), wl, ltol)
