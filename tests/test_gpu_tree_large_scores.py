"""Scores so large that float32 holds no fraction of them (2^24 and more): the position of the largest one has all the weight, and
its value is the output, finite and right."""

import pytest
import torch
import tree_ref as R
from test_gpu_tree import BF, E4, HF, I8, _call, _round

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act, dtype", [(BF, BF), (HF, HF), (BF, E4), (HF, I8)])
@pytest.mark.parametrize("T, G", [(3, 2), (7, 4), (17, 4), (40, 4)])
@pytest.mark.parametrize("scale", [0.25, 0.5, 1.0])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_the_largest_score_has_all_the_weight(device, order, scale, T, G, act, dtype):
    n = 500
    d = _round(81, bs=1, T=T, H=2, G=G, D=64, act=act, dtype=dtype, lens=[n], tree=True)
    k, v, ks, vs = d["cache"]
    rank = torch.arange(1, n + T + 1)
    rank = {"rising": rank, "falling": rank.flip(0), "mixed": rank[torch.randperm(n + T, generator=torch.Generator().manual_seed(82))]}[order]
    at = d["page_table"][0].long()
    d["q"] = torch.zeros_like(d["q"])
    d["q"][..., 0] = 2.0 ** 15  # score = scale * 2^19 * rank, exactly
    k[:] = torch.zeros_like(k)
    if ks is None:
        k[at, :, 0] = (16.0 * rank).to(k.dtype).unsqueeze(1)
    else:
        k[at, :, 0] = torch.ones(n + T, 2).to(k.dtype)
        ks[at] = (16.0 * rank).float().unsqueeze(1)
    d["scale"] = scale
    out, lse = _call(d, device)
    value = k[at, 0, 0].double() * (1.0 if ks is None else ks[at, 0].double())  # (bfloat16 rounds the ranks: equal ones tie)
    vals = R.values(v, vs)
    for i in range(T):
        seen = torch.tensor([p < n or bool(int(d["masks"][0, i]) >> (p - n) & 1) for p in range(n + T)])
        top = value[seen].max()
        best = seen & (value == top)
        want = vals[at[best]].mean(0)  # [H, D]
        most = vals[at[best]].abs().amax(0)
        # a weight's rounding, the output's, and the weights of equal scores by exp2's and the sum's
        tol = (R.half_step(dtype if dtype == BF else HF) + R.half_step(act) + 16 * R.U32) * most + 2.0 ** -25
        got = out.cpu().double()[i].view(2, G, 64)
        assert bool(torch.isfinite(got).all())
        assert bool(((got - want.unsqueeze(1)).abs() <= 1.01 * tol.unsqueeze(1)).all())
        assert bool(((lse.cpu().double()[i] - scale * 2.0 ** 15 * top).abs() <= 8 * R.U32 * scale * 2.0 ** 15 * top + 5).all())
