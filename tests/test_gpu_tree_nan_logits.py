"""Greedy acceptance of trees over rows with NaN logits: a NaN counts as -inf, wherever in the row it lies."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 23, 4099, 40003])
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("signalling", [False, True])
def test_nan_is_the_lowest(device, signalling, shift, V, dtype):
    from dspine_amd.verification.tree import accept_greedy_tree

    bs, g = 12, torch.Generator().manual_seed(V)
    logits = torch.randint(-40, 40, (bs, V), generator=g).float()
    logits[1, 0] = math.nan  # the row's ends
    logits[2, -1] = math.nan
    logits[3, : min(V - 1, 64)] = math.nan  # whole vectors: those that threads of the first piece begin with
    logits[4, V // 2:] = math.nan
    logits[5, torch.rand(V, generator=g) < 0.9] = math.nan
    logits[6, : V - 1] = math.nan  # one number left
    logits[7, 1:] = math.nan
    logits[8, :] = math.nan  # none: the lowest id
    logits[9, :] = -math.inf
    logits[9, ::3] = math.nan
    logits[10, : V // 2] = -math.nan
    logits[11, : V - 2] = math.nan
    logits[11, V - 2:] = -math.inf
    want = torch.nan_to_num(logits, nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    want = torch.stack([row.eq(row.max()).nonzero()[0, 0] for row in want])
    wide = torch.zeros(bs, V + 7)  # (rows begin anywhere)
    wide[:, shift: shift + V] = logits
    wide = wide.to(dtype)
    if signalling:
        raw = torch.int16 if dtype == torch.bfloat16 else torch.int32
        wide.view(raw)[torch.isnan(wide)] = {torch.int16: 0x7F81, torch.int32: 0x7F800001}[raw]
    outs, _ = accept_greedy_tree(candidates=torch.zeros(bs, 1, dtype=torch.int64, device=device),
                                 parents=torch.full((bs, 1), -1, dtype=torch.int32, device=device),
                                 next_token_logits=wide.to(device)[:, shift: shift + V],
                                 prefix_lens=torch.zeros(bs, dtype=torch.int32, device=device))
    assert outs[2].tolist() == want.tolist()
