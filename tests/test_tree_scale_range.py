"""The attention's scale: one whose base-2 factor leaves float32 is refused (no GPU)."""

import pytest
import torch
from test_tree_contracts import Q, _c_attention, _cache, lib  # noqa: F401 (a fixture)

from dspine_amd import _lib
from dspine_amd.kernels.attention import tree_attention


@pytest.mark.parametrize("scale", [2.0 ** 101, -1e38, 1e300, float("inf")])
def test_scales_out_of_range(lib, scale):  # noqa: F811
    with pytest.raises(ValueError, match="scale must be finite"):
        tree_attention(Q, _cache(), T=3, page_table=torch.zeros((2, 9), dtype=torch.int32),
                       prefix_lens=torch.zeros(2, dtype=torch.int32), scale=scale)
    assert lib.dsv_tree_attention(_c_attention(scale=scale), None) == _lib.DSV_ERR_INVALID


@pytest.mark.parametrize("scale", [2.0 ** 100, -(2.0 ** 100), 0.0])
def test_scales_in_range(lib, scale):  # noqa: F811
    with pytest.raises(ValueError, match="device .cuda. tensors"):
        tree_attention(Q, _cache(), T=3, page_table=torch.zeros((2, 9), dtype=torch.int32),
                       prefix_lens=torch.zeros(2, dtype=torch.int32), scale=scale)
    assert lib.dsv_tree_attention(_c_attention(scale=scale, workspace_bytes=0), None) == _lib.DSV_ERR_WORKSPACE
