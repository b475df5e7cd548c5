"""What the cache and tree entry points refuse, before any launch (no GPU): calls on CPU or meta tensors raise
ValueError, the C entries return DSV_ERR_INVALID or DSV_ERR_WORKSPACE with nothing launched.

Argument checks come before the check of the device, so a call that passes them all ends at "device (cuda)
tensors" here: every case starts from such a call."""

import ctypes
import os
import subprocess

import pytest
import torch

from dspine_amd import _lib
from dspine_amd.kernels.attention import tree_attention
from dspine_amd.kernels.cache import KVCache, new_cache, read_kv, write_kv
from dspine_amd.runtime.worker import commit_accept
from dspine_amd.verification.tree import accept_greedy_tree, tree_masks

BF, HF, E4, I8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cls_name, c_name", [("KvCache", "dsv_kv_cache"), ("TreeAttentionArgs", "dsv_tree_attention_args")])
def test_struct_layout_matches_c(tmp_path, cls_name, c_name):
    cls = getattr(_lib, cls_name)
    names = [f[0] for f in cls._fields_]
    src = tmp_path / "layout.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "dspine_verify.h"', "int main(void) {",
             f'  printf("%zu\\n", sizeof({c_name}));']
    lines += [f'  printf("%zu\\n", offsetof({c_name}, {n}));' for n in names]
    src.write_text("\n".join([*lines, "  return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, n).offset for n in names]


def _cache(dtype=E4, slots=40, heads=2, dim=32):
    return new_cache(slots, heads, dim, dtype=dtype, device="cpu")


def _with(cache, **fields):
    return KVCache(**{**vars(cache), **fields})


def _unaligned(shape, dtype):
    """A contiguous tensor that starts one element past a 16-byte boundary."""
    n = 1
    for s in shape:
        n *= s
    flat = torch.zeros(n + 16, dtype=dtype)
    at = (-flat.data_ptr() // flat.element_size()) % (16 // flat.element_size()) + 1
    return flat[at:at + n].view(shape)


CACHES = {
    "rank": (lambda c: _with(c, k=c.k[0], v=c.v[0]), "k and v must be"),
    "shapes": (lambda c: _with(c, v=c.v[:-1]), "k and v must be"),
    "dtypes": (lambda c: _with(c, v=c.v.view(I8)), "k and v must be"),
    "float32": (lambda c: KVCache(c.k.float(), c.v.float()), "k and v must be"),
    "dim 24": (lambda c: KVCache(c.k[..., :24], c.v[..., :24], c.k_scale, c.v_scale), "multiple of 16"),
    "dim 272": (lambda c: _cache(dim=272), "multiple of 16"),
    "no slots": (lambda c: _cache(slots=0), "needs slots"),
    "one scale": (lambda c: _with(c, v_scale=None), "scales belong"),
    "no scales": (lambda c: _with(c, k_scale=None, v_scale=None), "scales belong"),
    "scales of a 16-bit cache": (lambda c: _with(_cache(BF), k_scale=c.k_scale, v_scale=c.v_scale), "scales belong"),
    "scale shape": (lambda c: _with(c, k_scale=c.k_scale[:, :1]), "k_scale must be"),
    "scale dtype": (lambda c: _with(c, v_scale=c.v_scale.half()), "v_scale must be"),
    "last stride": (lambda c: _with(c, k=torch.zeros((40, 2, 64), dtype=E4)[..., ::2]), "contiguous last dimension"),
    "alignment": (lambda c: _with(c, k=_unaligned((40, 2, 32), E4)), "16-byte"),
    "row stride": (lambda c: _with(c, v=torch.zeros((40, 2, 40), dtype=E4)[..., :32]), "16-byte"),
}


@pytest.mark.parametrize("case", CACHES)
def test_caches_that_are_refused(case):
    make, match = CACHES[case]
    cache = make(_cache())
    heads, dim = cache.k.shape[-2:]
    x = torch.zeros((3, heads, dim), dtype=BF)
    slots = torch.arange(3)
    with pytest.raises(ValueError, match=match):
        write_kv(cache, x, x, slots)
    with pytest.raises(ValueError, match=match):
        read_kv(cache, slots)
    with pytest.raises(ValueError, match=match):
        tree_attention(x, cache, T=1, page_table=torch.zeros((3, 4), dtype=torch.int32),
                       prefix_lens=torch.ones(3, dtype=torch.int32))


@pytest.mark.parametrize("field", ["k", "v", "k_scale", "v_scale"])
def test_a_cache_that_overlaps_itself_is_not_written(field):
    c = _cache()
    c = _with(c, **{field: getattr(c, field)[:1].expand(getattr(c, field).shape)})
    x = torch.zeros((3, 2, 32), dtype=BF)
    with pytest.raises(ValueError, match="must not overlap itself"):
        write_kv(c, x, x, torch.arange(3))
    with pytest.raises(ValueError, match="device .cuda. tensors"):  # (reading it is fine)
        read_kv(c, torch.arange(3))


X = torch.zeros((3, 2, 32), dtype=BF)
WRITES = {
    "ok": (dict(), "device .cuda. tensors"),
    "slots dtype": (dict(slots=torch.zeros(3)), "slots must be"),
    "slots rank": (dict(slots=torch.zeros((3, 1), dtype=torch.int64)), "slots must be"),
    "slots strided": (dict(slots=torch.arange(6)[::2]), "slots must be"),
    "length": (dict(slots=torch.arange(4)), "k and v must be bfloat16 or float16"),
    "heads": (dict(k=X[:, :1], v=X[:, :1]), "k and v must be bfloat16 or float16"),
    "dim": (dict(k=X[..., :16], v=X[..., :16]), "k and v must be bfloat16 or float16"),
    "dtype": (dict(k=X.float(), v=X.float()), "k and v must be bfloat16 or float16"),
    "two dtypes": (dict(v=X.half()), "k and v must be bfloat16 or float16"),
    "type of a 16-bit cache": (dict(cache=_cache(HF)), "its own dtype only"),
    "alignment": (dict(k=_unaligned((3, 2, 32), BF)), "k must have its rows on 16-byte"),
    "rows": (dict(v=torch.zeros((3, 2, 36), dtype=BF)[..., :32]), "v must have its rows on 16-byte"),
    "last stride": (dict(v=torch.zeros((3, 2, 64), dtype=BF)[..., ::2]), "contiguous last dimension"),
}


@pytest.mark.parametrize("case", WRITES)
def test_write_kv_refusals(case):
    change, match = WRITES[case]
    args = {**dict(cache=_cache(), k=X, v=X, slots=torch.arange(3)), **change}
    with pytest.raises(ValueError, match=match):
        write_kv(**args)


READS = {
    "ok": (dict(), "device .cuda. tensors"),
    "slots": (dict(slots=torch.zeros(3)), "slots must be"),
    "dtype": (dict(dtype=torch.float64), "unsupported dtype"),
    "out shape": (dict(out=(X[:2], X[:2])), "out must be two"),
    "out dtypes": (dict(out=(X, X.half())), "out must be two"),
    "out strided": (dict(out=(X, X.transpose(0, 1).contiguous().transpose(0, 1))), "out must be two"),
    "out alignment": (dict(out=(X, _unaligned((3, 2, 32), BF))), "16-byte boundary"),
}


@pytest.mark.parametrize("case", READS)
def test_read_kv_refusals(case):
    change, match = READS[case]
    with pytest.raises(ValueError, match=match):
        read_kv(**{**dict(cache=_cache(), slots=torch.arange(3)), **change})


def test_nothing_to_write_is_no_call():
    write_kv(_cache(), X[:0], X[:0], torch.arange(0))


Q = torch.zeros((6, 4, 32), dtype=BF)
I32 = torch.int32
ATTENDS = {
    "ok": (dict(), "device .cuda. tensors"),
    "q rank": (dict(q=Q[0]), "q must be bfloat16"),
    "q dtype": (dict(q=Q.float()), "q must be bfloat16"),
    "dim": (dict(q=Q[..., :16]), "cache's dim"),
    "heads": (dict(q=Q[:, :3]), "multiple of its heads"),
    "no heads": (dict(q=Q[:, :0]), "multiple of its heads"),
    "type of a 16-bit cache": (dict(cache=_cache(HF)), "one dtype"),
    "T 0": (dict(T=0), "outside"),
    "T 65": (dict(T=65), "outside"),
    "rows": (dict(T=2), "dense layout"),
    "prefix dtype": (dict(prefix_lens=torch.zeros(2, dtype=torch.int64)), "prefix_lens must be"),
    "no requests": (dict(prefix_lens=torch.zeros(0, dtype=I32)), "empty attention batch"),
    "offsets": (dict(row_offsets=torch.zeros(3, dtype=I32)), "row_offsets must be"),
    "offsets dtype": (dict(row_offsets=torch.zeros(2)), "row_offsets must be"),
    "verify_lens": (dict(verify_lens=torch.zeros(2, dtype=torch.int64)), "verify_lens must be"),
    "masks shape": (dict(masks=torch.zeros((2, 4), dtype=torch.int64)), "masks must be"),
    "masks dtype": (dict(masks=torch.zeros((2, 3), dtype=I32)), "masks must be"),
    "table dtype": (dict(page_table=torch.zeros((2, 9), dtype=torch.int64)), "page_table must be"),
    "table rows": (dict(page_table=torch.zeros((3, 9), dtype=I32)), "page_table must be"),
    "table without columns": (dict(page_table=torch.zeros((2, 0), dtype=I32)), "page_table must be"),
    "table strided": (dict(page_table=torch.zeros((2, 18), dtype=I32)[:, ::2]), "page_table rows"),
    "scale": (dict(scale=float("nan")), "finite"),
    "out shape": (dict(out=Q[:5]), "out must have q's"),
    "out dtype": (dict(out=Q.half()), "out must have q's"),
    "out overlaps": (dict(out=Q[:1].expand(6, 4, 32)), "must not overlap itself"),
    "out alignment": (dict(out=_unaligned((6, 4, 32), BF)), "out must have its rows on 16-byte"),
    "q alignment": (dict(q=_unaligned((6, 4, 32), BF)), "q must have its rows on 16-byte"),
    "lse": (dict(lse=torch.zeros((6, 2))), "lse must be"),
}


@pytest.mark.parametrize("case", ATTENDS)
def test_tree_attention_refusals(case):
    change, match = ATTENDS[case]
    args = dict(q=Q, cache=_cache(), T=3, page_table=torch.zeros((2, 9), dtype=I32), prefix_lens=torch.zeros(2, dtype=I32))
    with pytest.raises(ValueError, match=match):
        tree_attention(**{**args, **change})


PARENTS = torch.tensor([[-1, 0, 1]] * 2, dtype=I32)


def test_tree_masks_refusals():
    for parents, match in ((PARENTS.long(), "parents must be"), (PARENTS[0], "parents must be"), (PARENTS[:, ::2], "parents must be"),
                           (torch.zeros((2, 65), dtype=I32), "1 to 64"), (torch.zeros((2, 0), dtype=I32), "1 to 64"),
                           (PARENTS, "device .cuda. tensors")):
        with pytest.raises(ValueError, match=match):
            tree_masks(parents)
    with pytest.raises(ValueError, match="masks must be"):
        tree_masks(PARENTS, masks=torch.zeros((2, 3), dtype=I32))
    with pytest.raises(ValueError, match="depths must be"):
        tree_masks(PARENTS, depths=torch.zeros((2, 3), dtype=torch.int64))


LOGITS = torch.zeros((6, 11))
ACCEPTS = {
    "ok": (dict(), "device .cuda. tensors"),
    "parents": (dict(parents=PARENTS.long()), "parents must be"),
    "candidates": (dict(candidates=torch.zeros((2, 3), dtype=I32)), "candidates must be"),
    "no requests": (dict(candidates=torch.zeros((0, 3), dtype=torch.int64), parents=PARENTS[:0]), "empty verification"),
    "rows": (dict(next_token_logits=LOGITS[:5]), "bs.T, V. logits"),
    "columns": (dict(next_token_logits=torch.zeros((11, 6)).t()), "bs.T, V. logits"),
    "dtype": (dict(next_token_logits=LOGITS.half()), "dtype"),
    "prefix": (dict(prefix_lens=torch.zeros(2, dtype=torch.int64)), "prefix_lens must be"),
    "verify_lens": (dict(verify_lens=torch.zeros(3, dtype=I32)), "verify_lens must be"),
    "outputs": (dict(outputs=(torch.zeros(2, dtype=I32),) * 4), "Expected accept"),
    "output dtype": (dict(outputs=(torch.zeros(2, dtype=I32),) * 5), "output buffers"),
    "path": (dict(path=torch.zeros((2, 3), dtype=torch.int64)), "output buffers"),
}


@pytest.mark.parametrize("case", ACCEPTS)
def test_accept_greedy_tree_refusals(case):
    change, match = ACCEPTS[case]
    args = dict(candidates=torch.zeros((2, 3), dtype=torch.int64), parents=PARENTS, next_token_logits=LOGITS,
                prefix_lens=torch.zeros(2, dtype=I32))
    with pytest.raises(ValueError, match=match):
        accept_greedy_tree(**{**args, **change})


# -- the C entries ---------------------------------------------------------------------------------------------------

AT = 1 << 20  # an address that no refused call follows


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return _lib.load()


def _c_cache(**change):
    c = _lib.KvCache(AT, AT, _lib.DSV_E4M3, 2, 32, 0, 40, 64, 32, 64, 32, AT, AT, 2, 1, 2, 1)
    for name, value in change.items():
        setattr(c, name, value)
    return c


BAD_CACHES = [dict(k=None), dict(v=None), dict(k=AT + 8), dict(v=AT + 1), dict(dtype=_lib.DSV_F32), dict(dtype=7), dict(heads=0),
              dict(heads=65536), dict(dim=24), dict(dim=272), dict(dim=0), dict(num_slots=0), dict(k_slot_stride=8),
              dict(v_head_stride=24), dict(k_scale=None), dict(v_scale=None)]


@pytest.mark.parametrize("change", BAD_CACHES, ids=lambda d: "%s=%s" % next(iter(d.items())))
def test_c_entries_refuse_a_cache(lib, change):
    c = _c_cache(**change)
    assert lib.dsv_kv_write(c, AT, AT, _lib.DSV_BF16, 3, 64, 32, 64, 32, AT, 1, None) == _lib.DSV_ERR_INVALID
    assert lib.dsv_kv_read(c, AT, AT, _lib.DSV_BF16, 3, AT, 1, None) == _lib.DSV_ERR_INVALID
    assert lib.dsv_tree_attention(_c_attention(cache=c), None) == _lib.DSV_ERR_INVALID


def test_c_kv_refusals(lib):
    c, bad = _c_cache(), _lib.DSV_ERR_INVALID
    assert lib.dsv_kv_write(None, AT, AT, _lib.DSV_BF16, 3, 64, 32, 64, 32, AT, 1, None) == bad
    for args in ((AT, AT, _lib.DSV_F32, 3, 64, 32, 64, 32, AT), (AT, AT, _lib.DSV_BF16, -1, 64, 32, 64, 32, AT),
                 (None, AT, _lib.DSV_BF16, 3, 64, 32, 64, 32, AT), (AT, None, _lib.DSV_BF16, 3, 64, 32, 64, 32, AT),
                 (AT, AT, _lib.DSV_BF16, 3, 64, 32, 64, 32, None), (AT + 2, AT, _lib.DSV_BF16, 3, 64, 32, 64, 32, AT),
                 (AT, AT, _lib.DSV_BF16, 3, 60, 32, 64, 32, AT), (AT, AT, _lib.DSV_BF16, 3, 64, 32, 64, 33, AT)):
        assert lib.dsv_kv_write(c, *args, 1, None) == bad, args
    half = _c_cache(dtype=_lib.DSV_F16, k_scale=None, v_scale=None)
    assert lib.dsv_kv_write(half, AT, AT, _lib.DSV_BF16, 3, 64, 32, 64, 32, AT, 1, None) == bad
    for args in ((AT, AT, _lib.DSV_I8, 3, AT), (AT, AT, _lib.DSV_F32, -1, AT), (None, AT, _lib.DSV_F32, 3, AT),
                 (AT, AT + 4, _lib.DSV_F32, 3, AT), (AT, AT, _lib.DSV_F32, 3, None)):
        assert lib.dsv_kv_read(c, *args, 1, None) == bad, args
    assert lib.dsv_kv_write(c, AT, AT, _lib.DSV_BF16, 0, 64, 32, 64, 32, AT, 1, None) == _lib.DSV_OK
    assert lib.dsv_kv_read(c, AT, AT, _lib.DSV_F32, 0, AT, 1, None) == _lib.DSV_OK


def _c_attention(**change):
    a = _lib.TreeAttentionArgs(_c_cache(), AT, AT, None, _lib.DSV_BF16, 4, 6, 128, 32, 128, 32, 2, 3, AT, None, None, 0, 0.125, None,
                               AT, 9, 9, AT, 1 << 40)
    for name, value in change.items():
        setattr(a, name, value)
    return a


BAD_ATTENTION = [dict(dtype=_lib.DSV_F32), dict(q_heads=3), dict(q_heads=0), dict(bs=0), dict(T=0), dict(T=65), dict(rows=5), dict(rows=-1),
                 dict(q=None), dict(out=None), dict(prefix_lens=None), dict(page_table=None), dict(page_cols=0),
                 dict(page_cols=0x7fffffff), dict(q=AT + 8), dict(out=AT + 8), dict(q_row_stride=130), dict(q_head_stride=33),
                 dict(out_row_stride=132), dict(out_head_stride=36), dict(scale=float("inf")), dict(scale=float("nan")),
                 dict(workspace=None), dict(workspace=AT + 8), dict(cache=_c_cache(k_slot_stride=1 << 32)),
                 dict(bs=1 << 10, rows=3 << 10, page_cols=0x7fffff00)]


@pytest.mark.parametrize("change", BAD_ATTENTION, ids=lambda d: "%s=%s" % next(iter(d.items())))
def test_c_attention_refusals(lib, change):
    assert lib.dsv_tree_attention(_c_attention(**change), None) == _lib.DSV_ERR_INVALID


def test_c_workspaces_that_are_too_small(lib):
    need = lib.dsv_tree_attention_workspace_bytes(2, 3, 2, 4, 32)
    assert need > 0 and lib.dsv_tree_attention(_c_attention(workspace_bytes=need - 1), None) == _lib.DSV_ERR_WORKSPACE
    assert lib.dsv_tree_attention_workspace_bytes(0, 3, 2, 4, 32) == 0
    need = lib.dsv_tree_verify_workspace_bytes(6, 11)
    args = [AT, _lib.DSV_F32, 6, 11, 11, 2, 3, AT, AT, None, AT, AT, AT, AT, AT, AT, AT, AT]
    assert need > 0 and lib.dsv_tree_verify(*args, need - 1, None) == _lib.DSV_ERR_WORKSPACE
    for at, value in ((0, None), (1, _lib.DSV_F16), (2, 5), (3, 0), (4, 10), (5, 0), (6, 65), (7, None), (8, None), (10, None),
                      (16, None), (17, None)):
        assert lib.dsv_tree_verify(*(value if i == at else x for i, x in enumerate(args)), need, None) == _lib.DSV_ERR_INVALID, at


def test_c_tree_refusals(lib):
    bad = _lib.DSV_ERR_INVALID
    assert lib.dsv_tree_masks(AT, 2, 65, AT, AT, None) == bad
    assert lib.dsv_tree_masks(AT, -1, 3, AT, AT, None) == bad
    assert lib.dsv_tree_masks(None, 2, 3, AT, AT, None) == bad
    assert lib.dsv_tree_masks(AT, 2, 3, None, AT, None) == bad
    assert lib.dsv_tree_masks(AT, 0, 3, AT, AT, None) == _lib.DSV_OK
    args = [2, 3, AT, AT, None, AT, 0, AT, 0, AT, 9, 9, None, None, None, 0, AT, AT]
    for at, value in ((0, -1), (1, 0), (1, 65), (2, None), (3, None), (5, None), (7, None), (9, None), (10, 8), (11, 0)):
        assert lib.dsv_commit_tree(*(value if i == at else x for i, x in enumerate(args)), None) == bad, at


def test_commit_of_a_path_on_the_cpu_is_refused():
    out = (torch.zeros(2, dtype=I32), None, None, torch.zeros((2, 3), dtype=torch.int64))
    with pytest.raises(ValueError, match="device .cuda. tensors"):
        commit_accept(out, prefix_lens=torch.zeros(2, dtype=I32), req_pool_indices=torch.zeros(2, dtype=I32),
                      req_to_token=torch.zeros((2, 9), dtype=I32), path=torch.zeros((2, 3), dtype=I32))
