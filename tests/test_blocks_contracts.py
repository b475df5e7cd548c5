"""What the block operators and the calls on requests refuse, before any launch (no GPU): calls on CPU tensors raise
ValueError, the C entries return DSV_ERR_INVALID or DSV_ERR_WORKSPACE with nothing launched.

Argument checks come before the check of the device, so a call that passes them all ends at "device (cuda)
tensors" here: every case starts from such a call."""

import ctypes
import math
import os
import subprocess

import blocks_ref as B
import pytest
import torch

from dspine_amd import _lib
from dspine_amd.kernels.blocks import (BlockIndex, block_attention, index_blocks, new_block_index, score_blocks,
                                       select_blocks)
from dspine_amd.kernels.cache import KVCache, copy_kv, new_cache, slot_rows
from dspine_amd.runtime.requests import compact_requests, fork_requests, free_requests

BF, HF, E4, I8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8
I32, I64, F32 = torch.int32, torch.int64, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GPU = "device .cuda. tensors"


@pytest.mark.parametrize("cls_name, c_name", [("BlockIndexC", "dsv_block_index"), ("ScoreBlocksArgs", "dsv_score_blocks_args"),
                                              ("BlockAttentionArgs", "dsv_block_attention_args"), ("SlotRows", "dsv_slot_rows")])
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


def _z(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


def _unaligned(shape, dtype):
    n = math.prod(shape)
    flat = torch.zeros(n + 16, dtype=dtype)
    at = (-flat.data_ptr() // flat.element_size()) % (16 // flat.element_size()) + 1
    return flat[at:at + n].view(shape)


def _index(dtype=BF, rows=9, heads=2, dim=32, size=16):
    return new_block_index(rows, heads, dim, block_size=size, dtype=dtype, device="cpu")


def _cache(dtype=E4, slots=40, heads=2, dim=32):
    return new_cache(slots, heads, dim, dtype=dtype, device="cpu")


INDEXES = {
    "rank": (lambda: BlockIndex(_z(9, 2, 32, dtype=BF), 16), "bounds must be"),
    "no pair": (lambda: BlockIndex(_z(9, 2, 3, 32, dtype=BF), 16), "bounds must be"),
    "dtype": (lambda: BlockIndex(_z(9, 2, 2, 32, dtype=F32), 16), "bounds must be"),
    "strided": (lambda: BlockIndex(_z(9, 2, 2, 64, dtype=BF)[..., :32], 16), "bounds must be"),
    "dim 24": (lambda: BlockIndex(_z(9, 2, 2, 24, dtype=BF), 16), "multiple of 16"),
    "dim 272": (lambda: BlockIndex(_z(9, 2, 2, 272, dtype=BF), 16), "multiple of 16"),
    "no rows": (lambda: BlockIndex(_z(0, 2, 2, 32, dtype=BF), 16), "needs rows"),
    "alignment": (lambda: BlockIndex(_unaligned((9, 2, 2, 32), BF), 16), "16-byte"),
    "size 8": (lambda: BlockIndex(_z(9, 2, 2, 32, dtype=BF), 8), "16, 32, 64 or 128"),
    "size 48": (lambda: BlockIndex(_z(9, 2, 2, 32, dtype=BF), 48), "16, 32, 64 or 128"),
    "size 256": (lambda: BlockIndex(_z(9, 2, 2, 32, dtype=BF), 256), "16, 32, 64 or 128"),
}


@pytest.mark.parametrize("case", INDEXES)
def test_indexes_that_are_refused(case):
    make, match = INDEXES[case]
    with pytest.raises(ValueError, match=match):
        index_blocks(make(), _cache(), page_table=_z(3, 40), block_table=_z(3, 2), from_lens=_z(3), to_lens=_z(3))
    with pytest.raises(ValueError, match=match):
        score_blocks(_z(3, 4, 32, dtype=BF), make(), T=1, block_table=_z(3, 2), prefix_lens=_z(3))


def test_new_block_index():
    x = _index(HF, 5, 3, 48, 128)
    assert x.bounds.shape == (5, 3, 2, 48) and x.bounds.dtype == HF and x.block_size == 128 and not bool(x.bounds.any())
    for bad in (dict(dtype=F32), dict(dtype=E4), dict(dim=20), dict(size=17), dict(heads=0)):
        with pytest.raises(ValueError):
            _index(**bad)


INDEX_CALLS = {
    "ok": (dict(), GPU), "ok, a growth": (dict(longest=5), GPU), "empty": (dict(longest=0), GPU),
    "heads": (dict(cache=_cache(heads=1)), "same heads and dim"), "dim": (dict(cache=_cache(dim=48)), "same heads and dim"),
    "from dtype": (dict(from_lens=_z(3, dtype=I64)), "from_lens must be"), "to length": (dict(to_lens=_z(4)), "to_lens must be"),
    "to strided": (dict(to_lens=_z(6)[::2]), "to_lens must be"), "pages": (dict(page_table=_z(2, 40)), "page_table must be"),
    "page dtype": (dict(page_table=_z(3, 40, dtype=I64)), "page_table must be"),
    "page rows": (dict(page_table=_z(3, 80)[:, ::2]), "page_table rows"), "no pages": (dict(page_table=_z(3, 0)), "page_table must be"),
    "blocks": (dict(block_table=_z(3)), "block_table must be"), "block rows": (dict(block_table=_z(2, 3).t()), "block_table rows"),
    "negative": (dict(longest=-1), "negative"),
}


@pytest.mark.parametrize("case", INDEX_CALLS)
def test_index_calls(case):
    change, match = INDEX_CALLS[case]
    args = dict(cache=_cache(), page_table=_z(3, 40), block_table=_z(3, 2), from_lens=_z(3), to_lens=_z(3))
    with pytest.raises(ValueError, match=match):
        index_blocks(_index(), **{**args, **change})


SCORES = {
    "ok": (dict(), GPU), "ok, compact rows": (dict(q=_z(5, 4, 32, dtype=BF), row_offsets=_z(3), verify_lens=_z(3)), GPU),
    "no rows": (dict(q=_z(0, 4, 32, dtype=BF), row_offsets=_z(3)), GPU),
    "q rank": (dict(q=_z(6, 32, dtype=BF)), "q must be"), "q dtype": (dict(q=_z(6, 4, 32, dtype=F32)), "q must be"),
    "two dtypes": (dict(q=_z(6, 4, 32, dtype=HF)), "one dtype"), "dim": (dict(q=_z(6, 4, 48, dtype=BF)), "index's dim"),
    "heads": (dict(q=_z(6, 3, 32, dtype=BF)), "multiple of its heads"), "T 0": (dict(T=0), "outside"), "T 65": (dict(T=65), "outside"),
    "rows": (dict(q=_z(7, 4, 32, dtype=BF)), "dense layout"), "offsets": (dict(row_offsets=_z(4)), "row_offsets must"),
    "lens": (dict(verify_lens=_z(3, dtype=I64)), "verify_lens must"), "prefix": (dict(prefix_lens=_z(3, dtype=I64)), "prefix_lens must"),
    "no batch": (dict(prefix_lens=_z(0)), "empty"), "table": (dict(block_table=_z(2, 5)), "block_table must"),
    "scale 0": (dict(scale=0.0), "scale"), "scale < 0": (dict(scale=-1.0), "scale"), "scale nan": (dict(scale=math.nan), "scale"),
    "scale inf": (dict(scale=math.inf), "scale"), "out": (dict(out=_z(3, 2, 4, dtype=F32)), "out must"),
    "out dtype": (dict(out=_z(3, 2, 5, dtype=BF)), "out must"), "q alignment": (dict(q=_unaligned((6, 4, 32), BF)), "16-byte"),
}


@pytest.mark.parametrize("case", SCORES)
def test_score_calls(case):
    change, match = SCORES[case]
    args = dict(q=_z(6, 4, 32, dtype=BF), index=_index(), T=2, block_table=_z(3, 5), prefix_lens=_z(3))
    with pytest.raises(ValueError, match=match):
        score_blocks(**{**args, **change})


SELECT = {
    "ok": (dict(), GPU), "ok, all forced": (dict(count=5, first=2, last=3), GPU), "ok, widest": (dict(scores=_z(3, 2, 32768, dtype=F32)), GPU),
    "rank": (dict(scores=_z(3, 5, dtype=F32)), "scores must"), "dtype": (dict(scores=_z(3, 2, 5, dtype=BF)), "scores must"),
    "strided": (dict(scores=_z(3, 2, 10, dtype=F32)[..., ::2]), "scores must"), "none": (dict(scores=_z(3, 2, 0, dtype=F32)), "32768"),
    "too wide": (dict(scores=_z(3, 2, 32769, dtype=F32)), "32768"), "no heads": (dict(scores=_z(3, 0, 5, dtype=F32)), "empty"),
    "prefix": (dict(prefix_lens=_z(2)), "prefix_lens"), "size": (dict(block_size=20), "16, 32, 64 or 128"),
    "count 0": (dict(count=0), "count 0"), "forced": (dict(count=4, first=2, last=3), "has to hold"),
    "first": (dict(first=-1), "has to hold"), "last": (dict(last=-1), "has to hold"), "count": (dict(count=2 ** 24 + 1), "count"),
    "out": (dict(out=_z(3, 2, 5)), "out must"), "out dtype": (dict(out=_z(3, 2, 4, dtype=I64)), "out must"),
}


@pytest.mark.parametrize("case", SELECT)
def test_select_calls(case):
    change, match = SELECT[case]
    args = dict(scores=_z(3, 2, 5, dtype=F32), count=4, prefix_lens=_z(3), block_size=16)
    with pytest.raises(ValueError, match=match):
        select_blocks(**{**args, **change})


ATTEND = {
    "ok": (dict(), GPU), "more blocks than pages": (dict(blocks=_z(3, 2, 99)), GPU),
    "size": (dict(block_size=40), "16, 32, 64 or 128"), "rank": (dict(blocks=_z(3, 4)), "blocks must"),
    "batch": (dict(blocks=_z(2, 2, 4)), "blocks must"), "heads": (dict(blocks=_z(3, 4, 4)), "blocks must"),
    "none": (dict(blocks=_z(3, 2, 0)), "blocks must"), "dtype": (dict(blocks=_z(3, 2, 4, dtype=I64)), "blocks must"),
    "strided": (dict(blocks=_z(3, 2, 8)[..., ::2]), "blocks must"),
    "as the tree's": (dict(T=65), "outside"), "masks": (dict(masks=_z(3, 2)), "masks must"), "scale": (dict(scale=2.0 ** 101), "scale"),
    "dtype of the cache": (dict(cache=_cache(HF)), "one dtype"),
}


@pytest.mark.parametrize("case", ATTEND)
def test_attention_calls(case):
    change, match = ATTEND[case]
    args = dict(q=_z(6, 4, 32, dtype=BF), cache=_cache(), T=2, blocks=_z(3, 2, 4), block_size=16, page_table=_z(3, 40),
                prefix_lens=_z(3))
    with pytest.raises(ValueError, match=match):
        block_attention(**{**args, **change})


TABLE = dict(req_to_token=_z(5, 30), seq_lens=_z(5), shared=_z(40))
TABLES = {
    "rank": (dict(req_to_token=_z(30)), "req_to_token must be"), "dtype": (dict(req_to_token=_z(5, 30, dtype=I64)), "req_to_token must be"),
    "rows": (dict(req_to_token=_z(5, 60)[:, ::2]), "req_to_token must be"), "overlap": (dict(req_to_token=_z(1, 30).expand(5, 30)), "overlap"),
    "no columns": (dict(req_to_token=_z(5, 0)), "req_to_token must be"), "lens": (dict(seq_lens=_z(4)), "seq_lens must"),
    "lens dtype": (dict(seq_lens=_z(5, dtype=F32)), "seq_lens must"), "lens strided": (dict(seq_lens=_z(10)[::2]), "seq_lens must"),
}
SHARED = {"shared dtype": (dict(shared=_z(40, dtype=I64)), "shared must"), "no slots": (dict(shared=_z(0)), "shared must"),
          "shared strided": (dict(shared=_z(80)[::2]), "shared must")}


@pytest.mark.parametrize("case", [*TABLES, *SHARED])
def test_tables_that_are_refused(case):
    change, match = {**TABLES, **SHARED}[case]
    args = {**TABLE, **change}
    with pytest.raises(ValueError, match=match):
        fork_requests(**args, parents=_z(2), children=_z(2))
    with pytest.raises(ValueError, match=match):
        free_requests(**args, rows=_z(2))
    with pytest.raises(ValueError, match=match):
        compact_requests(**args, rows=_z(2), caches=_cache())


def test_calls_on_requests():
    for change, match in [(dict(), GPU), (dict(parents=_z(0), children=_z(0)), GPU), (dict(children=_z(3)), "one length"),
                          (dict(children=_z(2, dtype=I64)), "one length and dtype"), (dict(parents=_z(2, dtype=F32)), "parents must"),
                          (dict(children=_z(4)[::2]), "children must")]:
        with pytest.raises(ValueError, match=match):
            fork_requests(**{**TABLE, **dict(parents=_z(2), children=_z(2)), **change})
    for change, match in [(dict(), GPU), (dict(rows=_z(0, dtype=I64)), GPU), (dict(rows=_z(2, 1)), "rows must"),
                          (dict(free_slots=_z(9)), "free_slots must"), (dict(free_slots=_z(18, dtype=I64)[::2]), "free_slots must"),
                          (dict(free_count=_z(1, dtype=I64)), "free_count must")]:
        with pytest.raises(ValueError, match=match):
            free_requests(**{**TABLE, "rows": _z(2), **change})
    for change, match in [(dict(), GPU), (dict(shared=None), GPU), (dict(caches=[_cache(), _index(rows=40)]), GPU),
                          (dict(caches=[]), "must be a cache"), (dict(caches=[_cache(), _cache(slots=41)]), "one number"),
                          (dict(caches=[_cache().k]), "KVCache or BlockIndex"), (dict(shared=_z(41)), "shared must count"),
                          (dict(moves=_z(2, 19, dtype=I64)), "moves must"), (dict(moves=_z(2, 20)), "moves must"),
                          (dict(moves=_z(3, 20, dtype=I64)), "moves must"), (dict(counts=_z(1)), "counts must"),
                          (dict(rows=_z(2, dtype=I8)), "rows must"),
                          (dict(caches=KVCache(_z(1, 2, 32, dtype=BF).expand(40, 2, 32), _cache(BF).v)), "overlap")]:
        with pytest.raises(ValueError, match=match):
            compact_requests(**{**TABLE, "rows": _z(2), "caches": _cache(), **change})
    for change, match in [(dict(), GPU), (dict(src=_z(3, dtype=F32)), "slots must"), (dict(dst=_z(2)), "one length"),
                          (dict(count=_z(1, dtype=I64)), "count must"), (dict(caches=[None]), "KVCache or BlockIndex")]:
        with pytest.raises(ValueError, match=match):
            copy_kv(**{**dict(caches=_cache(), src=_z(3), dst=_z(3, dtype=I64)), **change})


def test_slot_rows_of_caches():
    quant, plain, index = _cache(E4, 7, 3, 48), _cache(BF, 7, 1, 16), _index(HF, 7, 2, 32)
    wide = torch.zeros(7, 2, 3, 48, dtype=BF)
    rows, tensors, slots = slot_rows([quant, plain, index, KVCache(wide[:, 0], wide[:, 1])])
    assert slots == 7 and len(tensors) == len(rows) == 9
    got = [(r.slot_stride, r.head_stride if r.heads > 1 else 0, r.heads, r.bytes) for r in rows]
    assert got == [(144, 48, 3, 48)] * 2 + [(12, 4, 3, 4)] * 2 + [(32, 0, 1, 32)] * 2 + [(256, 0, 1, 256)] + [(576, 96, 3, 96)] * 2
    assert [r.base for r in rows] == [t.data_ptr() for t in tensors]


# ---------------------------------------------------------------------------------------------
# the C entries
# ---------------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.load()


P = 0x1000  # (an address that nothing reads: every call here is refused)


def _refused(lib, rc, match, code=_lib.DSV_ERR_INVALID):
    assert rc == code and match in lib.dsv_last_error().decode(), (rc, lib.dsv_last_error())


def _c_cache(**kw):
    f = dict(k=P, v=P, dtype=_lib.DSV_BF16, heads=2, dim=32, num_slots=40, k_slot_stride=64, k_head_stride=32, v_slot_stride=64,
             v_head_stride=32)
    return _lib.KvCache(**{**f, **kw})


def _c_index(**kw):
    return _lib.BlockIndexC(**{**dict(bounds=P, dtype=_lib.DSV_BF16, heads=2, dim=32, block_size=16, rows=9), **kw})


@pytest.mark.parametrize("change, match", [
    (dict(bounds=0), "bounds are required"), (dict(bounds=P + 8), "16-byte"), (dict(dtype=_lib.DSV_E4M3), "index type"),
    (dict(heads=0), "needs rows"), (dict(dim=40), "multiple of 16"), (dict(rows=0), "needs rows"), (dict(block_size=0), "16, 32, 64 or 128"),
    (dict(block_size=-16), "16, 32, 64 or 128"), (dict(heads=3), "same heads")])
def test_c_index_refuses(lib, change, match):
    _refused(lib, lib.dsv_index_blocks(_c_index(**change), _c_cache(), P, 40, 40, P, 3, 3, P, P, 3, 40, None), match)
    if match != "same heads":
        a = _lib.ScoreBlocksArgs(index=_c_index(**change), q=P, scores=P, q_heads=4, rows=3, q_row_stride=128, q_head_stride=32,
                                 bs=3, T=1, prefix_lens=P, scale=1.0, block_table=P, block_stride=3, block_cols=3)
        _refused(lib, lib.dsv_score_blocks(a, None), match)


def test_c_index_calls_refuse(lib):
    ok = [_c_index(), _c_cache(), P, 40, 40, P, 3, 3, P, P, 3, 40, None]
    for at, value, match in [(0, None, "no index"), (1, None, "k and v"), (2, None, "required"), (4, 0, "required"), (5, None, "required"),
                             (7, 0, "required"), (8, None, "required"), (9, None, "required"), (10, -1, "invalid layout"),
                             (11, -1, "invalid layout")]:
        _refused(lib, lib.dsv_index_blocks(*(value if i == at else x for i, x in enumerate(ok))), match)
    big = [_c_index(), _c_cache(), P, 40, 40, P, 3, 2 ** 30, P, P, 2 ** 20, 2 ** 31, None]
    _refused(lib, lib.dsv_index_blocks(*big), "too many")
    assert lib.dsv_index_blocks(*(0 if i == 10 else x for i, x in enumerate(ok))) == _lib.DSV_OK
    assert lib.dsv_index_blocks(*(0 if i == 11 else x for i, x in enumerate(ok))) == _lib.DSV_OK


@pytest.mark.parametrize("change, match", [
    (dict(bs=0), "invalid layout"), (dict(T=65), "invalid layout"), (dict(rows=4), "invalid layout"), (dict(q_heads=3), "query heads"),
    (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scores=0), "required"), (dict(prefix_lens=0), "required"),
    (dict(block_table=0), "required"), (dict(block_cols=0), "required"), (dict(q=0), "required"), (dict(q=P + 2), "16-byte"),
    (dict(q_row_stride=130), "16-byte"), (dict(bs=2 ** 24, rows=2 ** 24, block_cols=2 ** 26), "too many")])
def test_c_scores_refuse(lib, change, match):
    f = dict(index=_c_index(), q=P, scores=P, q_heads=4, rows=3, q_row_stride=128, q_head_stride=32, bs=3, T=1, prefix_lens=P,
             scale=1.0, block_table=P, block_stride=3, block_cols=3)
    _refused(lib, lib.dsv_score_blocks(_lib.ScoreBlocksArgs(**{**f, **change}), None), match)
    _refused(lib, lib.dsv_score_blocks(None, None), "no arguments")


def test_c_selection_refuses(lib):
    ok = [P, 3, 2, 5, P, 16, 4, 1, 2, P, None]
    for at, value, match in [(0, None, "null"), (1, 0, "ranked"), (2, 0, "ranked"), (3, 0, "ranked"), (3, 32769, "ranked"),
                             (4, None, "null"), (5, 17, "16, 32, 64 or 128"), (6, 0, "has to hold"), (6, 2, "has to hold"),
                             (7, -1, "has to hold"), (8, -1, "has to hold"), (9, None, "null")]:
        _refused(lib, lib.dsv_select_blocks(*(value if i == at else x for i, x in enumerate(ok))), match)


@pytest.mark.parametrize("change, tree, match", [
    (dict(blocks=0), {}, "lists of blocks"), (dict(count=0), {}, "0 blocks"), (dict(count=2 ** 27), {}, "blocks of"),
    (dict(block_size=8), {}, "16, 32, 64 or 128"), (dict(block_size=192), {}, "16, 32, 64 or 128"), ({}, dict(T=65), "invalid layout"),
    ({}, dict(q=0), "required"), ({}, dict(workspace=0), "workspace"), ({}, dict(scale=math.inf), "scale"),
    (dict(count=2 ** 26), dict(bs=2 ** 12, rows=2 ** 12), "too many")])
def test_c_attention_refuses(lib, change, tree, match):
    t = dict(cache=_c_cache(), q=P, out=P, dtype=_lib.DSV_BF16, q_heads=4, rows=3, q_row_stride=128, q_head_stride=32,
             out_row_stride=128, out_head_stride=32, bs=3, T=1, prefix_lens=P, scale=1.0, page_table=P, page_stride=40, page_cols=40,
             workspace=P, workspace_bytes=2 ** 40)
    a = _lib.BlockAttentionArgs(**{**dict(tree=_lib.TreeAttentionArgs(**{**t, **tree}), blocks=P, count=4, block_size=16), **change})
    _refused(lib, lib.dsv_block_attention(a, None), match)
    _refused(lib, lib.dsv_block_attention(None, None), "no arguments")
    t["workspace_bytes"] = 16
    small = _lib.BlockAttentionArgs(tree=_lib.TreeAttentionArgs(**t), blocks=P, count=4, block_size=16)
    _refused(lib, lib.dsv_block_attention(small, None), "workspace 16 <", _lib.DSV_ERR_WORKSPACE)


def test_c_calls_on_requests_refuse(lib):
    rows = (_lib.SlotRows * 1)(_lib.SlotRows(P, 256, 64, 2, 64))
    table = [P, 5, 30, 30, P, 0]  # table, rows, stride, columns, lengths, i64
    fork = [*table, P, 40, P, P, 0, 2, None]
    free = [*table, P, 40, P, 0, 2, P, 60, P, P, 2 ** 20, None]
    compact = [*table, P, 40, P, 0, 2, rows, 1, P, P, 20, P, P, 2 ** 20, None]
    for entry, ok, n in (("dsv_fork_requests", fork, 11), ("dsv_free_requests", free, 10), ("dsv_compact_requests", compact, 10)):
        for at, value, match in [(0, None, "required"), (1, 0, "required"), (2, 29, "required"), (3, 0, "required"), (4, None, "required"),
                                 (7, 0, "slots"), (7, 2 ** 31, "slots"), (8, None, "required"), (n, -1, "n -1"), (n, 2 ** 31, "n ")]:
            _refused(lib, getattr(lib, entry)(*(value if i == at else x for i, x in enumerate(ok))), match)
        wide = list(ok)
        wide[2], wide[3], wide[n] = 2 ** 31, 2 ** 31, 2 ** 10
        _refused(lib, getattr(lib, entry)(*wide), "too many")

    def all_of(entry, ok, changes):
        for at, value, match, *code in changes:
            _refused(lib, getattr(lib, entry)(*(value if i == at else x for i, x in enumerate(ok))), match, *code)

    all_of("dsv_fork_requests", fork, [(6, None, "required"), (9, None, "required")])
    all_of("dsv_free_requests", free, [(6, None, "required"), (11, None, "required"), (12, -1, "required"), (13, None, "required"),
                                       (14, None, "workspace"), (14, P + 4, "workspace"), (15, 3, "workspace 3 <", _lib.DSV_ERR_WORKSPACE)])
    all_of("dsv_compact_requests", compact, [(11, None, "rows are required"), (13, None, "room"), (14, None, "room"), (15, 19, "room"),
                                             (16, None, "room"), (17, None, "workspace"),
                                             (18, 40, "workspace 40 <", _lib.DSV_ERR_WORKSPACE)])
    copy = [rows, 1, 40, P, 0, P, 0, 3, None, None]
    all_of("dsv_copy_slots", copy, [(0, None, "required"), (1, -1, "required"), (2, 0, "required"), (2, 2 ** 31, "required"),
                                    (3, None, "null"), (5, None, "null"), (7, -1, "n -1")])
    for bad in ((0, 256, 64, 2, 64), (P, 256, 64, 0, 64), (P, 256, 64, 2, 0), (P, 256, 64, 2, 6), (P + 2, 256, 64, 2, 64),
                (P, 258, 64, 2, 64), (P, 256, -4, 2, 64), (P, 256, 64, 2 ** 20, 64)):
        _refused(lib, lib.dsv_copy_slots((_lib.SlotRows * 1)(_lib.SlotRows(*bad)), *copy[1:]), "4-byte words")
    assert lib.dsv_copy_slots(*(0 if i == 7 else x for i, x in enumerate(copy))) == _lib.DSV_OK
    assert lib.dsv_fork_requests(*(0 if i == 11 else x for i, x in enumerate(fork))) == _lib.DSV_OK


def test_workspace_sizes(lib):
    assert lib.dsv_free_requests_workspace_bytes(0) == lib.dsv_compact_requests_workspace_bytes(-5) == 0
    assert lib.dsv_free_requests_workspace_bytes(1) >= 4 and lib.dsv_compact_requests_workspace_bytes(4097) >= 2 * 4096 * 5 + 8


# ---------------------------------------------------------------------------------------------
# the references themselves, on cases done by hand
# ---------------------------------------------------------------------------------------------


def test_references_by_hand():
    s = torch.tensor([[[1.0, 5.0, math.nan, 5.0, -math.inf, 7.0, 9.0]]])
    got = B.select(s, 4, prefix_lens=torch.tensor([6 * 16 + 3]), block_size=16, first=1)
    assert got.tolist() == [[[0, 1, 3, 5]]]
    got = B.select(s, 4, prefix_lens=torch.tensor([3 * 16]), block_size=16, last=1)
    assert got.tolist() == [[[0, 1, 2, -1]]]
    table = torch.tensor([[5, 8, 1], [5, 8, 2], [0, 0, 0]], dtype=I32)
    lens, shared = torch.tensor([3, 3, 0], dtype=I32), _z(9)
    shared[[5, 8]] = 1
    B.fork(table, lens, shared, [0], [2])
    assert table[2].tolist() == [5, 8, 1] and lens.tolist() == [3, 3, 3] and shared.tolist() == [0, 1, 0, 0, 0, 2, 0, 0, 2]
    assert B.free(table, lens, shared, [1]) == [2] and shared.tolist() == [0, 1, 0, 0, 0, 1, 0, 0, 1]
    src, dst, used = B.compact(table, lens, [0, 2], 9, shared)
    assert (src, dst, used) == ([5, 8], [0, 2], 3) and table[[0, 2]].tolist() == [[0, 2, 1]] * 2 and shared.tolist() == [1, 1, 1] + [0] * 6
    assert B.free(table, lens, shared, [2, 2]) == [] and B.free(table, lens, shared, [0]) == [0, 1, 2]
