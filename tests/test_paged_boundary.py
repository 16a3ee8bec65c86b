"""Refusals of the paged-cache operators: constructors, buffers and the C entry points (no
launch happens in any of them, so they run without a GPU)."""

import ctypes

import pytest
import torch

from iron_b200 import _lib
from iron_b200.operators import PageAppend, PageCompact, PageFork, PageSelectAttention, TreeAttention

POOL = dict(num_kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4)
TREE = dict(batch=2, num_nodes=4, num_heads=4, **POOL)
SELECT = dict(batch=2, num_heads=4, top_pages=3, **POOL)
SLOTS = dict(slots=2, num_layers=1, **POOL)


@pytest.mark.parametrize("cls,good", [(TreeAttention, TREE), (PageSelectAttention, SELECT), (PageAppend, SLOTS | {"num_new": 3}),
                                      (PageFork, SLOTS), (PageCompact, SLOTS)])
@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(page_size=48), dict(num_pages=0), dict(max_pages=0), dict(num_kv_heads=0),
                                 dict(max_pages=1 << 27)])
def test_constructor_geometry(cls, good, bad):
    cls(**good)
    with pytest.raises(ValueError):
        cls(**(good | bad))


@pytest.mark.parametrize("cls,good,bad", [
    (TreeAttention, TREE, dict(num_nodes=0)), (TreeAttention, TREE, dict(num_nodes=129)), (TreeAttention, TREE, dict(batch=1025)),
    (TreeAttention, TREE, dict(num_heads=5)), (TreeAttention, TREE, dict(num_heads=34)), (PageSelectAttention, SELECT, dict(top_pages=0)),
    (PageSelectAttention, SELECT, dict(num_heads=3)), (PageSelectAttention, SELECT, dict(batch=0)), (PageAppend, SLOTS, dict(num_new=0)),
    (PageAppend, SLOTS, dict(slots=2049)), (PageFork, SLOTS, dict(num_layers=0)), (PageCompact, SLOTS, dict(slots=0))])
def test_constructor_sizes(cls, good, bad):
    with pytest.raises(ValueError):
        cls(**(good | bad))


def test_buffers_are_checked():
    op = PageSelectAttention(**SELECT)
    t = {torch.bfloat16: [], torch.int32: []}
    q, out = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16)
    codes, scales = torch.zeros(8, 2, 2, 64, dtype=torch.int8), torch.zeros(8, 2)
    table, lens, sel = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 3, dtype=torch.int32)
    good = [q, k, k, codes, scales, table, lens, out, sel]
    op._check_buffers(good)
    wide = torch.zeros(2, 6, 64, dtype=torch.bfloat16)
    op._check_buffers([wide[:, :4]] + good[1:])  # q may be a view of a wider buffer
    for i, bad, msg in [(0, q.float(), "needs torch.bfloat16"), (1, k[:7], "holds"), (5, table.long(), "needs torch.int32"),
                        (1, k.transpose(1, 2), "contiguous"), (0, q.transpose(1, 2).contiguous().transpose(1, 2), "last dimension"),
                        (8, sel[:1], "holds")]:
        with pytest.raises(ValueError, match=msg):
            op._check_buffers(good[:i] + [bad] + good[i + 1 :])
    with pytest.raises(ValueError, match="takes 9 buffers"):
        op._check_buffers(good[:-1])
    del t


def pool(**change):
    f = dict(k=4096, v=4096, codes=None, scales=None, page_table=4096, lens=4096, refs=4096, layers=1, slots=2, num_pages=8,
             max_pages=4, kv_heads=2, head_dim=64, page_size=16) | change
    return _lib.PagePool(**f)


def tree(p, q=4096, n=4, heads=4, ws=1 << 30, st=(0, 64, 64), kst=(0, 64, 64)):
    s = (ctypes.c_int64 * 3)(*st)
    ks = (ctypes.c_int64 * 3)(*kst)
    return _lib.load().iron_tree_attn(ctypes.byref(p) if p else None, q, 4096, 4096, 4096, 4096, n, heads, s, ks, s, 0.125, 4096, ws, 0, None)


def select(p, q=4096, top=3, heads=4, ws=1 << 30, st=(256, 64)):
    s = (ctypes.c_int64 * 2)(*st)
    return _lib.load().iron_page_select_attn(ctypes.byref(p) if p else None, q, 4096, 4096, heads, top, s, s, 0.125, 4096, ws, 0, None)


def append(p, k=4096, n=3, ws=1 << 30, index=4096):
    return _lib.load().iron_page_append(ctypes.byref(p) if p else None, k, 4096, index, n, 4096, 4096, 4096, ws, 0, None)


def fork(p, table=1 << 20, refs=1 << 21, ws=1 << 30):
    return _lib.load().iron_page_fork(ctypes.byref(p) if p else None, 4096, table, 4096, refs, 4096, 4096, ws, 0, None)


def compact(p, table=4096, refs=4096, ws=1 << 30):
    return _lib.load().iron_page_compact(ctypes.byref(p) if p else None, table, refs, 4096, 4096, ws, 0, None)


NULL, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, ARG = -1, -2, -3, -4, -6, -8
GEOMETRY = [(dict(k=None), NULL), (dict(v=None), NULL), (dict(page_table=None), NULL), (dict(slots=0), SHAPE), (dict(num_pages=0), SHAPE),
            (dict(max_pages=-1), SHAPE), (dict(kv_heads=0), SHAPE), (dict(num_pages=(1 << 24) + 1), SHAPE), (dict(head_dim=80), UNSUPPORTED),
            (dict(page_size=24), UNSUPPORTED), (dict(page_size=256), UNSUPPORTED), (dict(max_pages=1 << 27), SHAPE), (dict(k=4104), ALIGN),
            (dict(v=4098), ALIGN)]


@pytest.mark.parametrize("entry", [tree, select, append, fork, compact])
def test_entry_geometry(entry):
    assert entry(None) == NULL
    summaries = dict(codes=4096, scales=4096) if entry is select else {}
    for change, status in GEOMETRY:
        assert entry(pool(**(summaries | change))) == status, change
    assert entry(pool(codes=4096, scales=None)) == ARG
    assert entry(pool(codes=4100, scales=4096)) == ALIGN


def test_entry_arguments():
    assert tree(pool(), q=None) == NULL
    assert tree(pool(lens=None)) == NULL
    assert tree(pool(), q=4100) == ALIGN
    assert tree(pool(), st=(0, 60, 64)) == ALIGN
    assert tree(pool(), kst=(4, 64, 64)) == ALIGN
    assert tree(pool(), n=0) == SHAPE
    assert tree(pool(), n=129) == UNSUPPORTED
    assert tree(pool(), heads=5) == SHAPE
    assert tree(pool(), heads=34) == UNSUPPORTED
    assert tree(pool(layers=2)) == SHAPE
    assert tree(pool(slots=1025)) == UNSUPPORTED
    assert tree(pool(), ws=0) == WORKSPACE
    full = dict(codes=4096, scales=4096)
    assert select(pool()) == NULL  # no summaries
    assert select(pool(**full), q=None) == NULL
    assert select(pool(**full), q=4098) == ALIGN
    assert select(pool(**full), st=(256, 60)) == ALIGN
    assert select(pool(**full), top=0) == SHAPE
    assert select(pool(**full), heads=3) == SHAPE
    assert select(pool(**full), heads=34) == UNSUPPORTED
    assert select(pool(**full), ws=0) == WORKSPACE
    assert append(pool(refs=None)) == NULL
    assert append(pool(), k=None) == NULL
    assert append(pool(), index=None) == NULL
    assert append(pool(), k=4104) == ALIGN
    assert append(pool(), n=0) == SHAPE
    assert append(pool(slots=2049)) == UNSUPPORTED
    assert append(pool(), ws=4) == WORKSPACE
    assert fork(pool(refs=None)) == NULL
    assert fork(pool(), table=4096) == ARG
    assert fork(pool(), table=4096 + 16) == ARG
    assert fork(pool(), refs=4096) == ARG
    assert fork(pool(), ws=4) == WORKSPACE
    assert compact(pool(), table=4096 + 4) == ARG
    assert compact(pool(), refs=4096 + 4) == ARG
    assert compact(pool(), table=None) == NULL
    assert compact(pool(), ws=4) == WORKSPACE


def test_workspace_sizes_of_nothing():
    lib = _lib.load()
    assert lib.iron_tree_attn_workspace_bytes(0, 1, 4, 2, 64) == 0
    assert lib.iron_tree_attn_workspace_bytes(1, 1, 4, 2, 96) == 0
    assert lib.iron_page_select_attn_workspace_bytes(1, 4, 2, 64, 0, 1, 16) == 0
    assert lib.iron_page_append_workspace_bytes(0, 4) == 0
    assert lib.iron_page_fork_workspace_bytes(-1) == 0
    assert lib.iron_page_compact_workspace_bytes(0) == 0
