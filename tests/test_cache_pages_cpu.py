"""Refusals of the page-state calls (no GPU: every check is on the host)."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

from oracle import cache as oc
from parallel_tree_spec_b200 import _lib
from parallel_tree_spec_b200 import kernels as K

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "pts_b200.h")


def test_cpu_tensors_are_refused():
    refs, table, lens = torch.zeros(4, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    rows = torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(1, 4, 2, 4, 1, 8)
    for call in (lambda: K.cache_fork(refs, table, lens, rows, rows),
                 lambda: K.cache_extend(pool, refs, table, lens, rows, 1),
                 lambda: K.cache_truncate(refs, table, lens, 4, rows), lambda: K.cache_compact(pool, refs, table)):
        with pytest.raises(ValueError):
            call()


P = C.c_void_p(256)                                          # never read: the checks come first


def _extend(ws_bytes=1 << 20, **kw):
    a = dict.fromkeys((n for n, _ in _lib.CACHE_EXTEND_FIELDS), 256)
    a.update(row_bytes=32, table_stride=4, add_each=0, group_indptr=0, shared_pages=0, page_indices_size=8, num_layers=1,
             max_pages=8, page_len=4, num_rows=2, table_width=4, add=1, batch=2, num_groups=0)
    a.update(kw)
    return _lib.lib().pts_cache_extend(_lib.pack_cache_extend(*a.values()), P, ws_bytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(row_bytes=24), _lib.PTS_ERR_INVALID), (dict(kv_pool=8), _lib.PTS_ERR_INVALID),
    (dict(table_stride=3), _lib.PTS_ERR_INVALID), (dict(add=-1), _lib.PTS_ERR_INVALID),
    (dict(batch=0), _lib.PTS_ERR_INVALID), (dict(page_indices_size=7), _lib.PTS_ERR_INVALID),
    (dict(shared_pages=256), _lib.PTS_ERR_INVALID), (dict(page_refs=0), _lib.PTS_ERR_INVALID),
    (dict(ws_bytes=63), _lib.PTS_ERR_CAPACITY), (dict(batch=4097, page_indices_size=4097 * 4), _lib.PTS_ERR_CAPACITY),
    (dict(max_pages=(1 << 20) + 1), _lib.PTS_ERR_CAPACITY), (dict(num_rows=(1 << 17) + 1), _lib.PTS_ERR_CAPACITY)])
def test_extend_refusals(kw, code):
    assert _extend(**kw) == code


def test_fork_truncate_and_compact_refusals():
    lib = _lib.lib()
    assert lib.pts_cache_fork(P, P, 4, P, 2, 4, 8, P, P, 1025, P, None) == _lib.PTS_ERR_CAPACITY
    assert lib.pts_cache_fork(P, P, 4, P, 2, 4, 8, P, P, 0, P, None) == _lib.PTS_ERR_INVALID
    assert lib.pts_cache_truncate(P, P, 4, P, 2, 4, 8, 0, P, None, 1, P, None) == _lib.PTS_ERR_INVALID
    def compact(out_refs, ws_bytes=1 << 20, out_table=512):
        return lib.pts_cache_compact(_lib.pack_cache_compact(256, 32, 256, 256, 4, out_refs, out_table, 512, 512, 1, 8, 4, 2,
                                                             4), P, ws_bytes, None)

    assert compact(256) == _lib.PTS_ERR_INVALID              # the output is the input
    assert compact(512, out_table=256) == _lib.PTS_ERR_INVALID
    assert compact(512, ws_bytes=8) == _lib.PTS_ERR_CAPACITY


def _attend(ws_bytes=256, **kw):
    a = dict.fromkeys((n for n, _ in _lib.SHARED_ATTN_FIELDS), 256)
    a.update(error=0, mask_words=1, num_groups=1, batch=2, total_q=2, max_qo_len=1, max_kv_len=40, max_own_len=0,
             num_qo_heads=4, num_kv_heads=2, head_dim=96, page_len=16, max_pages=8, elem_bytes=4, sm_scale=0.1)
    a.update(kw)
    return _lib.lib().pts_tree_attn_run_shared(_lib.pack_shared_attn(*a.values()), P, ws_bytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=0), _lib.PTS_ERR_INVALID), (dict(q=264), _lib.PTS_ERR_INVALID), (dict(shared_pages=0), _lib.PTS_ERR_INVALID),
    (dict(num_groups=0), _lib.PTS_ERR_INVALID), (dict(num_qo_heads=5), _lib.PTS_ERR_INVALID),
    (dict(max_qo_len=65), _lib.PTS_ERR_INVALID), (dict(max_qo_len=1025, mask_words=17), _lib.PTS_ERR_CAPACITY),
    (dict(head_dim=48), _lib.PTS_ERR_UNSUPPORTED), (dict(head_dim=288), _lib.PTS_ERR_UNSUPPORTED),
    (dict(elem_bytes=1), _lib.PTS_ERR_UNSUPPORTED), (dict(), _lib.PTS_ERR_CAPACITY)])
def test_attention_refusals(kw, code):
    assert _attend(**kw) == code


@pytest.mark.parametrize("name,fields", [("pts_cache_extend_args", _lib.CACHE_EXTEND_FIELDS),
                                         ("pts_cache_compact_args", _lib.CACHE_COMPACT_FIELDS),
                                         ("pts_shared_attn_args", _lib.SHARED_ATTN_FIELDS)])
def test_argument_structures_match_the_header(name, fields):
    """Names, order and types of the packed fields are the header's, and their offsets C's."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
    want = []
    for decl in body.split(";"):
        if not decl.strip():
            continue
        kind, names = re.match(r"\s*((?:const )?\w+\s*\*?)\s*(.*)", decl.strip(), flags=re.S).groups()
        code = "P" if "*" in kind else {"int64_t": "q", "int": "i", "float": "f"}[kind.strip()]
        want += [(n.strip(), code) for n in names.split(",")]
    assert want == list(fields)
    types = {"P": C.c_void_p, "q": C.c_int64, "i": C.c_int, "f": C.c_float}
    S = type(name, (C.Structure,), {"_fields_": [(n, types[c]) for n, c in fields]})
    values = [3 * i + 1 for i in range(len(fields))]
    packed = _lib._packer(fields).pack(*values)
    assert len(packed) == C.sizeof(S)
    s = S.from_buffer_copy(packed)
    assert [getattr(s, n) for n, _ in fields] == values


def test_oracle_counts_holders():
    """The oracle's invariant: a page's count is the number of entries that hold it."""
    rng = np.random.default_rng(0)
    s = oc.PageState(6, 8, 70, 4, np.zeros((1, 70, 2, 4, 1, 1), np.int32))
    for _ in range(200):
        rows = rng.permutation(6)[:3].tolist()
        k = rng.integers(0, 3)
        if k == 0:
            s.fork(rng.integers(0, 6, size=3).tolist(), rows)
        elif k == 1:
            s.extend(rows, rng.integers(0, 9, size=3).tolist())
        else:
            s.truncate(rows, rng.integers(0, 30, size=3).tolist())
        held = np.bincount([p for row in s.table for p in row if p >= 0], minlength=70)
        assert held.tolist() == s.refs
        assert all(len([p for p in row if p >= 0]) == oc.pages_of(n, 4) for row, n in zip(s.table, s.lens))


@pytest.mark.parametrize("rows,batch,Hq,Hkv,D,page,dtype,pays", [
    (1, 64, 32, 8, 128, 16, torch.bfloat16, True), (65, 16, 32, 8, 128, 16, torch.bfloat16, False),
    (49, 16, 32, 8, 128, 16, torch.bfloat16, True), (50, 16, 32, 8, 128, 16, torch.bfloat16, False),
    (33, 16, 32, 8, 128, 16, torch.bfloat16, True), (65, 13, 32, 8, 128, 16, torch.bfloat16, True),
    (65, 14, 32, 8, 128, 16, torch.bfloat16, False), (67, 14, 32, 8, 128, 16, torch.bfloat16, True),
    (65, 16, 32, 8, 64, 16, torch.bfloat16, True), (65, 16, 32, 8, 128, 32, torch.bfloat16, True),
    (65, 16, 32, 8, 128, 16, torch.float32, True), (65, 64, 64, 2, 128, 16, torch.bfloat16, True)])
def test_sharing_pays(rows, batch, Hq, Hkv, D, page, dtype, pays):
    assert K.sharing_pays(rows, batch, Hq, Hkv, D, page, dtype) is pays


def test_small_calls_need_no_workspace():
    size = _lib.lib().pts_tree_attn_shared_workspace_size
    assert size(6, 1, 6, 1, 600, 0, 32, 8, 64, 16, 2) == 0
    assert size(64, 1, 64, 1, 9000, 300, 32, 8, 128, 16, 2) > 0
    assert size(6, 1, 6, 1, 600, 0, 32, 8, 64, 16, 4) > 0      # fp32
    assert size(0, 1, 6, 1, 600, 0, 32, 8, 64, 16, 2) == 0     # refused by the call


@pytest.mark.parametrize("dtype_bytes,head_dim,page", [(4, 64, 16), (2, 96, 16), (2, 128, 8), (2, 128, 16), (2, 64, 16)])
def test_the_largest_length_bounds_keep_the_columns_cut(dtype_bytes, head_dim, page):
    """A bound of 2^31 - 1 tokens (no bound known) cuts the columns as finely as a bound of
    a million does: the workspace, which holds a part per cut, is as large."""
    size = _lib.lib().pts_tree_attn_shared_workspace_size
    for rows in (1, 20, 65):                                  # single tokens, trees, trees with a tail tile
        at = lambda max_kv, own=0, n=rows: size(2, 1, 2 * rows, n, max_kv, own, 8, 2, head_dim, page, dtype_bytes)
        most = 2 ** 31 - 1
        assert at(1 << 20) > 0
        assert at(most) == at(1 << 20) == at(most - 40)
        assert at(most, most) == at(1 << 20, 1 << 20)
        assert at(1 << 20, 0, most) == at(1 << 20, 0, 2 * rows)   # no request has more rows than there are
