"""Refusals of the page-state calls (no GPU: every check is on the host)."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import cache as oc
from parallel_tree_spec_b200 import _lib
from parallel_tree_spec_b200 import kernels as K


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


def _extend(**kw):
    a = dict(pool=P, layers=1, pages=8, pl=4, row_bytes=32, refs=P, table=P, stride=4, lens=P, rows_n=2, width=4, rows=P,
             add_each=None, add=1, batch=2, groups=None, G=0, indptr=P, indices=P, size=8, last=P, seq=P, shared=None,
             status=P, ws=P, ws_bytes=1 << 20, stream=None)
    a.update(kw)
    return _lib.lib().pts_cache_extend(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(row_bytes=24), _lib.PTS_ERR_INVALID), (dict(pool=C.c_void_p(8)), _lib.PTS_ERR_INVALID),
    (dict(stride=3), _lib.PTS_ERR_INVALID), (dict(add=-1), _lib.PTS_ERR_INVALID), (dict(batch=0), _lib.PTS_ERR_INVALID),
    (dict(size=7), _lib.PTS_ERR_INVALID), (dict(shared=P), _lib.PTS_ERR_INVALID),
    (dict(ws_bytes=63), _lib.PTS_ERR_CAPACITY), (dict(batch=4097, size=4097 * 4), _lib.PTS_ERR_CAPACITY),
    (dict(pages=(1 << 20) + 1), _lib.PTS_ERR_CAPACITY), (dict(rows_n=(1 << 17) + 1), _lib.PTS_ERR_CAPACITY)])
def test_extend_refusals(kw, code):
    assert _extend(**kw) == code


def test_fork_truncate_and_compact_refusals():
    lib = _lib.lib()
    assert lib.pts_cache_fork(P, P, 4, P, 2, 4, 8, P, P, 1025, P, None) == _lib.PTS_ERR_CAPACITY
    assert lib.pts_cache_fork(P, P, 4, P, 2, 4, 8, P, P, 0, P, None) == _lib.PTS_ERR_INVALID
    assert lib.pts_cache_truncate(P, P, 4, P, 2, 4, 8, 0, P, None, 1, P, None) == _lib.PTS_ERR_INVALID
    other = C.c_void_p(512)
    ok = (P, 1, 8, 4, 32, P, P, 4, 2, 4)
    assert lib.pts_cache_compact(*ok, P, other, other, other, other, 1 << 20, None) == _lib.PTS_ERR_INVALID
    assert lib.pts_cache_compact(*ok, other, other, other, other, other, 8, None) == _lib.PTS_ERR_CAPACITY


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
