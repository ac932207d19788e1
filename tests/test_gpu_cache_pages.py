"""Fork, extend, truncate and compact of device page state against the oracle
(integers and byte copies: every comparison is exact)."""
import numpy as np
import pytest
import torch

from oracle import cache as oc
from parallel_tree_spec_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Pair:
    """The oracle's state and the device's, changed by the same calls."""

    def __init__(self, rows, width, pages, pl, layers=2, heads=2, dim=8, dtype=torch.float32, extra_columns=0, seed=0):
        shape = (layers, pages, 2, pl, heads, dim)
        bits = np.random.default_rng(seed).integers(-2 ** 15, 2 ** 15, size=shape, dtype=np.int16)
        if dtype == torch.float32:
            bits = bits.astype(np.int32)
        self.o = oc.PageState(rows, width, pages, pl, bits.copy())
        self.pool = torch.from_numpy(bits).to(DEV).view(dtype)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        wide = torch.full((rows, width + extra_columns), -1, dtype=torch.int32, device=DEV)
        self.table, self.beyond = wide[:, :width], wide[:, width:]
        self.lens = torch.zeros(rows, dtype=torch.int32, device=DEV)

    def fork(self, src, dst):
        s = K.cache_fork(self.refs, self.table, self.lens, i32(src), i32(dst))
        assert s.item() == self.o.fork(src, dst)

    def extend(self, rows, add, groups=None, scalar=False):
        adds = [add] * len(rows) if isinstance(add, int) else add
        W = self.table.shape[1]
        idx = torch.full((len(rows) * W,), -7, dtype=torch.int32, device=DEV)
        e = lambda n: torch.full((n,), -9, dtype=torch.int32, device=DEV)
        b = K.cache_extend(self.pool, self.refs, self.table, self.lens, i32(rows), add if scalar else i32(adds),
                           group_indptr=i32(groups) if groups else None,
                           out=(e(len(rows) + 1), idx, e(len(rows)), e(len(rows)), e(len(groups) - 1) if groups else None))
        code, lists, lens, shared = self.o.extend(rows, adds, groups)
        assert b.status.item() == code
        flat = sum(lists, [])
        assert b.page_indptr.tolist() == np.cumsum([0] + [len(x) for x in lists]).tolist()
        assert b.page_indices.tolist() == flat + [-7] * (len(rows) * W - len(flat))
        assert b.seq_lens.tolist() == lens
        assert b.last_page_len.tolist() == [(n - 1) % self.o.page_len + 1 if n else 0 for n in lens]
        if groups:
            assert b.shared_pages.tolist() == shared
        return code

    def truncate(self, rows, new=None):
        s = K.cache_truncate(self.refs, self.table, self.lens, self.o.page_len, i32(rows), i32(new) if new else None)
        assert s.item() == self.o.truncate(rows, new)

    def compact(self):
        r = K.cache_compact(self.pool, self.refs, self.table)
        refs, table, to, counts = self.o.compact()
        assert r.page_map.tolist() == to and r.counts.tolist() == counts
        assert r.page_refs.tolist() == refs and r.page_table.tolist() == table
        before = self.refs.tolist(), self.table.tolist()
        assert before == (self.o.refs, self.o.table)          # the inputs keep their values
        self.o.refs, self.o.table = refs, table
        self.refs, self.table = r.page_refs, r.page_table

    def check(self):
        assert self.refs.tolist() == self.o.refs
        assert self.table.tolist() == self.o.table
        assert self.lens.tolist() == self.o.lens
        held = np.bincount([p for row in self.o.table for p in row if p >= 0], minlength=len(self.o.refs))
        assert held.tolist() == self.o.refs
        assert np.array_equal(self.pool.view(torch.int32 if self.pool.dtype == torch.float32 else torch.int16)
                              .cpu().numpy(), self.o.pool)
        assert (self.beyond == -1).all()


def test_extend_from_empty_and_free():
    p = Pair(rows=4, width=6, pages=20, pl=16)
    p.extend([2, 0, 3], [16, 1, 0], groups=[0, 3])
    p.check()
    p.extend([0, 2], 17, scalar=True)
    p.check()
    p.truncate([2, 0, 3])
    p.check()
    assert p.refs.sum().item() == 0


def test_copy_on_write_keeps_the_page_with_its_last_holder():
    """Three holders of a partial page: two listed copy, the unlisted keeps it; then
    all remaining holders listed, the last of them keeps it."""
    p = Pair(rows=5, width=4, pages=30, pl=8, dtype=torch.bfloat16)
    p.extend([0], [13])
    p.fork([0, 0, 0], [1, 2, 3])
    p.check()
    p.extend([1, 2], [1, 5], groups=[0, 2])
    p.check()
    p.extend([3, 0], [2, 2], groups=[0, 1, 2])
    p.check()
    assert p.o.refs[p.o.table[0][1]] == 1


def test_fork_swaps_and_repeats():
    """A beam reorder: rows are sources and destinations at once."""
    p = Pair(rows=4, width=5, pages=40, pl=4)
    p.extend([0, 1, 2, 3], [3, 7, 12, 20])
    p.fork([1, 0, 1, 3], [0, 1, 2, 3])
    p.check()
    p.fork([2, 2, 0, 0], [3, 0, 1, 2])
    p.check()
    p.extend([0, 1, 2, 3], [0, 0, 0, 0], groups=[0, 2, 4])
    p.check()


@pytest.mark.parametrize("call", ["row", "negative row", "count", "twice", "wide", "pages"])
def test_refused_extend_changes_nothing(call):
    p = Pair(rows=3, width=3, pages=6, pl=4)
    p.extend([0, 1], [5, 6])
    p.fork([1], [2])
    rows, add = {"row": ([0, 3], [1, 1]), "negative row": ([-1, 0], [1, 1]), "count": ([0, 1], [1, -1]),
                 "twice": ([1, 0, 1], [1, 1, 1]), "wide": ([0, 1], [1, 7]), "pages": ([0, 1, 2], [7, 6, 6])}[call]
    expect = {"row": 1, "negative row": 1, "count": 1, "twice": 2, "wide": 4, "pages": 8}[call]
    if call == "wide":                                       # the oracle lists the rows as they are
        before = p.refs.tolist(), p.table.tolist(), p.lens.tolist()
    assert p.extend(rows, add) == expect
    p.check()
    if call == "wide":
        assert before == (p.refs.tolist(), p.table.tolist(), p.lens.tolist())


def test_refused_forks_and_skipped_truncations():
    p = Pair(rows=3, width=3, pages=9, pl=4)
    p.extend([0, 1], [9, 6])
    for src, dst in (([0, 5], [1, 2]), ([0, 0], [2, 2]), ([0, 1], [2, -1])):
        p.fork(src, dst)
        p.check()
    p.truncate([7, 0, -2, 0], [1, 6, 1, 2])                   # row 0 twice: the smaller length
    p.check()
    p.truncate([1], [100])                                   # longer than it is: unchanged
    p.check()
    p.truncate([1], [-3])
    p.check()


def test_status_errors():
    for code, err in ((1, IndexError), (2, ValueError), (4, RuntimeError), (8, RuntimeError), (3, IndexError)):
        with pytest.raises(err):
            K.check_cache_status(i32([code]))
    K.check_cache_status(i32([0]))


@pytest.mark.parametrize("pl,pages,dtype,columns", [(16, 97, torch.bfloat16, 0), (1, 333, torch.float32, 3),
                                                    (5, 64, torch.bfloat16, 1), (32, 1025, torch.float32, 0)])
def test_random_calls(pl, pages, dtype, columns):
    rng = np.random.default_rng(pages)
    R = 9
    p = Pair(rows=R, width=max(6, 40 // pl), pages=pages, pl=pl, layers=3, dtype=dtype, extra_columns=columns, seed=1)
    for step in range(40):
        what = rng.integers(0, 5)
        rows = rng.permutation(R)[:int(rng.integers(1, R + 1))].tolist()
        if what == 0:
            p.fork(rng.integers(0, R, size=len(rows)).tolist(), rows)
        elif what in (1, 2):
            cuts = sorted(set([0, len(rows)] + rng.integers(0, len(rows) + 1, size=2).tolist()))
            p.extend(rows, rng.integers(0, 3 * pl, size=len(rows)).tolist(), groups=cuts)
        elif what == 3:
            p.truncate(rows, [int(rng.integers(0, p.o.lens[r] + 2)) for r in rows])
        else:
            p.compact()
        p.check()


def test_large_pool_and_batch():
    """A pool of 70001 pages, 1500 sequences, forks of one sequence into 1000."""
    p = Pair(rows=1500, width=40, pages=70001, pl=4, layers=1, heads=1, dim=4, seed=3)
    rng = np.random.default_rng(5)
    rows = rng.permutation(1500).tolist()
    p.extend(rows, rng.integers(0, 140, size=1500).tolist(), groups=[0, 1500])
    p.check()
    p.fork([rows[3]] * 1000, [r for r in rows if r != rows[3]][:1000])
    p.check()
    p.extend(list(range(1500)), 3, groups=[0, 700, 1500], scalar=True)
    p.check()
    p.truncate(rows[:800], [int(x) for x in rng.integers(0, 100, size=800)])
    p.compact()
    p.check()


def test_empty_pool_and_full_pool():
    p = Pair(rows=2, width=2, pages=3, pl=2)
    p.compact()
    p.check()
    p.extend([0, 1], [2, 4])
    p.compact()
    p.check()
    p.fork([0], [1])
    assert p.extend([0, 1], [3, 1]) == 4
    p.check()


def test_replayed_graph_and_another_stream():
    """fork + extend + truncate captured once and replayed; then two states changed
    on two streams at the same time."""
    a, b = Pair(6, 8, 60, 16, seed=1), Pair(6, 8, 60, 16, seed=2)
    for p in (a, b):
        p.extend([0, 1], [40, 23])
    src, dst, keep = i32([0, 0, 1, 1]), i32([2, 3, 4, 5]), i32([40, 41, 23, 30])
    K.cache_fork(a.refs, a.table, a.lens, src, dst)           # modules are loaded before the capture
    K.cache_extend(a.pool, a.refs, a.table, a.lens, dst, 9)
    K.cache_truncate(a.refs, a.table, a.lens, 16, dst, keep)
    K.cache_compact(a.pool, a.refs, a.table)                 # moves pages; the table returned is dropped
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.cache_fork(a.refs, a.table, a.lens, src, dst)
        K.cache_extend(a.pool, a.refs, a.table, a.lens, dst, 9)
        K.cache_truncate(a.refs, a.table, a.lens, 16, dst, keep)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            g.replay()
        with torch.cuda.stream(s2):
            K.cache_fork(b.refs, b.table, b.lens, src, dst)
            K.cache_extend(b.pool, b.refs, b.table, b.lens, dst, 9)
            K.cache_truncate(b.refs, b.table, b.lens, 16, dst, keep)
    torch.cuda.synchronize()
    for k in range(4):
        a.o.fork([0, 0, 1, 1], [2, 3, 4, 5]), a.o.extend([2, 3, 4, 5], [9] * 4)
        a.o.truncate([2, 3, 4, 5], [40, 41, 23, 30])
        if k == 0:
            a.o.compact()                                    # its page copies; the returned table was not adopted
    a.check()
    for _ in range(3):
        b.o.fork([0, 0, 1, 1], [2, 3, 4, 5]), b.o.extend([2, 3, 4, 5], [9] * 4)
        b.o.truncate([2, 3, 4, 5], [40, 41, 23, 30])
    b.check()


def test_extend_refuses_an_output_without_shared_pages():
    """Groups need a place for their pages; nothing has changed after the refusal."""
    p = Pair(rows=2, width=3, pages=4, pl=4)
    out = (i32([0, 0]), i32([0] * 3), i32([0]), i32([0]), None)
    with pytest.raises(ValueError, match="shared_pages"):
        K.cache_extend(p.pool, p.refs, p.table, p.lens, i32([0]), 1, group_indptr=i32([0, 1]), out=out)
    p.check()
    b = K.cache_extend(p.pool, p.refs, p.table, p.lens, i32([0]), 1, out=out)
    assert b.status.item() == 0 and b.shared_pages is None


def test_failures_are_added_up_in_a_word_of_the_callers():
    """Every call ORs its status into the word; calls that could be done leave it; a word of
    another type, size or device is refused."""
    p = Pair(rows=3, width=3, pages=5, pl=4)                 # 5 and 6 tokens in four pages; 11 and 12 take six
    word = i32([0])
    rows = lambda *r: i32(list(r))
    p.extend([0, 1], [5, 6])
    K.cache_fork(p.refs, p.table, p.lens, rows(0), rows(2), failures=word)
    K.cache_truncate(p.refs, p.table, p.lens, 4, rows(2), failures=word)
    K.cache_extend(p.pool, p.refs, p.table, p.lens, rows(0), 0, failures=word)
    assert word.item() == 0
    expect = 0
    for code, call in ((2, lambda: K.cache_fork(p.refs, p.table, p.lens, rows(0, 1), rows(2, 2), failures=word)),
                       (8, lambda: K.cache_extend(p.pool, p.refs, p.table, p.lens, rows(0, 1), 6, failures=word).status),
                       (4, lambda: K.cache_extend(p.pool, p.refs, p.table, p.lens, rows(0), 99, failures=word).status),
                       (1, lambda: K.cache_truncate(p.refs, p.table, p.lens, 4, rows(7), failures=word)),
                       (0, lambda: K.cache_truncate(p.refs, p.table, p.lens, 4, rows(2), failures=word))):
        assert call().item() == code
        expect |= code
        assert word.item() == expect
    p.check()
    for bad in (i32([0, 0]), torch.zeros(1, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int32)):
        for call in (lambda: K.cache_fork(p.refs, p.table, p.lens, rows(0), rows(2), failures=bad),
                     lambda: K.cache_extend(p.pool, p.refs, p.table, p.lens, rows(0), 1, failures=bad),
                     lambda: K.cache_truncate(p.refs, p.table, p.lens, 4, rows(0), failures=bad)):
            with pytest.raises(ValueError):
                call()
    p.check()


def test_the_largest_tables():
    """2^17 sequences over 2^20 pages, 4096 of them extended and 1024 forked at once."""
    R, W, P = 1 << 17, 2, 1 << 20
    p = Pair(rows=R, width=W, pages=P, pl=1, layers=1, heads=1, dim=4, seed=2)
    rng = np.random.default_rng(6)
    held = rng.permutation(P)[:R].reshape(R // 2, W).tolist()  # half the sequences hold two scattered pages
    for r, pages in enumerate(held):
        p.o.table[2 * r], p.o.lens[2 * r] = list(pages), 2
        for page in pages:
            p.o.refs[page] = 1
    p.table.copy_(torch.tensor(p.o.table, dtype=torch.int32))
    p.refs.copy_(torch.tensor(p.o.refs, dtype=torch.int32))
    p.lens.copy_(torch.tensor(p.o.lens, dtype=torch.int32))
    empty = (2 * rng.permutation(R // 2)[:4096] + 1).tolist()
    p.extend(empty, rng.integers(0, 3, size=4096).tolist(), groups=[0, 1, 4000, 4096])
    p.fork((2 * rng.permutation(R // 2)[:1024]).tolist(), rng.permutation(R)[:1024].tolist())
    p.check()
    p.truncate(rng.permutation(R)[:20000].tolist(), rng.integers(0, 2, size=20000).tolist())
    p.compact()
    p.check()


@pytest.mark.parametrize("call", ["extend", "compact"])
def test_pages_past_4_gb_of_a_layer(call):
    """Copies between pages whose bytes lie past 32 bits, in both layers."""
    L, P, pl, H, D = 2, 70000, 16, 8, 128                      # 4.6 GB a layer
    pool = torch.empty(L, P, 2, pl, H, D, dtype=torch.bfloat16, device=DEV)
    refs, table, lens = i32([0] * P), torch.full((3, 4), -1, dtype=torch.int32, device=DEV), i32([0] * 3)
    src = [P - 3, P - 40000, 12]                               # 41 tokens: two pages and nine slots
    table[0, :3], lens[0], refs[i32(src).long()] = i32(src), 41, 1
    bits = pool.view(torch.int16)
    for page in src:
        bits[:, page] = torch.randint(-2 ** 15, 2 ** 15, (L, 2, pl, H, D), dtype=torch.int16, device=DEV)
    if call == "extend":
        last = P - 7
        table[0, 2], refs[12], refs[last] = last, 0, 1
        bits[:, last] = bits[:, 12]
        others = refs == 0                                     # all other pages but one high one belong to someone
        others[P - 1] = False
        refs[others] = 1
        K.cache_fork(refs, table, lens, i32([0]), i32([1]))
        b = K.cache_extend(pool, refs, table, lens, i32([1]), 1)
        assert b.status.item() == 0 and table[1].tolist() == [src[0], src[1], P - 1, -1]
        assert torch.equal(bits[:, P - 1, :, :9], bits[:, last, :, :9])
    else:
        want = [bits[:, page].clone() for page in src]
        r = K.cache_compact(pool, refs, table)
        assert r.counts.tolist() == [3, 3] and sorted(r.page_table[0, :3].tolist()) == [0, 1, 2]
        for page, x in zip(r.page_table[0, :3].tolist(), want):
            assert torch.equal(bits[:, page], x)
