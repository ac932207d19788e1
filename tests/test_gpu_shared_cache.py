"""Sequences that share pages, as they are used: ``SharedKvCache`` with the wrapper's
append and attention over several steps (forks, copies on write, truncations, a
compaction, graph replays) against dense attention over each sequence's own history;
beam search with ``shared_prefix``; and a wait of the attention that runs out."""
import math

import numpy as np
import pytest
import torch

from parallel_tree_spec_b200 import beam_search as pbs
from parallel_tree_spec_b200 import kernels as K
from parallel_tree_spec_b200.attention_wrapper import AttentionRotaryParams, BeFlashinferWrapper
from parallel_tree_spec_b200.cache_manager import KvCachePool, RequestKvCache, SharedKvCache
from tests.test_gpu_attention_shared import Case, chain, tree

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class History:
    """Every sequence's keys and values as they should be, [tokens, 2, Hkv, D] a layer."""

    def __init__(self, layers):
        self.kv = {}
        self.layers = layers

    def append(self, row, k, v):
        new = torch.stack([k, v], dim=2)                      # [layers, n, 2, Hkv, D]
        old = self.kv.get(row)
        self.kv[row] = new if old is None else torch.cat([old, new], dim=1)


def dense(q, kv, mask):
    """fp64 attention of q [n, Hq, D] over kv [L, 2, Hkv, D]; (o, sum p |v|)."""
    g = q.shape[1] // kv.shape[2]
    k, v = kv[:, 0].double().repeat_interleave(g, 1), kv[:, 1].double().repeat_interleave(g, 1)
    s = torch.einsum("nhd,lhd->nhl", q.double(), k) / math.sqrt(q.shape[2])
    p = torch.softmax(s.masked_fill(~mask[:, None], float("-inf")), -1)
    return torch.einsum("nhl,lhd->nhd", p, v), torch.einsum("nhl,lhd->nhd", p, v.abs())


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page", [(torch.bfloat16, 8, 2, 128, 16), (torch.bfloat16, 4, 4, 64, 32),
                                                 (torch.float32, 4, 2, 64, 16), (torch.bfloat16, 2, 1, 64, 8)])
def test_steps_of_shared_sequences(dtype, Hq, Hkv, D, page):
    """A prompt, samples forked from it, single tokens and draft trees of which some
    tokens are kept, a second generation of forks, a released sequence, a compaction.
    Attention tolerance: probabilities and output rounded to the type (2 h with h its
    half step, times sum p |v|), scores in fp32 (2^-12 covers (D + 3) 2^-24 |q||k| / sqrt D
    at |q||k| below 300, twice)."""
    layers, gen = 2, torch.Generator().manual_seed(D + page)
    pool = KvCachePool(120, layers, Hkv, D, page, dtype, torch.device(DEV))
    cache = SharedKvCache(pool, 8, 20)
    assert pool.num_free_pages() == 0
    w = BeFlashinferWrapper(Hq, Hkv, Hq * D, page, torch.device(DEV))
    h = History(layers)
    half = torch.finfo(dtype).eps / 2
    rnd = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(DEV)

    def step(rows, parents, groups=None):
        """Extend the rows by their trees (parents per row), append, attend in every layer."""
        bp = cache.extend(rows, [len(p) for p in parents], groups)
        flat = torch.tensor(sum(parents, []), dtype=torch.int32, device=DEV)
        w.set_tree_masks(flat, bp, max(len(p) for p in parents))
        T = flat.numel()
        q, k, v = rnd(layers, T, Hq, D), rnd(layers, T, Hkv, D), rnd(layers, T, Hkv, D)
        outs = [w.computeAttention(q[i], k[i], v[i], pool.cache_data[i], "tree", bp, AttentionRotaryParams(),
                                   i).view(T, Hq, D) for i in range(layers)]
        t0 = 0
        for row, par in zip(rows, parents):
            n = len(par)
            h.append(row, k[:, t0:t0 + n], v[:, t0:t0 + n])
            L = h.kv[row].shape[1]
            mask = torch.ones(n, L, dtype=torch.bool)
            mask[:, L - n:] = False
            for i in range(n):
                j = i
                while j >= 0:
                    mask[i, L - n + j] = True
                    j = par[j]
            for i in range(layers):
                o, A = dense(q[i, t0:t0 + n], h.kv[row][i], mask.to(DEV))
                bad = (outs[i][t0:t0 + n].double() - o).abs() / ((2 * half + 2.0 ** -12) * A + half * o.abs())
                assert bad.max().item() <= 1.0, (row, bad.max().item())
            t0 += n
        return bp

    def keep(rows, lens):
        cache.truncate(rows, lens)
        for r, n in zip(rows, lens):
            h.kv[r] = h.kv[r][:, :n]

    def fork(src, dst):
        cache.fork(src, dst)
        old = {a: h.kv[a] for a in src}
        for a, b in zip(src, dst):
            h.kv[b] = old[a]

    step([0], [chain(3 * page + 5)])                          # the prompt
    fork([0] * 4, [1, 2, 3, 4])
    bp = step([1, 2, 3, 4], [chain(1)] * 4)
    assert bp.shared_pages.tolist() == [3]
    step([0, 1, 2, 3, 4], [tree(1, 3, 3), tree(2, 2, 2), chain(1), tree(3, 4, 2), chain(2)], groups=[0, 1, 5])
    lens = cache.lengths()
    keep([0, 1, 3], [lens[0] - 6, lens[1] - 2, lens[3] - 8])
    step([4, 3, 2, 1, 0], [chain(1)] * 5)
    fork([1, 1, 3], [5, 6, 1])                                # row 1 is a source and a destination
    step([1, 3, 5, 6], [tree(4, 2, 3), tree(5, 2, 3), chain(1), chain(1)], groups=[0, 2, 4])
    cache.release([2])
    h.kv.pop(2)
    before = int((cache.page_refs > 0).sum())
    cache.compact()
    assert (cache.page_refs[:before] > 0).all() and (cache.page_refs[before:] == 0).all()
    step([0, 1, 3, 4, 5, 6], [chain(2)] * 6, groups=[0, 1, 3, 6])
    cache.check()
    held = np.bincount([p for r in cache.page_table.tolist() for p in r if p >= 0], minlength=120)
    assert held.tolist() == cache.page_refs.tolist()
    cache.close()
    assert pool.num_free_pages() == 120


def test_failed_calls_are_reported_and_change_nothing():
    pool = KvCachePool(6, 1, 1, 32, 4, torch.float32, torch.device(DEV))
    cache = SharedKvCache(pool, 3, 4)
    with pytest.raises(ValueError):
        SharedKvCache(pool, 1, 1)                             # no free pages
    cache.extend([0, 1], 10)
    cache.check()
    state = cache.page_refs.tolist(), cache.page_table.tolist(), cache.kv_lens.tolist()
    for call, error in ((lambda: cache.extend([0, 1], 4), RuntimeError), (lambda: cache.extend([0, 0], 1), ValueError),
                        (lambda: cache.extend([7], 1), IndexError), (lambda: cache.extend([0], 30), RuntimeError),
                        (lambda: cache.fork([0, 1], [2, 2]), ValueError)):
        call()
        with pytest.raises(error):
            cache.check()
        assert state == (cache.page_refs.tolist(), cache.page_table.tolist(), cache.kv_lens.tolist())
    cache.check()


def test_captured_step():
    """fork, extend, append and attention captured once: each replay forks the prompt
    anew, as it then is."""
    Hq, Hkv, D, page = 8, 2, 128, 16
    pool = KvCachePool(64, 1, Hkv, D, page, torch.bfloat16, torch.device(DEV))
    cache = SharedKvCache(pool, 5, 8)
    w = BeFlashinferWrapper(Hq, Hkv, Hq * D, page, torch.device(DEV))
    gen = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    hist = torch.empty(0, 2, Hkv, D, dtype=torch.bfloat16, device=DEV)

    def prompt(n):
        nonlocal hist
        bp = cache.extend([0], n)
        k, v = rnd(n, Hkv, D), rnd(n, Hkv, D)
        w.append_kv_cache(None, k, v, bp, pool.cache_data[0], page)
        hist = torch.cat([hist, torch.stack([k, v], 1)])

    src, dst, groups = i32([0] * 4), i32([1, 2, 3, 4]), i32([0, 4])
    seq, bits = i32([0, 1, 2, 3, 4]), torch.ones(4, 1, dtype=torch.int64, device=DEV)
    q, k, v = rnd(4, Hq, D), rnd(4, Hkv, D), rnd(4, Hkv, D)
    out = torch.empty_like(q)

    def body():
        K.cache_fork(cache.page_refs, cache.page_table, cache.kv_lens, src, dst)
        b = K.cache_extend(pool.cache_data, cache.page_refs, cache.page_table, cache.kv_lens, dst, 1, group_indptr=groups)
        bi, pos = K.batch_positions(seq, b.seq_lens, 4)
        K.kv_append(k, v, pool.cache_data[0], bi, pos, b.page_indptr, b.page_indices)
        K.tree_attention_shared(q, pool.cache_data[0], seq, b.page_indptr, b.page_indices, b.last_page_len, bits, 1,
                                8 * page, groups, b.shared_pages, out=out)

    prompt(20)
    body()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        body()
    for n in (0, 9, 33, 16):
        if n:
            prompt(n)
        q.copy_(rnd(4, Hq, D))
        k.copy_(rnd(4, Hkv, D))
        v.copy_(rnd(4, Hkv, D))
        g.replay()
        for i in range(4):
            kv = torch.cat([hist, torch.stack([k[i:i + 1], v[i:i + 1]], 1)])
            o, A = dense(q[i:i + 1], kv, torch.ones(1, kv.shape[0], dtype=torch.bool, device=DEV))
            bad = (out[i:i + 1].double() - o).abs() / ((2 ** -7 + 2.0 ** -12) * A + 2 ** -8 * o.abs())
            assert bad.max().item() <= 1.0
    cache.check()


@pytest.mark.parametrize("graph", [False, True])
def test_beam_search_with_a_shared_prefix(graph):
    """The same search with and without ``shared_prefix`` on the fp32 model finds the same
    tree (its scores differ in the last bits only), leaves the same free pages, and
    goes through the shared attention."""
    from tests.test_gpu_reference_flow import D, HKV, PAGE, V, _patched_model
    model = _patched_model()
    ids = torch.randint(0, V, (1, 75), generator=torch.Generator().manual_seed(3)).to(DEV)
    trees, free = [], []
    real, calls = K.tree_attention_shared, []
    for shared in (False, True):
        pool = KvCachePool(64, 2, HKV, D, PAGE, torch.float32, torch.device(DEV))
        req = RequestKvCache(pool, PAGE, 0)
        w = BeFlashinferWrapper(4, HKV, 256, PAGE, torch.device(DEV))
        cfg = pbs.BeamSearchConfig(topk_len=5, max_depth=6, use_cuda_graph=graph, shared_prefix=shared)
        K.tree_attention_shared = lambda *a, **kw: (calls.append(shared), real(*a, **kw))[1]
        try:
            tree_, _, runner = pbs.beam_search(model, req, ids, cfg, w)
            if graph:                                        # replays of the captured step, another prompt's length
                req2 = RequestKvCache(pool, PAGE, 0)
                tree_, _, _ = pbs.beam_search(model, req2, ids[:, :50], cfg, w, cuda_graph_runner=runner)
        finally:
            K.tree_attention_shared = real
        trees.append([(n.parent, n.token_id, n.depth) for n in tree_.nodes])
        free.append(pool.free_page_mask.tolist())
    assert trees[0] == trees[1] and len(trees[0]) > 20
    assert free[0] == free[1]
    assert calls and all(calls)


@pytest.mark.parametrize("groups", [[(40, [(30, chain(1))] * 40)], [(100, [(30, tree(1, 8, 8))] * 4)]])
def test_a_wait_that_runs_out_is_reported(groups):
    """With a wait limit of a few clocks the launches give up, report it and return; the
    next call is right again.  (The one launch of small decoding calls waits only for its
    own copies, which may land within any limit.)"""
    c = Case(groups, Hq=32, Hkv=8, seed=2)
    a = c.device()
    want = K.tree_attention_shared(**a)
    K.check_attention(torch.device(DEV))
    before = K.set_wait_limit(1)
    try:
        with pytest.raises(RuntimeError, match="gave up waiting"):
            K.tree_attention_shared(**a)
            K.check_attention(torch.device(DEV))
    finally:
        K.set_wait_limit(before)
    assert torch.equal(K.tree_attention_shared(**a), want)
    K.check_attention(torch.device(DEV))


def test_full_tree_tiles_go_to_the_call_that_reads_per_request():
    """Fourteen requests with trees that fill tree_attention's units: the wrapper takes
    that call, and the shared one after single tokens; both answers are the same up to the
    rounding of the probabilities and of the output."""
    page, Hq, Hkv, D, B = 16, 32, 8, 128, 14
    pool = KvCachePool(160, 1, Hkv, D, page, torch.bfloat16, torch.device(DEV))
    cache = SharedKvCache(pool, B, 16)
    w = BeFlashinferWrapper(Hq, Hkv, Hq * D, page, torch.device(DEV))
    gen = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(DEV)
    calls, real = [], (K.tree_attention, K.tree_attention_shared)

    def step(rows, parents):
        bp = cache.extend(rows, [len(p) for p in parents])
        w.set_tree_masks(torch.tensor(sum(parents, []), dtype=torch.int32, device=DEV), bp, max(map(len, parents)))
        T = sum(map(len, parents))
        q = rnd(T, Hq, D)
        K.tree_attention = lambda *a, **kw: (calls.append("tree"), real[0](*a, **kw))[1]
        K.tree_attention_shared = lambda *a, **kw: (calls.append("shared"), real[1](*a, **kw))[1]
        try:
            out = w.computeAttention(q, rnd(T, Hkv, D), rnd(T, Hkv, D), pool.cache_data[0], "tree", bp,
                                     AttentionRotaryParams(), 0)
        finally:
            K.tree_attention, K.tree_attention_shared = real
        args = (q, pool.cache_data[0], bp.seq_indptr, bp.kv_page_indptr, bp.kv_page_indices, bp.kv_last_page_len,
                w._plan["bits"], w._plan["max_qo"], w._plan["max_kv"])
        a = real[0](*args).double()
        b = real[1](*args, bp.group_indptr, bp.shared_pages).double()
        # sum p |v| is at most the largest |v|: two roundings to 2^-8 of each, and the output's
        most = pool.cache_data[0][:, 1].abs().max().item()
        assert (a - b).abs().max().item() <= 2 * (2 * 2.0 ** -8 + 2.0 ** -12) * most
        assert torch.equal(out.view(T, Hq, D).double(), a if calls[-1] == "tree" else b)

    step([0], [chain(70)])
    cache.fork([0] * (B - 1), list(range(1, B)))
    step(list(range(B)), [tree(i, 8, 8) for i in range(B)])
    cache.truncate(list(range(B)), [72] * B)
    step(list(range(B)), [chain(1)] * B)
    cache.check()
    assert calls == ["shared", "tree", "shared"]


def test_a_failed_extend_leaves_the_cache_to_later_calls_of_the_step():
    """The step goes on before its status is read: the append to the failed batch must not
    write over the sequences' last tokens, whose pages others hold."""
    page, Hkv, D = 4, 2, 64
    pool = KvCachePool(5, 1, Hkv, D, page, torch.bfloat16, torch.device(DEV))
    cache = SharedKvCache(pool, 3, 6)
    w = BeFlashinferWrapper(4, Hkv, 4 * D, page, torch.device(DEV))
    ones = lambda n, h: torch.ones(n, h, D, dtype=torch.bfloat16, device=DEV)

    def step(rows, n):
        bp = cache.extend(rows, n)
        w.set_tree_masks(torch.tensor(chain(n) * len(rows), dtype=torch.int32, device=DEV), bp, n)
        T = n * len(rows)
        return bp, w.computeAttention(ones(T, 4), ones(T, Hkv), 2 * ones(T, Hkv), pool.cache_data[0], "tree", bp,
                                      AttentionRotaryParams(), 0)

    pool.cache_data.zero_()
    bp, out = step([0], 14)
    assert bp.kv_page_indptr.tolist() == [0, 4] and (out == 2).all()
    cache.fork([0, 0], [1, 2])
    before = pool.cache_data.clone()
    bp, out = step([1, 2], 3)                                 # two copies and two pages: only one is free
    assert torch.equal(pool.cache_data, before)
    assert bp.kv_page_indptr.tolist() == [0, 0, 0] and bp.shared_pages.tolist() == [0] and (out == 0).all()
    with pytest.raises(RuntimeError):
        cache.check()
    assert cache.kv_lens.tolist() == [14, 14, 14]


def test_a_step_of_the_cache_is_captured():
    """The class's own calls with tensors, and the wrapper's: fork, extend, attention and
    truncation captured once, each replay on the prompt as it then is."""
    Hq, Hkv, D, page, n = 8, 2, 64, 16, 3
    pool = KvCachePool(40, 1, Hkv, D, page, torch.bfloat16, torch.device(DEV))
    cache = SharedKvCache(pool, 4, 8)
    w = BeFlashinferWrapper(Hq, Hkv, Hq * D, page, torch.device(DEV))
    gen = torch.Generator().manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    hist = torch.empty(0, 2, Hkv, D, dtype=torch.bfloat16, device=DEV)

    def prompt(m):
        nonlocal hist
        bp = cache.extend([0], m)
        k, v = rnd(m, Hkv, D), rnd(m, Hkv, D)
        w.append_kv_cache(None, k, v, bp, pool.cache_data[0], page)
        hist = torch.cat([hist, torch.stack([k, v], 1)])

    src, dst, none, parents = i32([0] * 3), i32([1, 2, 3]), i32([0] * 3), i32(chain(n) * 3)
    q, k, v = rnd(3 * n, Hq, D), rnd(3 * n, Hkv, D), rnd(3 * n, Hkv, D)
    out = torch.empty(3 * n, Hq * D, dtype=torch.bfloat16, device=DEV)

    def body():
        cache.fork(src, dst)
        bp = cache.extend(dst, n)
        w.set_tree_masks(parents, bp, n)
        out.copy_(w.computeAttention(q, k, v, pool.cache_data[0], "tree", bp, AttentionRotaryParams(), 0))
        cache.truncate(dst, none)

    prompt(21)
    body()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        body()
    for m in (0, 30, 1):
        if m:
            prompt(m)
        for x in (q, k, v):
            x.copy_(rnd(*x.shape))
        g.replay()
        for i in range(3):
            kv = torch.cat([hist, torch.stack([k[i * n:(i + 1) * n], v[i * n:(i + 1) * n]], 1)])
            mask = torch.ones(n, kv.shape[0], dtype=torch.bool, device=DEV).tril(kv.shape[0] - n)
            o, A = dense(q[i * n:(i + 1) * n], kv, mask)
            bad = (out.view(-1, Hq, D)[i * n:(i + 1) * n].double() - o).abs() / ((2 ** -7 + 2.0 ** -12) * A + 2 ** -8 * o.abs())
            assert bad.max().item() <= 1.0
        assert cache.kv_lens.tolist()[1:] == [0, 0, 0]
    cache.check()


def test_extend_by_nothing_lists_the_pages():
    pool = KvCachePool(8, 1, 1, 64, 4, torch.bfloat16, torch.device(DEV))
    cache = SharedKvCache(pool, 2, 4)
    cache.extend([0], 6)
    cache.fork([0], [1])
    bp = cache.extend([0, 1], 0)
    assert bp.kv_page_indices[:4].tolist() == [0, 1, 0, 1] and bp.shared_pages.tolist() == [1]
    assert bp.batch_indices.numel() == bp.positions.numel() == 0 and bp.seq_indptr.tolist() == [0, 0, 0]
    for bad in (-1, [1, -1], [1], []):
        with pytest.raises(ValueError):
            cache.extend([0, 1], bad)
    with pytest.raises(ValueError):
        cache.extend([], 1)
    cache.check()
    assert cache.lengths() == [6, 6]


def _full_cache():
    """Two sequences of ten tokens that hold all six pages of the pool."""
    pool = KvCachePool(6, 1, 1, 32, 4, torch.float32, torch.device(DEV))
    cache = SharedKvCache(pool, 3, 4)
    cache.extend([0, 1], 10)
    cache.check()
    return cache


def test_a_failure_is_reported_however_many_calls_follow():
    """300 steps without a check after one that could not be done: the check raises for
    it, the next one does not."""
    cache = _full_cache()
    cache.extend([0, 1], 4)
    for _ in range(300):
        cache.fork([0], [0])
    with pytest.raises(RuntimeError, match="free pages"):
        cache.check()
    cache.check()
    cache.fork([0, 9, 1], [2, 2, 2])                          # two faults in one call
    cache.truncate([5])
    with pytest.raises(IndexError, match="listed twice"):
        cache.check()
    cache.check()


def test_a_failed_replay_is_reported():
    """Captured calls report in every replay, also after a check; those that could be done
    report nothing."""
    cache = _full_cache()
    cache.release([1])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    rows, src, dst, gone = i32([0]), i32([0]), i32([2]), i32([2])

    def body():
        cache.fork(src, dst)
        cache.extend(rows, 3)
        cache.truncate(gone)

    body()                                                    # 13 tokens in four pages
    cache.check()
    cache.truncate([0], [5])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        body()
    cache.check()                                             # nothing has run
    for n, fails in ((8, False), (11, False), (14, False), (14, True), (14, True)):
        g.replay()
        if fails:                                             # 17 tokens in a table of 16
            with pytest.raises(RuntimeError, match="wide"):
                cache.check()
        cache.check()
        assert cache.kv_lens.tolist() == [n, 0, 0]
    g.replay()                                                # one more failure, then replays that could be done
    for _ in range(300):
        cache.truncate([0], [2])
        g.replay()
    with pytest.raises(RuntimeError, match="wide"):
        cache.check()
    assert cache.kv_lens.tolist() == [5, 0, 0]
    cache.check()


@pytest.mark.parametrize("captured_compaction", [False, True])
def test_a_captured_step_goes_on_after_a_compaction(captured_compaction):
    """A step captured once, the pool compacted between its replays (as a call or as a
    graph of its own): each replay reads and grows the sequences where they now are."""
    Hq, Hkv, D, page, n = 8, 2, 64, 16, 3
    pool = KvCachePool(30, 1, Hkv, D, page, torch.bfloat16, torch.device(DEV))
    cache = SharedKvCache(pool, 4, 8)
    w = BeFlashinferWrapper(Hq, Hkv, Hq * D, page, torch.device(DEV))
    gen = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    rows, parents = i32([0, 1]), i32(chain(n) * 2)
    q, k, v = rnd(2 * n, Hq, D), rnd(2 * n, Hkv, D), rnd(2 * n, Hkv, D)
    out = torch.empty(2 * n, Hq * D, dtype=torch.bfloat16, device=DEV)
    hist = [torch.empty(0, 2, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(4)]

    def grow(row, m):
        bp = cache.extend([row], m)
        a, b = rnd(m, Hkv, D), rnd(m, Hkv, D)
        w.append_kv_cache(None, a, b, bp, pool.cache_data[0], page)
        hist[row] = torch.cat([hist[row], torch.stack([a, b], 1)])

    def step():
        bp = cache.extend(rows, n)
        w.set_tree_masks(parents, bp, n)
        out.copy_(w.computeAttention(q, k, v, pool.cache_data[0], "tree", bp, AttentionRotaryParams(), 0))

    def noted():
        for i in range(2):
            hist[i] = torch.cat([hist[i], torch.stack([k[i * n:(i + 1) * n], v[i * n:(i + 1) * n]], 1)])

    grow(2, 50)                                               # low pages, released below
    grow(0, 21)
    cache.fork([0], [1])
    hist[1] = hist[0]
    step()
    noted()
    cache.compact()                                           # (modules loaded before the captures)
    torch.cuda.synchronize()
    g, gc = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    if captured_compaction:
        with torch.cuda.graph(gc):
            cache.compact()
    table = cache.page_table.tolist()
    for gap in (2, None, 3):
        if gap:
            cache.release([gap])
            gc.replay() if captured_compaction else cache.compact()
            assert cache.page_table.tolist()[:2] != table[:2]     # pages moved
            live = int((cache.page_refs > 0).sum())
            assert (cache.page_refs[:live] > 0).all()
        for x in (q, k, v):
            x.copy_(rnd(*x.shape))
        g.replay()
        noted()
        for i in range(2):
            L = hist[i].shape[0]
            o, A = dense(q[i * n:(i + 1) * n], hist[i], torch.ones(n, L, dtype=torch.bool, device=DEV).tril(L - n))
            bad = (out.view(-1, Hq, D)[i * n:(i + 1) * n].double() - o).abs() / ((2 ** -7 + 2.0 ** -12) * A + 2 ** -8 * o.abs())
            assert bad.max().item() <= 1.0
        assert cache.kv_lens.tolist()[:2] == [h.shape[0] for h in hist[:2]]
        held = np.bincount([p for r in cache.page_table.tolist() for p in r if p >= 0], minlength=30)
        assert held.tolist() == cache.page_refs.tolist()
        if gap == 2:
            grow(3, 40)
            for row, m in ((0, 20), (1, 9)):                  # pages behind row 3's
                grow(row, m)
        table = cache.page_table.tolist()
    cache.check()


def test_a_failed_extend_of_full_trees_gives_zeros():
    """Trees that the wrapper gives to tree_attention: a batch that could not be extended
    is one of empty sequences, its outputs are 0 whatever the memory held."""
    page, Hq, Hkv, D, B, n = 16, 32, 8, 128, 14, 65
    pool = KvCachePool(20, 1, Hkv, D, page, torch.bfloat16, torch.device(DEV))
    cache = SharedKvCache(pool, B, 16)
    w = BeFlashinferWrapper(Hq, Hkv, Hq * D, page, torch.device(DEV))
    cache.extend([0], 70)
    cache.fork([0] * (B - 1), list(range(1, B)))
    bp = cache.extend(list(range(B)), n)
    assert not K.sharing_pays(n, B, Hq, Hkv, D, page, torch.bfloat16)
    w.set_tree_masks(torch.tensor(chain(n) * B, dtype=torch.int32, device=DEV), bp, n)
    x = lambda h: torch.ones(B * n, h, D, dtype=torch.bfloat16, device=DEV)
    q, k = x(Hq), x(Hkv)
    for _ in range(3):
        junk = [torch.full((B * n, Hq, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(4)]
        del junk
        assert (w.computeAttention(q, k, k, pool.cache_data[0], "tree", bp, AttentionRotaryParams(), 0) == 0).all()
    with pytest.raises(RuntimeError):
        cache.check()


def test_a_stream_reports_only_its_own_waits():
    """A launch that gave up is reported on its own stream, whichever stream is checked
    first."""
    a = Case([(40, [(30, chain(1))] * 40)], Hq=32, Hkv=8, seed=2).device()
    K.tree_attention_shared(**a)
    torch.cuda.synchronize()
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    before = K.set_wait_limit(1)
    try:
        with torch.cuda.stream(s):
            K.tree_attention_shared(**a)
    finally:
        K.set_wait_limit(before)
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        K.tree_attention_shared(**a)
        K.check_attention(torch.device(DEV))
    with torch.cuda.stream(s):
        with pytest.raises(RuntimeError, match="gave up waiting"):
            K.check_attention(torch.device(DEV))
        K.check_attention(torch.device(DEV))


def test_a_captured_launch_that_gives_up_is_reported_after_its_replays():
    a = Case([(40, [(30, chain(1))] * 40)], Hq=32, Hkv=8, seed=2).device()
    K.tree_attention_shared(**a)
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    before = K.set_wait_limit(1)
    try:
        with torch.cuda.graph(g):
            K.tree_attention_shared(**a)
    finally:
        K.set_wait_limit(before)
    K.check_attention(torch.device(DEV))
    for _ in range(2):
        with torch.cuda.stream(s):
            g.replay()
            with pytest.raises(RuntimeError, match="gave up waiting"):
                K.check_attention(torch.device(DEV))
            K.check_attention(torch.device(DEV))


def test_boolean_masks_for_a_cache_whose_lengths_are_bounds():
    """prepareAttention takes the masks' widths from the sequences' lengths, also where
    the host only has bounds of them."""
    page, Hq, Hkv, D = 16, 4, 2, 64
    pool = KvCachePool(12, 1, Hkv, D, page, torch.float32, torch.device(DEV))
    cache = SharedKvCache(pool, 3, 4)
    w = BeFlashinferWrapper(Hq, Hkv, Hq * D, page, torch.device(DEV))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    cache.extend([0], 30)
    cache.fork([0], [1])
    cache.truncate([0, 1], i32([20, 11]))
    n = [3, 2]
    bp = cache.extend([0, 1], n)
    lens = [23, 13]
    masks = [torch.rand(a, L, generator=torch.Generator().manual_seed(L)) < 0.5 for a, L in zip(n, lens)]
    for m, a, L in zip(masks, n, lens):
        m[:, :L - a] = True
    w.prepareAttention("tree", bp, page, "NONE", torch.float32, torch.cat([m.reshape(-1) for m in masks]))
    want = [[sum(1 << j for j in range(a) if m[i, L - a + j]) for i in range(a)] for m, a, L in zip(masks, n, lens)]
    assert w._plan["bits"][:, 0].tolist() == sum(want, [])
    # the same through the attention: what set_tree_masks plans for chains
    chains = [torch.ones(a, L, dtype=torch.bool).tril(L - a) for a, L in zip(n, lens)]
    q, k = torch.randn(5, Hq, D, device=DEV), torch.randn(5, Hkv, D, device=DEV)
    outs = []
    for plan in (lambda: w.prepareAttention("tree", bp, page, "NONE", torch.float32, torch.cat([m.reshape(-1) for m in chains])),
                 lambda: w.set_tree_masks(i32(chain(3) + chain(2)), bp, 3)):
        plan()
        outs.append(w.computeAttention(q, k, k, pool.cache_data[0], "tree", bp, AttentionRotaryParams(), 0))
    assert torch.equal(*outs)
    with pytest.raises(ValueError, match="entries"):
        w.prepareAttention("tree", bp, page, "NONE", torch.float32, torch.cat([m.reshape(-1) for m in masks])[1:])
    bp = cache.extend([0, 1], 60)                             # cannot be done: no request has tokens
    with pytest.raises(ValueError, match="fewer tokens"):
        w.prepareAttention("tree", bp, page, "NONE", torch.float32, torch.zeros(0, dtype=torch.bool))
    with pytest.raises(RuntimeError):
        cache.check()


def test_bf16_beam_search_with_a_shared_prefix():
    """The bf16 search with ``shared_prefix``: every attention of a step that shares pages is
    what tree_attention gives for the same batch, up to the rounding of the probabilities
    and of the output (2^-8 of the largest value each, in both calls); the search leaves the
    pages that the one without it leaves."""
    from tests.test_gpu_reference_flow import D, HKV, PAGE, V, _patched_model
    model = _patched_model().to(torch.bfloat16)
    ids = torch.randint(0, V, (1, 75), generator=torch.Generator().manual_seed(3)).to(DEV)
    real, pairs, free = K.tree_attention_shared, [], []

    def both(q, kv, qo, pi, px, last, bits, max_qo, max_kv, groups, shared, **kw):
        got = real(q, kv, qo, pi, px, last, bits, max_qo, max_kv, groups, shared, **kw)
        want = K.tree_attention(q, kv, qo, pi, px, last, bits, max_qo, max_kv, sm_scale=kw["sm_scale"])
        pairs.append((shared.item(), (got.double() - want.double()).abs().max().item(), kv[px.long(), 1].abs().max().item()))
        return got

    for shared in (False, True):
        pool = KvCachePool(64, 2, HKV, D, PAGE, torch.bfloat16, torch.device(DEV))
        w = BeFlashinferWrapper(4, HKV, 256, PAGE, torch.device(DEV))
        K.tree_attention_shared = both
        try:
            tree_, _, _ = pbs.beam_search(model, RequestKvCache(pool, PAGE, 0), ids,
                                          pbs.BeamSearchConfig(topk_len=5, max_depth=6, shared_prefix=shared), w)
        finally:
            K.tree_attention_shared = real
        assert len(tree_.nodes) > 20
        free.append(pool.num_free_pages())
        assert bool(pairs) == shared
    assert all(n == 75 // PAGE and diff <= 2 * (2 * 2.0 ** -8 + 2.0 ** -12) * most for n, diff, most in pairs)
    assert len(pairs) >= 2 * 5                                # two layers, five steps or more
