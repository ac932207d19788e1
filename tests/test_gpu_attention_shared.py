"""Tree attention for requests that share leading pages, against dense attention in
fp64 over each request's own table.

Tolerances, per output element, with A = sum_j p_j |v_j| (p the exact probabilities),
u = 2^-24 and h the type's half step (bf16 2^-8, fp32 2^-24):
* the scores are fp32 dot products of D terms, each off by at most
  (D + 3) u scale sum |q||k|, so a probability is off by a factor within
  e^(2 ds) of 1, ds that bound over the row's columns (softmax quotients carry it
  twice), plus 2^-21 for exp of the difference and the join's second exp;
* the sums of n columns in fp32 add at most (n + 16) u each to O and to the row sum;
* the bf16 kernels round the probabilities to bf16 before the value product (at
  most h A) -- the row sum is taken before -- and every kernel rounds the output
  (h |o|)."""
import math

import numpy as np
import pytest
import torch

from oracle import attention as att
from parallel_tree_spec_b200 import kernels as K
from parallel_tree_spec_b200 import workload as wl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def chain(n):
    return [i - 1 for i in range(n)]


def tree(seed, width, depth):
    return wl.make_tree(np.random.default_rng(seed), width, depth, 100).parents.tolist()


class Case:
    """groups: [(shared pages, [(own prefix tokens, parents), ...]), ...]; parents []: a
    request without rows."""

    def __init__(self, groups, Hq=8, Hkv=2, D=128, pl=16, dtype=torch.bfloat16, seed=0, k_std=1.5, pad_rows=0):
        gen = torch.Generator().manual_seed(seed)
        self.Hq, self.Hkv, self.D, self.pl, self.dtype = Hq, Hkv, D, pl, dtype
        reqs = [(g, s, o, p) for g, (s, rs) in enumerate(groups) for o, p in rs]
        own = [-(-(o + len(p)) // pl) for _, _, o, p in reqs]
        P = sum(s for s, _ in groups) + sum(own) + 4
        perm = torch.randperm(P, generator=gen).tolist()
        heads = []
        for s, _ in groups:
            heads.append(perm[:s])
            perm = perm[s:]
        self.tables, self.lens, self.parents = [], [], []
        for (g, s, o, par), n in zip(reqs, own):
            self.tables.append(heads[g] + perm[:n])
            perm = perm[n:]
            self.lens.append(s * pl + o + len(par))
            self.parents.append(par)
        self.qo = np.cumsum([0] + [len(p) for p in self.parents]).tolist()
        self.groups = np.cumsum([0] + [len(rs) for _, rs in groups]).tolist()
        self.shared = [s for s, _ in groups]
        T = self.qo[-1] + pad_rows
        self.q = torch.randn(T, Hq, D, generator=gen).to(dtype)
        kv = torch.randn(P, 2, pl, Hkv, D, generator=gen)
        kv[:, 0] *= k_std
        self.kv = kv.to(dtype)
        self.masks = [torch.from_numpy(att.tree_mask(p, L - len(p))) if p else None
                      for p, L in zip(self.parents, self.lens)]
        self.causal = False
        self.scale = 1.0 / math.sqrt(D)

    def device(self):
        words = K.mask_words_for(max(len(p) for p in self.parents))
        bits = None
        if not self.causal:
            rows = []
            for p, m, L in zip(self.parents, self.masks, self.lens):
                for i in range(len(p)):
                    v = sum(1 << j for j in range(len(p)) if m[i, L - len(p) + j])
                    w = [(v >> (64 * k)) & (2 ** 64 - 1) for k in range(words)]
                    rows.append([x - 2 ** 64 if x >= 2 ** 63 else x for x in w])
            rows += [[-1] * words] * (self.q.shape[0] - len(rows))
            bits = torch.tensor(rows, dtype=torch.int64, device=DEV)
        last = [(L - 1) % self.pl + 1 if L else 0 for L in self.lens]
        return dict(q=self.q.to(DEV), kv_layer=self.kv.to(DEV), qo_indptr=i32(self.qo),
                    page_indptr=i32(np.cumsum([0] + [len(t) for t in self.tables]).tolist()),
                    page_indices=i32(sum(self.tables, []) or [0]), last_page_len=i32(last), mask_bits=bits,
                    max_qo_len=max(len(p) for p in self.parents), max_kv_len=max(self.lens),
                    group_indptr=i32(self.groups), shared_pages=i32(self.shared), sm_scale=self.scale)

    def exact(self):
        """(o, A, tolerance) in fp64 on the device."""
        n = self.qo[-1]
        o = torch.zeros(n, self.Hq, self.D, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(o)
        g, u = self.Hq // self.Hkv, 2.0 ** -24
        h = torch.finfo(self.dtype).eps / 2
        for b, par in enumerate(self.parents):
            if not par:
                continue
            lo, hi, L = self.qo[b], self.qo[b + 1], self.lens[b]
            x = self.kv[self.tables[b]].to(DEV).double()
            mask = self.masks[b].to(DEV)
            if self.causal:
                mask = torch.from_numpy(att.tree_mask(chain(len(par)), L - len(par))).to(DEV)
            for hk in range(self.Hkv):
                k, v = x[:, 0, :, hk].reshape(-1, self.D)[:L], x[:, 1, :, hk].reshape(-1, self.D)[:L]
                q = self.q[lo:hi, hk * g:(hk + 1) * g].to(DEV).double()
                seen = mask[:, None]
                any_ = mask.any(1)[:, None, None]
                # columns that no row sees hold anything
                k = torch.where(mask.any(0)[:, None], k, torch.zeros_like(k))
                v = torch.where(mask.any(0)[:, None], v, torch.zeros_like(v))
                s = (torch.einsum("ngd,ld->ngl", q, k) * self.scale).masked_fill(~seen, float("-inf"))
                p = torch.where(any_, torch.softmax(s, -1), torch.zeros_like(s))
                ds = (self.D + 3) * u * self.scale * torch.einsum("ngd,ld->ngl", q.abs(), k.abs()) \
                    .masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                A = torch.einsum("ngl,ld->ngd", p, v.abs())
                r = torch.einsum("ngl,ld->ngd", p, v)
                o[lo:hi, hk * g:(hk + 1) * g] = r
                rel = torch.expm1(2 * ds) + 2.0 ** -20 + 2 * (L + 16) * u + (h if self.dtype == torch.bfloat16 else 0.0)
                tol[lo:hi, hk * g:(hk + 1) * g] = rel * A * (1 + h) + h * r.abs() + 1e-30
        return o, tol


def check(c, out=None, **kw):
    a = c.device()
    a.update(kw)
    got = K.tree_attention_shared(**a) if out is None else out
    K.check_attention(torch.device(DEV))
    o, tol = c.exact()
    n = c.qo[-1]
    assert torch.isfinite(got[:n].float()).all()
    bad = (got[:n].double() - o).abs() / tol
    assert bad.max().item() <= 1.0, bad.max().item()
    return got


BOTH = [torch.bfloat16, torch.float32]
SMALL = [(3, [(5, tree(1, 3, 2)), (0, tree(2, 2, 2)), (20, chain(1))])]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("Hq,Hkv,D,pl", [(8, 2, 128, 16), (8, 8, 64, 16), (7, 1, 64, 32), (4, 2, 96, 16), (2, 1, 256, 8),
                                         (6, 3, 32, 5), (16, 1, 128, 64), (24, 8, 128, 48), (34, 2, 128, 16)])
def test_shapes(dtype, Hq, Hkv, D, pl):
    check(Case(SMALL, Hq=Hq, Hkv=Hkv, D=D, pl=pl, dtype=dtype, seed=D + pl))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("shared", [0, 1, 7, 8, 9, 16, 33, 130])
def test_shared_lengths(dtype, shared):
    """Nothing shared, less than a tile, whole tiles and one page more."""
    check(Case([(shared, [(3, chain(1)), (40, chain(1)), (0, tree(3, 2, 3))])], dtype=dtype, seed=shared))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("own", [0, 1, 15, 16, 17, 63, 64, 65, 500])
def test_own_lengths(dtype, own):
    check(Case([(10, [(own, chain(1)), (own + 1, chain(1)), (own, tree(own, 4, 4))])], dtype=dtype, seed=own))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", [1, 2, 31, 64, 65, 130, 300])
def test_decoding_batches(dtype, n):
    """n single tokens: row tiles of the group that end anywhere."""
    rng = np.random.default_rng(n)
    check(Case([(20, [(int(rng.integers(0, 40)), chain(1)) for _ in range(n)])], Hq=8, Hkv=2, D=64, dtype=dtype, seed=n))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("D", [64, 128])
def test_tree_sizes(dtype, D):
    """Trees of 1 to 129 rows: masks of one to three words, several row tiles each."""
    reqs = [(10, tree(1, 8, 8)), (33, tree(2, 16, 8)), (0, chain(1)), (5, tree(3, 1, 63)), (7, tree(4, 3, 5))]
    check(Case([(17, reqs)], D=D, dtype=dtype, seed=D))


@pytest.mark.parametrize("dtype", BOTH)
def test_groups(dtype):
    """Several groups: none shared, one request, requests without rows, empty caches."""
    reqs = lambda s: [(int(x), tree(int(x) + s, 2, 3)) for x in np.random.default_rng(s).integers(0, 90, size=4)]
    groups = [(12, reqs(1)), (0, reqs(2)), (40, [(6, chain(1))]), (3, [(5, []), (9, chain(2)), (0, [])]), (9, reqs(5))]
    check(Case(groups, Hq=12, Hkv=4, dtype=dtype, seed=11))


@pytest.mark.parametrize("dtype", BOTH)
def test_causal_rows(dtype):
    """Without masks a request's rows are causal (a chunk of a prompt, decoding)."""
    c = Case([(6, [(10, chain(40)), (0, chain(1)), (3, chain(90))]), (2, [(0, chain(17))])], dtype=dtype, seed=3)
    c.causal = True
    check(c)


@pytest.mark.parametrize("dtype", BOTH)
def test_rows_that_see_nothing_or_only_shared(dtype):
    """Rows whose mask is empty: 0 without a prefix, the prefix alone with one."""
    c = Case([(0, [(0, tree(1, 2, 3))]), (5, [(0, tree(2, 2, 3)), (0, tree(3, 2, 3))])], dtype=dtype, seed=4)
    for m, par, L in zip(c.masks, c.parents, c.lens):
        m[2:4, L - len(par):] = False
    got = check(c)
    assert (got[2:4] == 0).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_bad_values_in_places_that_are_not_seen(dtype, bad):
    """Slots past the length, pages of nobody, and tree slots that a row does not see:
    NaN and infinities there change nothing."""
    c = Case([(3, [(5, tree(1, 3, 3)), (2, tree(2, 3, 3)), (1, chain(1))])], dtype=dtype, seed=5)
    for tb, L in zip(c.tables, c.lens):
        if L % c.pl:
            c.kv[tb[-1], :, L % c.pl:] = bad
    used = set(sum(c.tables, []))
    c.kv[[i for i in range(c.kv.shape[0]) if i not in used]] = bad
    for b in (0, 1):                                         # the last tree slot: only its own row saw it
        L, n = c.lens[b], len(c.parents[b])
        c.masks[b][n - 1, L - 1] = False
        c.kv[c.tables[b][(L - 1) // c.pl], :, (L - 1) % c.pl] = bad
    check(c)


@pytest.mark.parametrize("dtype", BOTH)
def test_bad_value_reaches_only_the_rows_that_see_it(dtype):
    c = Case([(3, [(5, tree(1, 3, 3)), (2, chain(3))])], dtype=dtype, seed=6)
    L, n = c.lens[0], len(c.parents[0])
    c.kv[c.tables[0][(L - 1) // c.pl], 1, (L - 1) % c.pl, 0, 7] = float("nan")
    out = K.tree_attention_shared(**c.device()).float()
    g = c.Hq // c.Hkv
    assert torch.isnan(out[n - 1, :g, 7]).all()
    out[n - 1, :g, 7] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("shared,rows", [(3, 1), (3, 6), (0, 1), (40, 13)])
def test_nan_key_makes_the_rows_that_see_it_nan(dtype, shared, rows):
    """A NaN score is no masked one: its row is NaN in every dimension, the other KV
    head's rows and the other requests' are not; a shared key reaches all requests."""
    for at in ["own"] + ["shared"] * (shared > 0):
        c = Case([(shared, [(9, chain(rows)), (6, chain(1))])], dtype=dtype, seed=8)
        page = c.tables[0][shared if at == "own" else shared - 1]
        c.kv[page, 0, 2, 1, 5] = float("nan")
        out = K.tree_attention_shared(**c.device()).float()
        g = c.Hq // c.Hkv
        assert torch.isnan(out[:rows, g:2 * g]).all() and torch.isfinite(out[:, :g]).all()
        assert (torch.isnan if at == "shared" else torch.isfinite)(out[rows:, g:2 * g]).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_large_scores(dtype):
    """Scores far apart and rising along the cache: the running maximum moves often."""
    c = Case([(40, [(50, chain(1)), (70, tree(1, 3, 3))])], dtype=dtype, seed=7, k_std=6.0)
    for tb in c.tables:
        for j, page in enumerate(tb):
            c.kv[page, 0] = c.kv[page, 0] * (0.2 + 0.05 * j) if j > 39 or tb is c.tables[0] else c.kv[page, 0]
    check(c)


@pytest.mark.parametrize("dtype", BOTH)
def test_shared_pages_are_cut_to_the_prefix(dtype):
    """More shared pages than lie before the rows: the rest is each request's own."""
    c = Case([(6, [(0, tree(1, 2, 2)), (0, tree(2, 2, 2))])], dtype=dtype, seed=8)
    c.tables[1][6:] = c.tables[0][6:]                         # every page is the same
    a = c.device()
    want = K.tree_attention_shared(**a)
    a["shared_pages"] = i32([100])
    assert torch.equal(K.tree_attention_shared(**a), want)
    check(c)


@pytest.mark.parametrize("dtype", BOTH)
def test_rows_behind_the_last_request_are_left(dtype):
    c = Case(SMALL, dtype=dtype, seed=9, pad_rows=13)
    out = torch.full_like(c.q, 7.0).to(DEV)
    got = K.tree_attention_shared(**dict(c.device(), out=out))
    check(c, out=got)
    assert got is out and (out[c.qo[-1]:] == 7.0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_agrees_with_tree_attention(D):
    """The same tables read as unshared requests."""
    c = Case([(70, [(100, tree(1, 8, 8)), (9, tree(2, 8, 8)), (40, chain(1))]), (300, [(0, tree(3, 4, 4))])], D=D,
             seed=10)
    a = c.device()
    got = check(c)
    plain = {k: a[k] for k in ("q", "kv_layer", "qo_indptr", "page_indptr", "page_indices", "last_page_len", "mask_bits",
                               "max_qo_len", "max_kv_len", "sm_scale")}
    _, tol = c.exact()
    assert ((got.double() - K.tree_attention(**plain).double()).abs() <= 2 * tol).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_long_prefix_and_long_own(dtype):
    check(Case([(520, [(int(x), chain(1)) for x in (3000, 10, 700)])], Hq=4, Hkv=1, D=128, dtype=dtype, seed=12))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("bounds", [dict(max_kv_len=1), dict(max_kv_len=1 << 30), dict(max_kv_len=2 ** 40, max_own_len=1),
                                    dict(max_own_len=0), dict(max_own_len=1 << 40)])
def test_wrong_length_bounds_change_only_the_schedule(dtype, rows, bounds):
    check(Case([(60, [(200, chain(rows)), (3, chain(1))] * 5), (0, [(90, chain(rows))])], dtype=dtype, seed=14), **bounds)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("D", [64, 128])
def test_group_ranges_and_last_pages_are_cut(dtype, D):
    """Group ends past the batch, and a last page said to hold more than a page: as if they
    named the batch and the whole page."""
    c = Case([(30, [(11, chain(n)), (25, chain(n))]) for n in (1, 7)], D=D, dtype=dtype, seed=15)
    a = c.device()
    B = a["last_page_len"].numel()
    groups = a["group_indptr"].clone()
    groups[-1] = B + 1000
    check(c, group_indptr=groups)
    full = a["last_page_len"].clone().fill_(c.pl)
    want = K.tree_attention_shared(**dict(a, last_page_len=full))
    assert torch.equal(K.tree_attention_shared(**dict(a, last_page_len=full + 1000)), want)


def test_repeat_is_the_same():
    c = Case([(200, [(50, chain(1))] * 40)], Hq=32, Hkv=8, seed=13)
    a = c.device()
    assert torch.equal(K.tree_attention_shared(**a), K.tree_attention_shared(**a))


def test_graph_replays_with_other_lengths():
    """A captured call reads lengths and tables on the device: replayed with a longer
    shared prefix it gives that prefix's result."""
    c1 = Case([(10, [(20, chain(1))] * 6)], seed=14)
    c2 = Case([(37, [(90, chain(1))] * 6)], seed=15)
    a1, a2 = c1.device(), c2.device()
    for a in (a1, a2):
        a["max_kv_len"] = max(c1.lens[0], c2.lens[0])
    bufs = {k: a1[k].clone() for k in ("q", "qo_indptr", "page_indptr", "last_page_len", "group_indptr", "shared_pages",
                                       "mask_bits")}
    n = max(a["page_indices"].numel() for a in (a1, a2))
    bufs["page_indices"] = torch.zeros(n, dtype=torch.int32, device=DEV)
    P = max(c1.kv.shape[0], c2.kv.shape[0])
    bufs["kv_layer"] = torch.zeros(P, *c1.kv.shape[1:], dtype=c1.dtype, device=DEV)
    out = torch.empty_like(bufs["q"])

    def load(a):
        for k, t in bufs.items():
            t[:a[k].shape[0]].copy_(a[k]) if k in ("page_indices", "kv_layer") else t.copy_(a[k])

    load(a1)
    call = dict(a1, out=out, **bufs)
    K.tree_attention_shared(**call)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.tree_attention_shared(**call)
    for c, a in ((c2, a2), (c1, a1), (c2, a2)):
        load(a)
        out.zero_()
        g.replay()
        check(c, out=out)


def test_two_streams_at_once():
    cs = [Case([(60, [(50, chain(1))] * 20)], seed=16 + i, dtype=d) for i, d in enumerate(BOTH)]
    args = [c.device() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] = K.tree_attention_shared(**args[i])
    torch.cuda.synchronize()
    for c, o in zip(cs, outs):
        check(c, out=o)


def test_refusals():
    c = Case(SMALL, seed=20)
    a = c.device()
    for k, v in (("q", a["q"].half()), ("q", a["q"].transpose(0, 1)), ("kv_layer", a["kv_layer"][:, :, ::2]),
                 ("kv_layer", a["kv_layer"].float()), ("group_indptr", a["group_indptr"].long()),
                 ("group_indptr", i32([0, 1, 3])), ("last_page_len", a["last_page_len"][:-1]),
                 ("mask_bits", a["mask_bits"][:-1]), ("mask_bits", a["mask_bits"].int()), ("max_qo_len", 200),
                 ("max_qo_len", 0), ("out", torch.empty(1, 8, 128, device=DEV)), ("q", a["q"].cpu()),
                 ("page_indptr", a["page_indptr"].cpu())):
        with pytest.raises(ValueError):
            K.tree_attention_shared(**dict(a, **{k: v}))
    odd = Case(SMALL, D=128, seed=21)
    odd.q, odd.kv = odd.q[..., :48].contiguous(), odd.kv[..., :48].contiguous()
    with pytest.raises(Exception, match="head_dim"):
        K.tree_attention_shared(**odd.device())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("shared,own", [(0, 0), (0, 5), (3, 0), (3, 21), (600, 40)])
def test_a_lone_row_that_does_not_see_its_own_slot(dtype, bad, shared, own):
    """One row per request, masked from its own slot, whose value is infinite or NaN."""
    c = Case([(shared, [(own, chain(1)), (own + 16, chain(1))] * 8)], dtype=dtype, seed=17)
    for b in range(0, 16, 3):
        L = c.lens[b]
        c.masks[b][0, L - 1] = False
        c.kv[c.tables[b][(L - 1) // c.pl], 1, (L - 1) % c.pl] = bad
    got = check(c)
    if not shared and not own:
        assert (got[0] == 0).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("scale", [-0.25, 0.0, 1e-40, -1e-3])
@pytest.mark.parametrize("shared,rows", [(5, 1), (5, 6), (700, 1), (20, 70)])
def test_scales_that_are_not_positive(dtype, scale, shared, rows):
    """Negative scales and 0 (the mean of what a row sees), through each of the kernels: the
    queries' negatives with the scale's magnitude say what they give."""
    c = Case([(shared, [(9, chain(rows)), (6, chain(1))])], dtype=dtype, seed=9)
    c.scale = abs(scale)
    q = c.q
    if scale < 0:
        c.q = -q
    check(c, q=q.to(DEV), sm_scale=scale)


@pytest.mark.parametrize("rows,Hq,Hkv,pl", [(1, 32, 8, 16), (3, 32, 8, 48), (1, 8, 8, 128), (2, 48, 6, 16)])
@pytest.mark.parametrize("groups", [1, 3])
def test_decoding_with_more_own_columns_than_shared(rows, Hq, Hkv, pl, groups):
    """Few rows, head_dim 128 and a bound of the own columns that says that they are more
    than the shared ones: the ring of three slots, own columns in slices beside it."""
    rng = np.random.default_rng(rows + groups)
    B = 60 // groups
    gs = [(int(rng.integers(1, 30)), [(int(x), chain(rows)) for x in rng.integers(0, 300, size=B)]) for _ in range(groups)]
    c = Case(gs, Hq=Hq, Hkv=Hkv, D=128, pl=pl, seed=30 + rows)
    own = 300 + rows
    longest = max(c.lens)
    assert rows * Hq // Hkv <= 16 and B * groups * own >= groups * (longest - own)
    assert -(-B * groups * Hkv // 148) * (600 + longest) > 3600     # not the one launch of small calls
    check(c, max_own_len=own)


@pytest.mark.parametrize("groups,per_group,rows", [(1, 511, 5), (1, 512, 5), (2, 260, 5), (512, 1, 1), (513, 1, 1), (600, 2, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_plans_of_more_column_sets_than_fit_shared_memory(groups, per_group, rows, D):
    """512 column sets and more: the groups' shared columns and, for trees, each request's
    own; from 513 on the plan is made in global memory."""
    rng = np.random.default_rng(groups + per_group)
    gs = [(int(rng.integers(0, 12)), [(int(rng.integers(0, 40)), tree(int(rng.integers(100)), 2, 2) if rows == 5 else chain(1))
                                      for _ in range(per_group)]) for _ in range(groups)]
    c = Case(gs, Hq=8, Hkv=2, D=D, seed=groups + rows)
    assert all(len(p) == rows for p in c.parents)
    assert rows > 4 or -(-len(c.parents) * 2 // 148) * (600 + max(c.lens)) > 3600
    check(c)


@pytest.mark.parametrize("rows,own", [(1, 0), (1, 300), (9, 40), (65, 70)])
@pytest.mark.parametrize("pl", [112, 128, 192, 256, 1024])
@pytest.mark.parametrize("D", [64, 128])
def test_long_pages(D, pl, rows, own):
    """Pages of a block and more: one copy per block, or several where a page's length is no
    multiple of a block's."""
    par = chain(rows) if rows < 9 else tree(rows, 8, 8) if rows == 65 else tree(rows, 2, 4)
    reqs = [(own + i, par) for i in range(40 if rows == 1 else 3)]
    check(Case([(3, reqs), (0, reqs[:2])], Hq=8 if rows > 1 else 32, Hkv=2 if rows > 1 else 8, D=D, pl=pl, seed=pl + rows))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["beams", "decoding", "trees", "nan"])
def test_pages_past_32_bits(dtype, D, kind):
    """The pages are the last ones of a layer of more than 2^31 elements."""
    par = tree(1, 8, 8) if kind in ("trees", "nan") else chain(1)
    c = Case([(20, [(9, par), (30, chain(1))] * (40 if kind == "decoding" else 2))], Hq=32, Hkv=8, D=D, dtype=dtype, seed=18)
    if kind == "nan":                                         # the last tree slot, which only its own row saw, holds one
        L, n = c.lens[0], len(par)
        c.masks[0][n - 1, L - 1] = False
        c.kv[c.tables[0][(L - 1) // c.pl], 1, (L - 1) % c.pl] = float("nan")
    a = c.device()
    P = 2 ** 31 // (2 * c.pl * 8 * D) + c.kv.shape[0] + 100
    layer = torch.empty(P, *c.kv.shape[1:], dtype=dtype, device=DEV)
    assert layer.numel() > 2 ** 31
    at = P - c.kv.shape[0]
    layer[at:] = c.kv.to(DEV)
    check(c, kv_layer=layer, page_indices=a["page_indices"] + at)
