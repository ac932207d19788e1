"""The operators of a cache whose sequences share pages, as they are measured.

Two families, each in a plain form (elementary torch operations in fp32) and as
calls of this package (``own``):

* ``attend``   tree attention for a batch whose requests share long prefixes: the
               leading ``shared_pages[g]`` pages of every request of group g are the
               same physical pages;
* ``branch``   forking sequences (children take their parents' pages) and extending
               the children, which copies the partial last page that they share;
* ``step``     extending every sequence by a draft tree and truncating back, the page
               bookkeeping of a verification step;
* ``compact``  moving the live pages to the pool's low end and rewriting the tables.

Page state: ``page_refs`` int32 [P] counts the tables that hold a page (0: free),
``page_table`` int32 [R, W] lists each sequence's pages (-1 past its end),
``kv_lens`` int32 [R] their tokens.  Free pages are handed out lowest first.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a draft model's beam search: six beams one token past a short prompt
        dict(name="attend_beams", op="attend", dtype="bf16", Hq=32, Hkv=8, D=64, pl=16, groups=1, seqs=6, shared=512,
             own=10, width=0, depth=0),
        # decoding 64 samples of one long prompt
        dict(name="attend_decode", op="attend", dtype="bf16", Hq=32, Hkv=8, D=128, pl=16, groups=1, seqs=64,
             shared=8192, own=300, width=0, depth=0),
        # decoding 32 answers about one very long document
        dict(name="attend_document", op="attend", dtype="bf16", Hq=32, Hkv=8, D=128, pl=16, groups=1, seqs=32,
             shared=65536, own=500, width=0, depth=0),
        # verifying 16 draft trees (65 nodes) after one 4096-token system prompt
        dict(name="attend_trees", op="attend", dtype="bf16", Hq=32, Hkv=8, D=128, pl=16, groups=1, seqs=16,
             shared=4096, own=200, width=8, depth=8),
        # small trees (13 nodes) of 40 requests under three system prompts of odd lengths
        dict(name="attend_prompts", op="attend", dtype="bf16", Hq=28, Hkv=4, D=128, pl=32, groups=3, seqs=40,
             shared=3000, own=700, width=3, depth=4),
        # the small fp32 configuration: 15-node trees after a shared 128-token prefix
        dict(name="attend_fp32", op="attend", dtype="fp32", Hq=4, Hkv=2, D=64, pl=16, groups=1, seqs=8, shared=128,
             own=40, width=2, depth=7),
        # a beam step of a 16-layer draft model: 6 children of 3 surviving beams, one token each
        dict(name="branch_beams", op="branch", dtype="bf16", layers=16, Hkv=8, D=64, pl=16, parents=3, children=6,
             length=512, add=1, pages=2048),
        # 128 samples of 16 prompts in a 16-layer cache, room for one token each
        dict(name="branch_samples", op="branch", dtype="bf16", layers=16, Hkv=8, D=128, pl=16, parents=16,
             children=128, length=1500, add=1, pages=2500),
        # room for one 65-node tree per request and back, the benchmark's batch
        dict(name="step_trees", op="step", dtype="bf16", layers=1, Hkv=8, D=128, pl=16, seqs=16, length=4096, add=65,
             pages=8192),
        # the same for a large batch in a large pool
        dict(name="step_batch", op="step", dtype="bf16", layers=1, Hkv=2, D=64, pl=16, seqs=512, length=2048, add=49,
             pages=100000),
        # closing the gaps of a small fp32 pool
        dict(name="compact_small", op="compact", dtype="fp32", layers=2, Hkv=2, D=64, pl=16, seqs=12, length=300,
             pages=512),
        # closing the gaps that finished requests left in a 16-layer cache
        dict(name="compact_pool", op="compact", dtype="bf16", layers=16, Hkv=8, D=128, pl=16, seqs=24, length=1800,
             pages=4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "branch", "step", "compact"])
    if op == "attend":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        Hq, Hkv = rng.choice([(32, 8), (16, 2), (8, 8), (28, 4), (4, 2), (24, 8), (64, 8)])
        D = rng.choice([64, 128])
        width, depth = rng.choice([(0, 0), (0, 0), (2, 3), (3, 4), (4, 8), (8, 8)])
        groups = rng.choice([1, 1, 2, 5])
        while True:
            seqs = groups * _log(rng, 2, 64)
            shared, left = _log(rng, 64, 65536), _log(rng, 1, 2000)
            c = dict(op=op, dtype=dtype, Hq=Hq, Hkv=Hkv, D=D, pl=rng.choice([16, 16, 32, 64]), groups=groups,
                     seqs=seqs, shared=shared, own=left, width=width, depth=depth)
            flops = 4.0 * D * Hq * seqs * (1 + width * depth) * (shared + left)
            size = 4.0 * D * Hkv * (groups * shared + seqs * (left + width * depth)) * (2 if dtype == "fp32" else 1)
            if flops <= (60e9 if dtype == "bf16" else 6e9) and size <= 3e8:
                return c
    if op == "branch":
        parents = _log(rng, 1, 16)
        children, length = _log(rng, parents, 128), _log(rng, 1, 1500)
        layers, (Hkv, D) = rng.choice([2, 8, 16]), rng.choice([(8, 128), (8, 64), (2, 64), (3, 32)])
        pl = rng.choice([16, 16, 32, 8])
        pages = parents * (length // pl + 2) + children * 3 + rng.randrange(64)
        return dict(op=op, dtype=rng.choice(["bf16", "fp32"]), layers=layers, Hkv=Hkv, D=D, pl=pl, parents=parents,
                    children=children, length=length, add=rng.randrange(1, 17), pages=pages)
    if op == "step":
        seqs, length, pl = _log(rng, 1, 512), _log(rng, 1, 4096), rng.choice([16, 16, 32, 8])
        add = rng.randrange(1, 130)
        return dict(op=op, dtype="bf16", layers=rng.choice([1, 2]), Hkv=2, D=64, pl=pl, seqs=seqs, length=length,
                    add=add, pages=min(100000, seqs * ((length + add) // pl + 3)) + rng.randrange(999))
    seqs, length, pl = _log(rng, 1, 24), _log(rng, 10, 1800), rng.choice([16, 16, 32])
    Hkv, D = rng.choice([(8, 128), (8, 64), (2, 64)])
    return dict(op=op, dtype=rng.choice(["bf16", "fp32"]), layers=rng.choice([2, 8]), Hkv=Hkv, D=D, pl=pl, seqs=seqs,
                length=length, pages=seqs * (length // pl + 2) + _log(rng, 1, 1000))


# ------------------------------------------------------- shapes of a case
def _attend_shapes(case):
    """Host lengths of an attention case: the groups' first requests, the shared pages of each
    group, each request's own prefix tokens (after the shared pages) and its rows."""
    rng = random.Random("attend %(seqs)d %(groups)d %(shared)d %(own)d %(width)d %(depth)d" % case)
    B, G, pl = case["seqs"], case["groups"], case["pl"]
    cuts = sorted(rng.sample(range(1, B), G - 1)) if G > 1 else []
    starts = [0] + cuts + [B]
    pages = [max(1, case["shared"] // pl - (rng.randrange(case["shared"] // pl // 2 + 1) if G > 1 else 0))
             for _ in range(G)]
    own_prefix = [rng.randint(case["own"] // 2, case["own"]) for _ in range(B)]
    n = 1 + case["width"] * case["depth"]
    rows = [n if n == 1 or rng.random() < 0.7 else rng.randint(2, n) for _ in range(B)]
    rows[0] = n
    return starts, pages, own_prefix, rows


def _tree_parents(rng, n, width):
    """Parents of an n-node draft tree in breadth-first order: a root, then levels of `width`."""
    parents, prev, level = [-1], [0], []
    for i in range(1, n):
        parents.append(rng.choice(prev))
        level.append(i)
        if len(level) == width:
            prev, level = level, []
    return parents


def _trees(case):
    _, _, _, rows = _attend_shapes(case)
    rng = random.Random("trees %(seqs)d %(width)d %(depth)d" % case)
    return [_tree_parents(rng, n, max(1, case["width"])) for n in rows]


def _lengths(case):
    rng = random.Random("lengths %(op)s %(length)d %(pages)d" % case)
    n = case["parents"] if case["op"] == "branch" else case["seqs"]
    return [rng.randint(max(1, case["length"] // 2), case["length"]) for _ in range(n)]


def _pages_of(tokens, pl):
    return (tokens + pl - 1) // pl


# ---------------------------------------------------------------- prepare
def prepare(case, seed):
    return _PREPARE[case["op"]](case, seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _prepare_attend(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    starts, shared, own_prefix, rows = _attend_shapes(case)
    B, pl, Hq, Hkv, D, dt = case["seqs"], case["pl"], case["Hq"], case["Hkv"], case["D"], DTYPES[case["dtype"]]
    own_len = [o + n for o, n in zip(own_prefix, rows)]
    own_pages = [_pages_of(t, pl) for t in own_len]
    P = sum(shared) + sum(own_pages) + 3
    perm = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
    at, group_pages = 0, []
    for s in shared:
        group_pages.append(perm[at:at + s])
        at += s
    indptr, indices, last, group_of = [0], [], [], []
    for g in range(case["groups"]):
        group_of += [g] * (starts[g + 1] - starts[g])
    for b in range(B):
        indices += group_pages[group_of[b]] + perm[at:at + own_pages[b]]
        at += own_pages[b]
        indptr.append(len(indices))
        last.append((own_len[b] - 1) % pl + 1)
    qo, bits, words = [0], [], (max(rows) + 63) // 64
    for parents in _trees(case):
        anc = []
        for i, p in enumerate(parents):
            anc.append((anc[p] if p >= 0 else 0) | (1 << i))
        for m in anc:
            w = [(m >> (64 * k)) & (2 ** 64 - 1) for k in range(words)]
            bits.append([x - 2 ** 64 if x >= 2 ** 63 else x for x in w])
        qo.append(qo[-1] + len(parents))
    # queries and keys of a trained model score a few tokens well above the rest
    kv = torch.randn(P, 2, pl, Hkv, D, generator=gen, device=DEV)
    kv[:, 0] *= 1.5
    return dict(op="attend", q=torch.randn(qo[-1], Hq, D, generator=gen, device=DEV).to(dt), kv=kv.to(dt), qo=_i32(qo),
                indptr=_i32(indptr), indices=_i32(indices), last=_i32(last), groups=_i32(starts), shared=_i32(shared),
                bits=torch.tensor(bits, dtype=torch.int64, device=DEV), max_qo=max(rows),
                max_kv=max(pl * s for s in shared) + max(own_len), max_own=max(own_len), max_shared=max(shared),
                max_group=max(qo[starts[g + 1]] - qo[starts[g]] for g in range(case["groups"])))


def _pool(case, gen):
    shape = (case["layers"], case["pages"], 2, case["pl"], case["Hkv"], case["D"])
    return torch.randn(shape, generator=gen, device=DEV, dtype=DTYPES[case["dtype"]])


def _table(case, seed, lengths, rows, width):
    """Scattered pages for the first sequences of a table of `rows`."""
    perm = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed))
    table = torch.full((rows, width), -1, dtype=torch.int32)
    refs = torch.zeros(case["pages"], dtype=torch.int32)
    at = 0
    for i, n in enumerate(lengths):
        k = _pages_of(n, case["pl"])
        table[i, :k] = perm[at:at + k].int()
        refs[perm[at:at + k]] = 1
        at += k
    lens = torch.zeros(rows, dtype=torch.int32)
    lens[:len(lengths)] = torch.tensor(lengths, dtype=torch.int32)
    return refs.to(DEV), table.to(DEV), lens.to(DEV)


def _prepare_branch(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    p, c = case["parents"], case["children"]
    width = _pages_of(case["length"] + case["add"], case["pl"]) + 1
    refs, table, lens = _table(case, seed, _lengths(case), p + c, width)
    rng = random.Random("beams %(parents)d %(children)d %(length)d" % case)
    src = sorted(rng.randrange(p) for _ in range(c))
    starts = [0] + [i for i in range(1, c) if src[i] != src[i - 1]] + [c]
    return dict(op="branch", pool=_pool(case, gen), refs=refs, table=table, lens=lens, src=_i32(src),
                dst=torch.arange(p, p + c, dtype=torch.int32, device=DEV), add=case["add"], groups=_i32(starts),
                out=_batch_buffers(c, width, len(starts) - 1))


def _batch_buffers(B, width, groups):
    """page_indptr, page_indices, last_page_len, seq_lens, shared_pages of a batch."""
    return (_i32([0] * (B + 1)), torch.full((B * width,), -1, dtype=torch.int32, device=DEV), _i32([0] * B),
            _i32([0] * B), _i32([0] * groups))


def _prepare_step(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, width = case["seqs"], _pages_of(case["length"] + case["add"], case["pl"])
    lengths = _lengths(case)
    room = case["pages"] - sum(_pages_of(case["add"], case["pl"]) + 1 for _ in lengths)
    kept = []                                          # as many of the sequences as the pool holds pages for
    for n in lengths:
        room -= _pages_of(n, case["pl"])
        kept.append(n if room >= 0 else 0)
        room += 0 if room >= 0 else _pages_of(n, case["pl"])
    refs, table, lens = _table(case, seed, kept, B, width)
    rows = torch.randperm(B, generator=torch.Generator().manual_seed(seed + 1)).int().to(DEV)
    return dict(op="step", pool=_pool(case, gen), refs=refs, table=table, lens=lens, rows=rows,
                add=torch.full((B,), case["add"], dtype=torch.int32, device=DEV), keep=lens[rows.long()].clone(),
                groups=_i32([0, B]), out=_batch_buffers(B, width, 1))


def _prepare_compact(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    width = _pages_of(case["length"], case["pl"]) + 1
    refs, table, lens = _table(case, seed, _lengths(case), case["seqs"] + 1, width)
    table[-1] = table[0]                               # a fork of the first sequence
    refs[table[0][table[0] >= 0].long()] += 1
    return dict(op="compact", pool=_pool(case, gen), refs=refs, table=table)


_PREPARE = {"attend": _prepare_attend, "branch": _prepare_branch, "step": _prepare_step, "compact": _prepare_compact}


# -------------------------------------------------------------------- run
def run(state):
    if own:
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


def _own_attend(s):
    from parallel_tree_spec_b200 import kernels as K
    return K.tree_attention_shared(s["q"], s["kv"], s["qo"], s["indptr"], s["indices"], s["last"], s["bits"],
                                   s["max_qo"], s["max_kv"], s["groups"], s["shared"], max_own_len=s["max_own"])


def _own_branch(s):
    from parallel_tree_spec_b200 import kernels as K
    forked = K.cache_fork(s["refs"], s["table"], s["lens"], s["src"], s["dst"])
    b = K.cache_extend(s["pool"], s["refs"], s["table"], s["lens"], s["dst"], s["add"], group_indptr=s["groups"],
                       out=s["out"])
    return dict(pool=s["pool"], refs=s["refs"], table=s["table"], lens=s["lens"], batch=list(b[:5]), forked=forked,
                status=b.status)


def _own_step(s):
    from parallel_tree_spec_b200 import kernels as K
    b = K.cache_extend(s["pool"], s["refs"], s["table"], s["lens"], s["rows"], s["add"], group_indptr=s["groups"],
                       out=s["out"])
    back = K.cache_truncate(s["refs"], s["table"], s["lens"], s["pool"].shape[3], s["rows"], s["keep"])
    return dict(pool=s["pool"], refs=s["refs"], table=s["table"], lens=s["lens"], batch=list(b[:5]), status=b.status,
                back=back)


def _own_compact(s):
    from parallel_tree_spec_b200 import kernels as K
    r = K.cache_compact(s["pool"], s["refs"], s["table"])
    return dict(pool=s["pool"], refs=r.page_refs, table=r.page_table, map=r.page_map, counts=r.counts)


_OWN = {"attend": _own_attend, "branch": _own_branch, "step": _own_step, "compact": _own_compact}


def _masked_softmax_parts(scores, visible, values):
    """exp(s - m) V with the row max m and the row sum, over the visible columns only."""
    s = scores.masked_fill(~visible, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    return p @ values, m, p.sum(-1, keepdim=True)


def _plain_attend(s):
    q, kv, pl = s["q"].float(), s["kv"], s["kv"].shape[2]
    T, Hq, D = q.shape
    Hkv = kv.shape[3]
    g = Hq // Hkv
    scale = 1.0 / math.sqrt(D)
    qo, indptr, groups, shared = s["qo"].long(), s["indptr"].long(), s["groups"].long(), s["shared"].long()
    B, G = qo.numel() - 1, groups.numel() - 1
    dev = q.device
    token = torch.arange(T, device=dev)
    req = torch.searchsorted(qo, token, right=True) - 1
    grp = torch.searchsorted(groups, torch.arange(B, device=dev), right=True) - 1
    shared_of = shared[grp]
    q = q.view(T, Hkv, g, D)
    # the shared pages, once for each group: rows of all its requests
    t0 = qo[groups[:-1]]
    col = torch.arange(s["max_group"], device=dev)
    rows = (t0[:, None] + col).clamp(max=T - 1)
    qs = q[rows].permute(0, 2, 1, 3, 4).reshape(G, Hkv, -1, D)
    page = torch.arange(s["max_shared"], device=dev)
    idx = s["indices"].long()[(indptr[groups[:-1]][:, None] + page).clamp(max=s["indices"].numel() - 1)]
    seen = (torch.arange(s["max_shared"] * pl, device=dev) < shared[:, None] * pl)[:, None, None, :]
    ks = kv[idx, 0].reshape(G, -1, Hkv, D).permute(0, 2, 1, 3).float()
    vs = kv[idx, 1].reshape(G, -1, Hkv, D).permute(0, 2, 1, 3).float()
    o1, m1, l1 = _masked_softmax_parts(qs @ ks.transpose(-1, -2) * scale, seen, vs)
    # each request's own pages
    pages = -(-s["max_own"] // pl)
    first = indptr[:-1] + shared_of
    at = first[:, None] + torch.arange(pages, device=dev)
    idx = s["indices"].long()[torch.minimum(at, indptr[1:, None] - 1)]
    n = qo[1:] - qo[:-1]
    own_len = (indptr[1:] - first - 1) * pl + s["last"].long()
    slot = torch.arange(pages * pl, device=dev)
    node = slot - (own_len - n)[:, None]                                      # [B, S]
    col = torch.arange(s["max_qo"], device=dev)
    rows = (qo[:-1, None] + col).clamp(max=T - 1)
    word = s["bits"][rows]                                                    # [B, N, words]
    where = node.clamp(min=0)[:, None, :].expand(B, rows.shape[1], -1)
    bit = (torch.gather(word, 2, (where >> 6).clamp(max=word.shape[2] - 1)) >> (where & 63)) & 1
    seen = ((node[:, None] < 0) | ((node[:, None] < n[:, None, None]) & (bit == 1))) & (slot < own_len[:, None])[:, None]
    seen = seen[:, None, :, None, :].expand(B, Hkv, -1, g, -1).reshape(B, Hkv, -1, pages * pl)
    qs = q[rows].permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    ks = kv[idx, 0].reshape(B, -1, Hkv, D).permute(0, 2, 1, 3).float()
    vs = kv[idx, 1].reshape(B, -1, Hkv, D).permute(0, 2, 1, 3).float()
    o2, m2, l2 = _masked_softmax_parts(qs @ ks.transpose(-1, -2) * scale, seen, vs)
    # joined row by row
    a = lambda x: x.view(G, Hkv, -1, g, x.shape[-1])[grp[req], :, token - t0[grp[req]]]
    b = lambda x: x.view(B, Hkv, -1, g, x.shape[-1])[req, :, token - qo[:-1][req]]
    m = torch.maximum(a(m1), b(m2))
    w1, w2 = torch.exp(a(m1) - m), torch.exp(b(m2) - m)
    out = (w1 * a(o1) + w2 * b(o2)) / (w1 * a(l1) + w2 * b(l2))
    return out.reshape(T, Hq, D).to(s["q"].dtype)


def _count(index, weight, n):
    return torch.zeros(n, dtype=torch.int32, device=index.device).index_add_(0, index, weight.int())


def _plain_fork(s):
    table, refs, src, dst = s["table"], s["refs"], s["src"].long(), s["dst"].long()
    old, new = table[dst].long(), table[src].long()
    P = refs.numel()
    refs += _count(new.clamp(min=0).view(-1), (new >= 0).view(-1), P) - _count(old.clamp(min=0).view(-1),
                                                                               (old >= 0).view(-1), P)
    table[dst] = new.int()
    s["lens"][dst] = s["lens"][src]
    return torch.zeros(1, dtype=torch.int32, device=refs.device)


def _plain_extend(s, rows, add):
    pool, refs, table, lens = s["pool"], s["refs"], s["table"], s["lens"]
    P, pl, W = refs.numel(), pool.shape[3], table.shape[1]
    r = rows.long()
    B, dev = r.numel(), r.device
    old = lens[r].long()
    new = old + add
    n_old, n_new = (old + pl - 1) // pl, (new + pl - 1) // pl
    # a partial last page that another table holds too is copied; when the listed rows are its only
    # holders, the last of them keeps it
    order = torch.arange(B, device=dev)
    part = (new > old) & (old % pl != 0)
    last = table[r, (n_old - 1).clamp(min=0)].long().clamp(min=0)
    here = _count(last, part, P)
    final = torch.full((P,), -1, device=dev).scatter_reduce_(0, last, torch.where(part, order, -1), "amax")
    copy = part & (refs[last] > 1) & ~((here[last] == refs[last]) & (final[last] == order))
    need = n_new - n_old + copy
    start = need.cumsum(0) - need
    total = need.sum()
    free = (refs == 0).nonzero().view(-1)
    status = torch.where(total > free.numel(), 8, 0).int().view(1)
    most = (n_new - n_old).max() + 1
    k = torch.arange(int(most), device=dev)
    wanted = k < need[:, None]
    got = free[(start[:, None] + k).clamp(max=free.numel() - 1)]              # [B, most]
    refs -= _count(last, copy, P)
    refs[got[wanted]] = 1
    off = torch.where(copy, old % pl, 0)
    who = copy.nonzero().view(-1)
    slots = (torch.arange(pl, device=dev) < off[who, None])[None, :, None, :, None, None]
    pool[:, got[who, 0]] = torch.where(slots, pool[:, last[who]], pool[:, got[who, 0]])
    where = n_old[:, None] + k - copy[:, None].long()
    table[r[:, None].expand_as(where)[wanted], where[wanted]] = got[wanted].int()
    lens[r] = new.int()
    # the batch's page lists
    indptr, indices, last_len, seq, shared = s["out"]
    indptr[1:] = n_new.cumsum(0)
    col = torch.arange(W, device=dev)
    inside = col < n_new[:, None]
    indices[(indptr[:-1].long()[:, None] + col)[inside]] = table[r][inside]
    last_len.copy_(torch.where(new > 0, (new - 1) % pl + 1, 0))
    seq.copy_(new)
    groups = s["groups"].long()
    grp = torch.searchsorted(groups, order, right=True) - 1
    same = (table[r] == table[r[groups[:-1]]][grp]) & (col < (old // pl)[:, None])
    run_ = same.int().cumprod(1).sum(1)
    shared.copy_(torch.full_like(shared, W).scatter_reduce_(0, grp, run_.int(), "amin"))
    return status


def _plain_truncate(s, rows, keep):
    refs, table, lens, pl = s["refs"], s["table"], s["lens"], s["pool"].shape[3]
    r = rows.long()
    new = torch.minimum(keep, lens[r])
    col = torch.arange(table.shape[1], device=r.device)
    mine = table[r]
    drop = (col >= ((new + pl - 1) // pl)[:, None]) & (mine >= 0)
    refs -= _count(mine.long().clamp(min=0).view(-1), drop.view(-1), refs.numel())
    table[r] = mine.masked_fill(drop, -1)
    lens[r] = new
    return torch.zeros(1, dtype=torch.int32, device=refs.device)


def _plain_branch(s):
    forked = _plain_fork(s)
    status = _plain_extend(s, s["dst"], s["add"])
    return dict(pool=s["pool"], refs=s["refs"], table=s["table"], lens=s["lens"], batch=list(s["out"]), forked=forked,
                status=status)


def _plain_step(s):
    status = _plain_extend(s, s["rows"], s["add"])
    back = _plain_truncate(s, s["rows"], s["keep"])
    return dict(pool=s["pool"], refs=s["refs"], table=s["table"], lens=s["lens"], batch=list(s["out"]), status=status,
                back=back)


def _plain_compact(s):
    pool, refs, table = s["pool"], s["refs"], s["table"]
    live = refs > 0
    n = live.sum()
    index = torch.arange(refs.numel(), device=refs.device)
    holes = (~live & (index < n)).nonzero().view(-1)
    movers = (live & (index >= n)).nonzero().view(-1)
    to = torch.where(live, index, -1)
    to[movers] = holes
    pool[:, holes] = pool[:, movers]
    new_refs = torch.zeros_like(refs)
    new_refs[to[live]] = refs[live]
    new_table = torch.where(table >= 0, to[table.long().clamp(min=0)].int(), -1)
    return dict(pool=pool, refs=new_refs, table=new_table, map=to.int(),
                counts=torch.stack([n, (holes >= 0).sum()]).int())


_PLAIN = {"attend": _plain_attend, "branch": _plain_branch, "step": _plain_step, "compact": _plain_compact}


# ------------------------------------------------------------------- work
def work(case):
    es = DTYPES[case["dtype"]].itemsize
    pl, D, Hkv = case["pl"], case["D"], case["Hkv"]
    if case["op"] == "attend":
        starts, shared, own_prefix, rows = _attend_shapes(case)
        T, words = sum(rows), (max(rows) + 63) // 64
        kv = 2 * Hkv * D * es * (sum(shared) * pl + sum(own_prefix) + T)
        ints = 4 * (sum(shared) + sum(_pages_of(o + n, pl) for o, n in zip(own_prefix, rows))) + 8 * words * T
        pairs = 0
        for g in range(case["groups"]):
            for b in range(starts[g], starts[g + 1]):
                pairs += rows[b] * (shared[g] * pl + own_prefix[b])
        for parents in _trees(case):
            depth = []
            for p in parents:
                depth.append(depth[p] + 1 if p >= 0 else 1)
            pairs += sum(depth)
        return {"bytes": kv + 2 * T * case["Hq"] * D * es + ints, "flops": 4.0 * D * case["Hq"] * pairs}
    row = case.get("layers", 1) * 2 * Hkv * D * es                            # bytes of one token in every layer
    if case["op"] == "branch":
        lens, c = _lengths(case), case["children"]
        part = [n % pl for n in lens]
        mean_part, mean_pages = sum(part) / len(part), sum(_pages_of(n, pl) for n in lens) / len(lens)
        # the parents' partial pages are read once and written to every child; each child's table is
        # written and read for the batch's lists, its pages are counted, the pool's counts are searched
        return {"bytes": row * (sum(part) + c * mean_part) + 4 * (4 * c * mean_pages + 2 * case["pages"]), "flops": 0.0}
    if case["op"] == "step":
        pages = sum(_pages_of(n, pl) for n in _lengths(case))
        fresh = case["seqs"] * (case["add"] / pl)
        return {"bytes": 4 * (case["pages"] + 2 * pages + 6 * fresh), "flops": 0.0}
    live = sum(_pages_of(n, pl) for n in _lengths(case))
    moved = live * (1 - live / case["pages"])                                 # live pages past the live count
    table = (case["seqs"] + 1) * (_pages_of(case["length"], pl) + 1)
    return {"bytes": 2 * moved * pl * row + 4 * (3 * case["pages"] + 2 * table), "flops": 0.0}


# ------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["op"]](case, s)


def _exact_attend(case, s):
    """softmax(q K^T / sqrt(D)) V in fp64, request by request, over all its pages."""
    pl, Hkv, D = case["pl"], case["Hkv"], case["D"]
    qo, indptr, last = s["qo"].tolist(), s["indptr"].tolist(), s["last"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, parents in enumerate(_trees(case)):
        pages = s["indices"][indptr[b]:indptr[b + 1]].long()
        n, total = len(parents), (len(pages) - 1) * pl + last[b]
        mask = torch.ones(n, total, dtype=torch.bool)
        mask[:, total - n:] = False
        for i in range(n):
            j = i
            while j >= 0:
                mask[i, total - n + j] = True
                j = parents[j]
        mask = mask.to(DEV)
        x = s["kv"][pages].double()
        for h in range(Hkv):
            k, v = x[:, 0, :, h].reshape(-1, D)[:total], x[:, 1, :, h].reshape(-1, D)[:total]
            g = case["Hq"] // Hkv
            z = torch.einsum("ngd,ld->ngl", s["q"][qo[b]:qo[b + 1], h * g:(h + 1) * g].double(), k) / D ** 0.5
            z = z.masked_fill(~mask[:, None], float("-inf"))
            out[qo[b]:qo[b + 1], h * g:(h + 1) * g] = torch.einsum("ngl,ld->ngd", torch.softmax(z, -1), v)
    return out


class _Pages:
    """The page state as Python lists, changed one page at a time."""

    def __init__(self, s, pl):
        self.refs, self.table, self.pl = s["refs"].tolist(), s["table"].tolist(), pl
        self.lens = s["lens"].tolist() if "lens" in s else None

    def take(self):
        p = next(i for i in range(self.low, len(self.refs)) if self.refs[i] == 0)
        self.low = p
        self.refs[p] = 1
        return p

    def extend(self, rows, add, starts):
        self.low, B = 0, len(rows)
        old = [self.lens[r] for r in rows]
        tail = {}
        for i, r in enumerate(rows):
            if add > 0 and old[i] % self.pl:
                tail.setdefault(self.table[r][old[i] // self.pl], []).append(i)
        held = {p: self.refs[p] for p in tail}
        taken_from = {}
        for i, r in enumerate(rows):
            n, at = _pages_of(old[i], self.pl), old[i] // self.pl
            p = self.table[r][at] if add > 0 and old[i] % self.pl else None
            if p is not None and held[p] > 1 and not (len(tail[p]) == held[p] and tail[p][-1] == i):
                self.table[r][at] = self.take()
                taken_from[p] = taken_from.get(p, 0) + 1
            for j in range(n, _pages_of(old[i] + add, self.pl)):
                self.table[r][j] = self.take()
            self.lens[r] += add
        for p, k in taken_from.items():
            self.refs[p] -= k
        lists = [self.table[r][:_pages_of(self.lens[r], self.pl)] for r in rows]
        shared = []
        for a, z in zip(starts[:-1], starts[1:]):
            n = 0
            while all(n < old[i] // self.pl and lists[i][n] == lists[a][n] for i in range(a, z)):
                n += 1
            shared.append(n)
        self.lists, self.shared = lists, shared
        return B

    def batch(self, rows, like):
        flat = [p for x in self.lists for p in x]
        indptr = [0]
        for x in self.lists:
            indptr.append(indptr[-1] + len(x))
        lens = [self.lens[r] for r in rows]
        flat += [-1] * (like[1].numel() - len(flat))
        return [_i32(indptr), _i32(flat), _i32([(n - 1) % self.pl + 1 if n else 0 for n in lens]), _i32(lens),
                _i32(self.shared)]


def _exact_branch(case, s):
    p = _Pages(s, case["pl"])
    src, dst = s["src"].tolist(), s["dst"].tolist()
    for a, b in zip(src, dst):
        for x in p.table[a]:
            if x >= 0:
                p.refs[x] += 1
        p.table[b], p.lens[b] = list(p.table[a]), p.lens[a]
    p.extend(dst, case["add"], s["groups"].tolist())
    return dict(pool=None, refs=_i32(p.refs), table=_i32(p.table), lens=_i32(p.lens), batch=p.batch(dst, s["out"]),
                forked=_i32([0]), status=_i32([0]))


def _exact_step(case, s):
    p, rows = _Pages(s, case["pl"]), s["rows"].tolist()
    before = dict(refs=s["refs"].clone(), table=s["table"].clone(), lens=s["lens"].clone())
    p.extend(rows, case["add"], s["groups"].tolist())
    return dict(pool=None, batch=p.batch(rows, s["out"]), status=_i32([0]), back=_i32([0]), **before)


def _exact_compact(case, s):
    p = _Pages(s, case["pl"])
    live = [i for i, r in enumerate(p.refs) if r]
    n = len(live)
    holes = iter([i for i in range(n) if not p.refs[i]])
    to = {i: (i if i < n else next(holes)) for i in live}
    refs = [0] * len(p.refs)
    for i in live:
        refs[to[i]] = p.refs[i]
    return dict(pool=None, refs=_i32(refs), table=_i32([[to.get(x, -1) for x in row] for row in p.table]),
                map=_i32([to.get(i, -1) for i in range(len(refs))]),
                counts=_i32([n, sum(i != j for i, j in to.items())]))


_EXACT = {"attend": _exact_attend, "branch": _exact_branch, "step": _exact_step, "compact": _exact_compact}
