"""Paged KV cache manager, interface of the reference's ``flashinfer/cache_manager.py``.

``KvCachePool`` / ``RequestKvCache`` / ``KvCacheBatchPosition`` /
``getKvCacheBatchPosition`` keep the reference's constructors, attributes and
tensor layout (``cache_data[L, max_pages, 2, page_len, Hkv, D]``, host-side
free-page mask with first-fit allocation, ``cache_manager.py:23-213``).  The
device work goes through libpts_b200:

* ``getKvCacheBatchPosition`` computes append batch indices / positions with
  ``pts_batch_positions``, one append segment per request (the reference
  builds a single segment, ``cache_manager.py:263-271``, which is the same
  thing for one request);
* ``reorder_cache_with_offset`` moves only the accepted rows with
  ``pts_kv_compact`` instead of cloning the whole pool twice
  (``cache_manager.py:130-140``).  The pool-level method addresses flat
  physical slots like the reference; the request-level method follows the
  request's page table, which is identical whenever the request owns
  physical pages 0..n-1 in order (the only case in which the reference's
  flat-slot arithmetic addresses the request's own pages).

``SharedKvCache`` (no counterpart in the reference, whose requests share no pages)
keeps the page state of many sequences on the device, where they may share pages:
several samples of one prompt, beams, requests under one system prompt.
"""
from __future__ import annotations

import math
from itertools import accumulate
from typing import List, Optional, Sequence, Union

import numpy as np
import torch

from . import kernels as K


class KvCacheBatchPosition:
    """Batch descriptor (``cache_manager.py:23-48``).  Also keeps host copies
    of the per-request lengths so planning needs no device sync."""

    def __init__(self, seq_indptr, kv_page_indptr, kv_page_indices, kv_last_page_len, batch_indices, positions):
        self.seq_indptr = seq_indptr
        self.kv_page_indptr = kv_page_indptr
        self.kv_page_indices = kv_page_indices
        self.kv_last_page_len = kv_last_page_len
        self.batch_indices = batch_indices
        self.positions = positions
        self.host_qo_lens = None
        self.host_kv_lens = None
        # host_kv_lens are upper bounds, the lengths are on the device only (SharedKvCache)
        self.host_kv_bounds = False
        # requests that share leading pages (SharedKvCache.extend, beam_search): groups of
        # consecutive requests and each group's common pages, for tree_attention_shared
        self.group_indptr = None
        self.shared_pages = None
        self.max_own_len = None

    def print_info(self):
        for k in ("seq_indptr", "kv_page_indptr", "kv_page_indices", "kv_last_page_len", "batch_indices", "positions"):
            print(f"  {k + ':':<18}{getattr(self, k)}")


class KvCachePool:
    """Device pool of fixed-size pages (``cache_manager.py:51-140``)."""

    def __init__(self, max_pages: int, num_layers: int, num_heads: int, head_dim: int, page_len: int,
                 dtype: torch.dtype, device):
        self.cache_data = torch.zeros(num_layers, max_pages, 2, page_len, num_heads, head_dim, dtype=dtype,
                                      device=device)
        self.num_layers = num_layers
        self.device = device
        self.max_pages = max_pages
        self.page_len = page_len
        self.num_heads = num_heads
        self.head_dims = head_dim
        self.dtype = dtype
        self.free_page_mask = torch.ones(max_pages, dtype=torch.bool, device="cpu")
        self._identity_pages = None

    def reset(self):
        self.cache_data.zero_()
        self.free_page_mask.fill_(True)

    def num_free_pages(self):
        return self.free_page_mask.sum().item()

    def allocate(self, num_pages: int) -> List[int]:
        """First-fit allocation (``cache_manager.py:89-97``)."""
        free = self.free_page_mask.nonzero()
        assert len(free) >= num_pages, f"Out of cache pages: asked {num_pages}, only {len(free)} free"
        got = free[:num_pages]
        self.free_page_mask[got] = False
        return got.squeeze(1).tolist()

    def deallocate(self, kv_page_indices: List[int]):
        self.free_page_mask[kv_page_indices] = True

    def _compact(self, pages: List[int], beam_idx: torch.Tensor, base: int):
        dev = self.cache_data.device
        idx = torch.as_tensor(beam_idx, device=dev).to(torch.int32).reshape(1, -1)
        n = idx.shape[1]
        if n == 0:
            return
        if pages is None:
            if self._identity_pages is None:
                self._identity_pages = torch.arange(self.max_pages, dtype=torch.int32, device=dev)
            pidx = self._identity_pages
        else:
            pidx = torch.as_tensor(pages, dtype=torch.int32, device=dev)
        pind = torch.tensor([0, pidx.numel()], dtype=torch.int32, device=dev)
        counts = torch.tensor([n], dtype=torch.int32, device=dev)
        offs = torch.tensor([base], dtype=torch.int32, device=dev)
        K.kv_compact(self.cache_data, pind, pidx, idx, counts, offs)

    def reorder_cache_with_offset(self, beam_idx: torch.LongTensor, offset: int = 0, num_new_tokens: int = 0):
        """Flat physical slot ``offset + beam_idx[i]`` -> ``offset + i`` in every
        layer, K and V (``cache_manager.py:103-140``)."""
        self._compact(None, beam_idx, offset)


class RequestKvCache:
    """Per-request page list and length (``cache_manager.py:143-213``)."""

    def __init__(self, kvCachePool: KvCachePool, page_len: int, seq_init_len: int):
        self.kvCachePool = kvCachePool
        self.page_len = page_len
        n = math.ceil(seq_init_len / page_len) if seq_init_len > 0 else 0
        self.kv_last_page_len = seq_init_len - (n - 1) * page_len if n > 0 else 0
        self.kv_page_indices = kvCachePool.allocate(n) if n > 0 else []
        self.kv_len = seq_init_len
        self.is_released = False

    def get_seq_length(self):
        return self.kv_len

    def increment(self, num_tokens: int = 1):
        if num_tokens <= 0:
            return
        if len(self.kv_page_indices) == 0:
            self.kv_page_indices.extend(self.kvCachePool.allocate(1))
            self.kv_last_page_len = 0
        self.kv_len += num_tokens
        self.kv_last_page_len += num_tokens
        while self.kv_last_page_len > self.page_len:
            self.kv_last_page_len -= self.page_len
            self.kv_page_indices.extend(self.kvCachePool.allocate(1))

    def decrement(self, num_tokens: int = 1):
        if num_tokens <= 0:
            return
        num_tokens = min(num_tokens, self.kv_len)
        self.kv_len -= num_tokens
        need = math.ceil(self.kv_len / self.page_len) if self.kv_len > 0 else 0
        while len(self.kv_page_indices) > need:
            self.kvCachePool.deallocate([self.kv_page_indices.pop()])
        self.kv_last_page_len = 0 if self.kv_len == 0 else (self.kv_len - 1) % self.page_len + 1

    def release(self):
        if not self.is_released:
            self.kvCachePool.deallocate(self.kv_page_indices)
            self.is_released = True

    def reorder_cache_with_offset(self, beam_idx: torch.LongTensor, offset: int = 0, num_new_tokens: int = 0):
        """Keep the accepted rows: slot ``offset-1 + beam_idx[i]`` ->
        ``offset-1 + i`` through this request's page table, then truncate."""
        if offset != 0:
            offset -= 1
        self.kvCachePool._compact(self.kv_page_indices, beam_idx, offset)
        self.kv_len = offset + int(torch.as_tensor(beam_idx).numel())
        self.kv_last_page_len = 0 if self.kv_len == 0 else (self.kv_len - 1) % self.page_len + 1
        need = math.ceil(self.kv_len / self.page_len) if self.kv_len > 0 else 0
        if len(self.kv_page_indices) > need:
            self.kvCachePool.deallocate(self.kv_page_indices[need:])
            self.kv_page_indices = self.kv_page_indices[:need]


def getKvCacheBatchPosition(request_kv_caches: List[RequestKvCache], mode: str, device,
                            treeTokens: int = 0) -> KvCacheBatchPosition:
    """Batch descriptor for ``mode`` in {"prefill", "decode", "tree"}
    (``cache_manager.py:216-280``)."""
    pages, page_indptr, seq_indptr, last, kv_lens, app = [], [0], [0], [], [], []
    for r in request_kv_caches:
        pages.extend(r.kv_page_indices)
        page_indptr.append(page_indptr[-1] + len(r.kv_page_indices))
        last.append(r.kv_last_page_len)
        kv_lens.append(r.kv_len)
        if mode == "prefill":
            n = r.kv_len
        elif mode == "decode":
            n = 1
        elif mode == "tree":
            n = treeTokens
        else:
            raise ValueError(f"Invalid mode: {mode}")
        app.append(n)
        seq_indptr.append(seq_indptr[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    seq = i32(seq_indptr)
    bp = KvCacheBatchPosition(seq, i32(page_indptr), i32(pages), i32(last), None, None)
    bp.batch_indices, bp.positions = K.batch_positions(seq, i32(kv_lens), seq_indptr[-1])
    bp.host_qo_lens = app
    bp.host_kv_lens = kv_lens
    return bp


class SharedKvCache:
    """Sequences over a ``KvCachePool`` that share pages, their page state (counts of
    holders, page tables, lengths) on the device.

    ``fork`` makes a sequence hold another's pages without moving K/V; ``extend`` makes
    room for new tokens, copying a partial last page that others hold too, and returns the
    batch position for the append and the attention, with each group's common pages;
    ``truncate`` and ``release`` give pages back; ``compact`` closes the pool's gaps.  Rows
    (sequence numbers) and lengths may be lists or int32 tensors on the pool's device;
    with tensors (and one int for all rows in ``extend``) no call copies from the host or
    waits for it, so a step can be captured in a CUDA graph, ``compact`` too.  A call that
    cannot be done changes nothing (the batch position of such an ``extend`` has
    empty sequences, so an append to it writes nothing); ``check`` raises for it.  The
    cache takes all pages of the pool, which must be free, until ``close``.

    The host keeps bounds of the lengths for the attention's schedule: exact for lists (of
    calls that could be done); device rows raise every sequence's bound and device
    truncations lower none, so a loop of such calls should ask for ``lengths`` now and then
    (small calls run in one launch only while their bounds are short).  Tokens after the
    shared pages are not bounded: decoding is scheduled as by ``tree_attention_shared``
    without ``max_own_len``."""

    def __init__(self, pool: KvCachePool, max_sequences: int, max_pages_per_sequence: int):
        if pool.num_free_pages() != pool.max_pages:
            raise ValueError("the pool's pages must all be free")
        self.pool = pool
        self._held = pool.allocate(pool.max_pages)
        dev = pool.cache_data.device
        self.page_refs = torch.zeros(pool.max_pages, dtype=torch.int32, device=dev)
        self.page_table = torch.full((max_sequences, max_pages_per_sequence), -1, dtype=torch.int32, device=dev)
        self.kv_lens = torch.zeros(max_sequences, dtype=torch.int32, device=dev)
        self._bound = [0] * max_sequences                 # upper bounds of the lengths, for schedules only
        self._status = torch.zeros(1, dtype=torch.int32, device=dev)       # the last call's
        self._failures = torch.zeros(1, dtype=torch.int32, device=dev)     # of all calls and replays since the last check

    def _ints(self, x) -> torch.Tensor:
        if isinstance(x, torch.Tensor):
            return x
        return torch.tensor(list(x), dtype=torch.int32, device=self.page_refs.device)

    def _limit(self) -> int:
        return self.page_table.shape[1] * self.pool.page_len

    def fork(self, src_rows, dst_rows) -> None:
        """``dst_rows[i]`` becomes a fork of ``src_rows[i]`` (all read before any is
        written; the destinations' former pages are given back)."""
        K.cache_fork(self.page_refs, self.page_table, self.kv_lens, self._ints(src_rows), self._ints(dst_rows),
                     self._status, self._failures)
        if isinstance(src_rows, torch.Tensor) or isinstance(dst_rows, torch.Tensor):
            self._bound = [max(self._bound)] * len(self._bound)
        else:
            old = list(self._bound)
            for a, b in zip(src_rows, dst_rows):
                if 0 <= a < len(old) and 0 <= b < len(old):
                    self._bound[b] = old[a]

    def extend(self, rows, add: Union[int, Sequence[int]], groups: Optional[Sequence[int]] = None) -> KvCacheBatchPosition:
        """Room for ``add`` more tokens (an int, or one per row) in every listed sequence.
        Returns the batch position of these rows: append positions of the new tokens, page
        lists, and for ``groups`` (starts of consecutive groups of the listed rows and
        their number at the end, by default one group of all) the pages that each group's
        rows hold in common."""
        r = self._ints(rows)
        B = r.numel()
        adds = [int(add)] * B if isinstance(add, int) else [int(n) for n in add]
        if len(adds) != B:
            raise ValueError(f"add has {len(adds)} entries, expected {B}")
        if not adds or min(adds) < 0:
            raise ValueError("add is empty or negative")
        dev = self.page_refs.device
        up_to = lambda n: torch.arange(n, dtype=torch.int32, device=dev)    # (made there: nothing is copied)
        if min(adds) == max(adds):
            each, seq = adds[0], up_to(B + 1) * adds[0]
        else:
            each, seq = self._ints(adds), self._ints(accumulate(adds, initial=0))
        gi = up_to(2) * B if groups is None else self._ints(groups)
        out = K.cache_extend(self.pool.cache_data, self.page_refs, self.page_table, self.kv_lens, r, each, group_indptr=gi,
                             status=self._status, failures=self._failures)
        bp = KvCacheBatchPosition(seq, out.page_indptr, out.page_indices, out.last_page_len, None, None)
        bp.batch_indices, bp.positions = K.batch_positions(seq, out.seq_lens, sum(adds)) if any(adds) else (up_to(0), up_to(0))
        if isinstance(rows, torch.Tensor):
            top = max(self._bound) + max(adds)
            self._bound = [min(top, self._limit())] * len(self._bound)
            lens = [self._bound[0]] * B
        else:
            for row, n in zip(rows, adds):
                if 0 <= row < len(self._bound):
                    self._bound[row] = min(self._bound[row] + n, self._limit())
            lens = [self._bound[row] if 0 <= row < len(self._bound) else 0 for row in rows]
        bp.host_qo_lens, bp.host_kv_lens, bp.host_kv_bounds = adds, [max(1, n) for n in lens], True
        bp.group_indptr, bp.shared_pages = gi, out.shared_pages
        return bp

    def truncate(self, rows, new_lens=None) -> None:
        """Cut the listed sequences to ``new_lens`` tokens (None: free them)."""
        K.cache_truncate(self.page_refs, self.page_table, self.kv_lens, self.pool.page_len, self._ints(rows),
                         None if new_lens is None else self._ints(new_lens), self._status, self._failures)
        if not isinstance(rows, torch.Tensor) and not isinstance(new_lens, torch.Tensor):
            for i, row in enumerate(rows):
                if 0 <= row < len(self._bound):
                    self._bound[row] = min(self._bound[row], max(0, new_lens[i]) if new_lens is not None else 0)

    def release(self, rows) -> None:
        self.truncate(rows)

    def compact(self) -> torch.Tensor:
        """Close the pool's gaps; returns the map from old to new page (-1: free).  Batch
        positions from before name the old pages; captured steps of this class stay valid
        (the state's tensors stay where they are)."""
        r = K.cache_compact(self.pool.cache_data, self.page_refs, self.page_table)
        self.page_refs.copy_(r.page_refs)
        self.page_table.copy_(r.page_table)
        return r.page_map

    def lengths(self) -> List[int]:
        """The lengths, read from the device (they then also bound the schedules)."""
        self._bound = self.kv_lens.tolist()
        return list(self._bound)

    def check(self) -> None:
        """Raise for a call, or a replay of a captured one, since the last check that could
        not be done (waits for the current stream)."""
        code = int(self._failures.item())
        if code:
            self._failures.zero_()
            K.raise_cache_status(code)

    def close(self) -> None:
        """Give the pool's pages back; the sequences are gone."""
        if self._held:
            self.pool.deallocate(self._held)
            self._held = []
