"""Host side of ``SharedKvCache``, with the kernels replaced by recording stand-ins."""
import torch

from parallel_tree_spec_b200 import kernels as K
from parallel_tree_spec_b200.cache_manager import KvCachePool, SharedKvCache


def _cache(pages=6, rows=3, width=4):
    return SharedKvCache(KvCachePool(pages, 1, 1, 8, 4, torch.float32, torch.device("cpu")), rows, width)


def test_compact_keeps_the_state_where_it_is(monkeypatch):
    """A captured step holds the addresses of the counts and of the table: a compaction
    writes the new values into the same tensors."""
    cache = _cache()
    refs, table = torch.arange(6, dtype=torch.int32), torch.arange(12, dtype=torch.int32).view(3, 4)
    moved = torch.tensor([2, 0, 1, -1, -1, -1], dtype=torch.int32)
    monkeypatch.setattr(K, "cache_compact", lambda *a: K.CompactedCache(refs, table, moved, torch.tensor([3, 1])))
    before = cache.page_refs, cache.page_table
    at = [t.data_ptr() for t in before]
    assert cache.compact() is moved
    assert cache.page_refs is before[0] and cache.page_table is before[1]
    assert [cache.page_refs.data_ptr(), cache.page_table.data_ptr()] == at
    assert torch.equal(cache.page_refs, refs) and torch.equal(cache.page_table, table)
