"""Host side of the 8-bit cache: its class, dropped pages of a sequence, and the runner's refusals (CPU)."""
import numpy as np
import pytest
import torch

from infurnace_amd.cache import BlockPool, KVCacheError, KVManager, PagedKVCacheFP8
from infurnace_amd.runner import PagedKVRunner, RunnerError


def test_cache_class():
    c = PagedKVCacheFP8(3, 10, 2, 64, device="cpu")
    assert c.shape == (3, 2, 10, 2, 16, 64) and c.kv.dtype == torch.float8_e4m3fn
    assert tuple(c.scales.shape) == (3, 2, 10, 2) and bool((c.scales == 2.0 ** -32).all())
    assert c.page_bytes == 2 * 2 * (16 * 64 + 4) and c.size_bytes == 3 * 10 * c.page_bytes
    c.kv[1].view(torch.uint8)[1, 4, 1, 3, 5] = 0x40  # 2.0
    c.scales[1, 1, 4, 1] = 0.25
    v = c.values(1, [7, 4])
    assert v.shape == (2, 2, 16, 2, 64) and v.dtype == torch.float16
    assert float(v[1, 1, 3, 1, 5]) == 0.5 and int((v != 0).sum()) == 1
    for kw in (dict(block_size=32), dict(head_dim=96), dict(num_kv_heads=0), dict(num_blocks=0)):
        with pytest.raises(KVCacheError):
            PagedKVCacheFP8(**{**dict(num_layers=1, num_blocks=4, num_kv_heads=1, head_dim=64, device="cpu"), **kw})
    with pytest.raises(KVCacheError):
        c.clear_pages([10])
    with pytest.raises(KVCacheError):
        c.copy_pages([1, 2], [3])


def test_evict_blocks():
    pool = BlockPool(32, 16)
    mgr = KVManager(pool)
    shared = pool.allocate(3, owner="prefix")
    mgr.add_sequence("a", prefix_blocks=shared, prefix_len=48)
    mgr.append("a", 70)  # 118 tokens: 3 borrowed and 5 own pages, the last with 6
    before = mgr.blocks("a")
    with pytest.raises(KVCacheError):
        mgr.evict_blocks("a", [7])  # not full
    with pytest.raises(KVCacheError):
        mgr.evict_blocks("a", [1, 1])
    with pytest.raises(KVCacheError):
        mgr.evict_blocks("a", [-1])
    assert mgr.blocks("a") == before
    freed = mgr.evict_blocks("a", [5, 1])
    assert freed == [before[5]]  # (the borrowed page stays the prefix cache's)
    assert mgr.blocks("a") == [before[i] for i in (0, 2, 3, 4, 6, 7)] and mgr.length("a") == 118 - 32
    slots = mgr.append("a", 12)  # fills the last page and starts the next
    assert slots[:10].tolist() == [before[7] * 16 + o for o in range(6, 16)] and len(mgr.blocks("a")) == 7
    with pytest.raises(KVCacheError):
        mgr.replace_blocks("a", [1])  # (two pages are still borrowed)
    mgr.free_sequence("a")
    pool.free(shared, owner="prefix")
    assert pool.num_free == 32 - (pool.dummy_block is not None)


def test_runner_refusals():
    args = (1, 4, 256, 2, 64, 40)
    with pytest.raises(RunnerError):
        PagedKVRunner(*args, device="cpu", kv_dtype="int8")
    with pytest.raises(RunnerError):
        PagedKVRunner(*args, device="cpu", track_page_weights=True)
    run = PagedKVRunner(*args, device="cpu", kv_dtype="float8_e4m3fn")
    with pytest.raises(RunnerError):
        run.evict(4)
    run = PagedKVRunner(*args, device="cpu", kv_dtype="float8_e4m3fn", track_page_weights=True)
    for kw in (dict(keep_pages=1), dict(keep_pages=4, recent_pages=0), dict(keep_pages=4, sink_pages=-1),
               dict(keep_pages=4, slots=[4]), dict(keep_pages=4, slots=[1, 1])):
        with pytest.raises(RunnerError):
            run.evict(**kw)
    run.begin_prefill(2, 0, 30)
    assert run.evict(2) == [] and run.position(2) == 30
    assert np.array_equal(run.page_weights.numpy(), np.zeros((4, 2, 16)))
