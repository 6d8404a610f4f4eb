"""PagedKVRunner on the 8-bit cache: prompts, decode steps with page weights, eviction and what follows, against the
definitions in 64 bits (fp8_util)."""
import types

import numpy as np
import pytest
import torch

import oracle
from fp8_util import RefCache, attend, check, evict_ref, gather
from gpu_util import say
from infurnace_amd.kernels import rope_table
from infurnace_amd.runner import PagedKVRunner, RunnerError

pytestmark = pytest.mark.gpu

L, SLOTS, HQ, HKV, D = 2, 5, 4, 2, 64


class Engine:
    """A runner and the definition beside it."""

    def __init__(self, dev, blocks=90, context=512, **kw):
        self.dev = dev
        self.run = PagedKVRunner(L, SLOTS, context, HKV, D, blocks, device=dev, kv_dtype="float8_e4m3fn", **kw)
        self.ref = [RefCache(blocks, HKV, D) for _ in range(L)]
        self.gen = torch.Generator().manual_seed(blocks)
        self.weights = torch.zeros((SLOTS, HKV, self.run.max_pages), dtype=torch.float64)

    def rows(self, t, h):
        return torch.randn((t, h, D), generator=self.gen).half()

    def prefill(self, slot, n):
        start = self.run.position(slot)
        step = self.run.begin_prefill(slot, start, n)
        first = self.run.length(slot) - n
        for i in range(L):
            q, k, v = self.rows(n, HQ), self.rows(n, HKV), self.rows(n, HKV)
            o = step.store_attend(i, q.to(self.dev), k.to(self.dev), v.to(self.dev))
            self.ref[i].store(step.slot_mapping.tolist(), k, v)
            kk, vv = gather(self.ref[i].values(), self.run._table([slot])[0], first + n)
            out, tol, _, _ = attend(q, kk, vv, first + 1 + torch.arange(n))
            check(o, out, tol, f"prefill layer {i}")

    def decode(self, slots, active=None):
        active = [True] * len(slots) if active is None else active
        pos = [self.run.position(s) for s in slots]
        plan = types.SimpleNamespace(slots=tuple(slots), positions=tuple(pos), active_mask=tuple(active))
        step = self.run.begin_decode(plan)
        for i in range(L):
            q, k, v = self.rows(len(slots), HQ), self.rows(len(slots), HKV), self.rows(len(slots), HKV)
            o = step.store_attend(i, q.to(self.dev), k.to(self.dev), v.to(self.dev))
            self.ref[i].store(step.slot_mapping.tolist(), k, v)
            for r, s in enumerate(slots):
                if not active[r]:
                    assert not o[r].any()
                    continue
                n = self.run.length(s)
                kk, vv = gather(self.ref[i].values(), self.run._table([s])[0], n)
                out, tol, w, _ = attend(q[r:r + 1], kk, vv, [n])
                check(o[r:r + 1], out, tol, f"decode layer {i} slot {s}")
                pad = torch.zeros((HKV, -(-n // 16) * 16), dtype=torch.float64)
                pad[:, :n] = w
                self.weights[s, :, :pad.shape[1] // 16] += pad.unflatten(-1, (-1, 16)).sum(-1)

    def caches_agree(self):
        for i in range(L):
            self.ref[i].same(*self.run.cache.layer(i))


def test_serving_with_eviction(dev):
    say("runner fp8 serving")
    e = Engine(dev, track_page_weights=True)
    run = e.run
    for s, n in enumerate((200, 33, 100, 16)):
        e.prefill(s, n)
    e.prefill(0, 47)  # a second chunk, from inside a page
    for step in range(5):
        e.decode([0, 1, 2, 3], [True, step != 2, True, True])
    e.caches_agree()
    run.synchronize()
    assert torch.allclose(run.page_weights.cpu().double(), e.weights, rtol=1e-4, atol=1e-6)
    # two slots over eight pages
    held = run.page_weights.cpu().numpy()
    lens = np.array([run.length(s) for s in range(4)], np.int32)
    exp = evict_ref(run._table(range(4)), lens, held[:4].copy(), 8, 1, 2)
    free = run.pool.num_free
    freed = run.evict(8, sink_pages=1, recent_pages=2)
    run.synchronize()
    assert run.pool.num_free == free + int(exp[3].sum()) and len(freed) == int(exp[3].sum())
    for s in range(4):
        n = -(-int(exp[1][s]) // 16)
        assert run.length(s) == exp[1][s] and run.mgr.blocks(s) == exp[0][s, :n].tolist()
        assert run.position(s) == lens[s] and run._evicted.get(s, 0) == 16 * exp[3][s]
    assert np.array_equal(run.page_weights.cpu().numpy()[:4], np.where(exp[3][:, None, None] > 0, exp[2], held[:4]))
    e.weights = run.page_weights.cpu().double()
    # and on: decode, another chunk, decode
    for _ in range(3):
        e.decode([2, 0, 3])
    e.prefill(0, 70)
    e.decode([0, 1, 2, 3])
    e.caches_agree()
    run.synchronize()
    assert torch.allclose(run.page_weights.cpu().double(), e.weights, rtol=1e-4, atol=1e-6)
    with pytest.raises(RunnerError):
        run.begin_decode(types.SimpleNamespace(slots=(0,), positions=(run.length(0),), active_mask=(True,)))
    run.clear_slot(0)
    assert run.position(0) == 0 and not run.page_weights[0].any()
    e.prefill(0, 20)  # its pages are others' old ones
    e.decode([0, 2])
    run.synchronize()


def test_steps_on_other_streams(dev):
    """Steps on streams of their own, closed, cleared and evicted from another: the same weights and tables."""
    say("runner fp8 streams")
    e = Engine(dev, track_page_weights=True)
    run = e.run
    side = [torch.cuda.Stream() for _ in range(2)]
    for i, (s, n) in enumerate(((0, 200), (1, 90))):
        with torch.cuda.stream(side[i]):
            e.prefill(s, n)
    torch.cuda.synchronize()
    for step in range(4):
        with torch.cuda.stream(side[step % 2]):
            e.decode([0, 1])
    run.evict(6, recent_pages=2)
    assert len(run.mgr.blocks(0)) == 6 and len(run.mgr.blocks(1)) == 6
    run.synchronize()
    for s, had in ((0, 13), (1, 6)):
        w = e.weights[s, :, :had]
        if had > 6:
            assert torch.all(run.page_weights[s, :, 6:] == 0)
            assert torch.all(run.page_weights[s].cpu().double().sum(-1) < w.sum(-1) + 1e-6)
        else:
            assert torch.allclose(run.page_weights[s, :, :had].cpu().double(), w, rtol=1e-4, atol=1e-6)
    e.weights = run.page_weights.cpu().double()
    with torch.cuda.stream(side[0]):
        e.decode([0, 1])
    run.clear_slot(1)
    torch.cuda.synchronize()
    assert not run.page_weights[1].any()
    assert torch.allclose(run.page_weights[0].cpu().double(), e.weights[0], rtol=1e-4, atol=1e-6)
    e.caches_agree()


def test_prefix_sharing_and_eviction(dev):
    """An evicted shared page stays the prefix cache's; an evicted slot publishes nothing."""
    say("runner fp8 prefix")
    e = Engine(dev, track_page_weights=True, prefix_namespace=("m", "fp8"))
    run = e.run
    prompt = list(range(130))
    run.attach_prefix(0, prompt)
    e.prefill(0, 130)
    run.publish_prefix(0, prompt)
    n = run.attach_prefix(1, prompt)
    assert n == 128
    e.prefill(1, 2)
    e.decode([0, 1])
    common = run.mgr.blocks(1)[:8]
    run.evict(3, slots=[1])
    run.synchronize()
    assert run.mgr.blocks(0)[:8] == common and all(run.pool.refcount(p) > 0 for p in common)
    with pytest.raises(RunnerError):
        run.publish_prefix(1, prompt[:32])
    e.decode([0, 1])
    assert run.attach_prefix(2, prompt) == 128
    run.synchronize()


def test_prepared_rows(dev):
    """From fp32 projections: the pre-append's fp16 rows, stored in 8 bits (the fp16 rows from the oracle's pre-append)."""
    say("runner fp8 prep")
    rng = np.random.default_rng(5)
    run = PagedKVRunner(1, 2, 128, HKV, D, 20, device=dev, kv_dtype="float8_e4m3fn")
    ref = RefCache(20, HKV, D)
    rope = rope_table(128, D, 1e4)
    qw, kw = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32), (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731

    def prep(n, pos):
        q, k, v = (rng.standard_normal((n, h, D)).astype(np.float32) for h in (HQ, HKV, HKV))
        pool = np.zeros((2, -(-n // 16), 16, HKV, D), np.float16)
        q16 = oracle.qk_norm_rope_append(q, k, v, qw, kw, rope.numpy(), pos.astype(np.int32), np.arange(n, dtype=np.int32),
                                         None, pool)
        flat = pool.reshape(2, -1, HKV, D)[:, :n]
        return (q, k, v), torch.from_numpy(q16), torch.from_numpy(flat[0].copy()), torch.from_numpy(flat[1].copy())

    step = run.begin_prefill(0, 0, 37)
    (q, k, v), q16, k16, v16 = prep(37, np.arange(37))
    o = step.prep_store_attend(0, t(q), t(k), t(v), t(qw), t(kw), rope.to(dev))
    ref.store(step.slot_mapping.tolist(), k16, v16)
    kk, vv = gather(ref.values(), run._table([0])[0], 37)
    out, tol, _, _ = attend(q16, kk, vv, 1 + torch.arange(37))
    # (the oracle's fp16 rows and the kernel's may differ in the last bit: a code step, 2^-4, of a few values)
    assert torch.allclose(o.cpu().double(), out, atol=2e-2, rtol=2e-2)
    step = run.begin_decode(types.SimpleNamespace(slots=(1, 0), positions=(0, 37), active_mask=(False, True)))
    (q, k, v), q16, k16, v16 = prep(2, np.array([0, 37]))
    o = step.prep_store_attend(0, t(q), t(k), t(v), t(qw), t(kw), rope.to(dev))
    ref.store(step.slot_mapping.tolist(), k16, v16)
    kk, vv = gather(ref.values(), run._table([0])[0], 38)
    out, tol, _, _ = attend(q16[1:], kk, vv, [38])
    assert torch.allclose(o[1:].cpu().double(), out, atol=2e-2, rtol=2e-2) and not o[0].any()
    run.synchronize()


def test_clear_and_copy_pages(dev):
    say("cache fp8 pages")
    from infurnace_amd.cache import PagedKVCacheFP8
    c = PagedKVCacheFP8(2, 12, HKV, D, device=dev)
    c.kv.view(torch.uint8).copy_(torch.randint(0, 120, c.kv.shape, device=dev, dtype=torch.uint8))
    c.scales.copy_(2.0 ** torch.randint(-8, 3, c.scales.shape, device=dev).float())
    kv, sc = c.kv.view(torch.uint8).clone(), c.scales.clone()
    c.copy_pages([3, 5], [7, 1])
    c.clear_pages([9, 0])
    kv[:, :, [7, 1]], sc[:, :, [7, 1]] = kv[:, :, [3, 5]], sc[:, :, [3, 5]]
    kv[:, :, [9, 0]], sc[:, :, [9, 0]] = 0, 2.0 ** -32
    assert torch.equal(c.kv.view(torch.uint8), kv) and torch.equal(c.scales, sc)
