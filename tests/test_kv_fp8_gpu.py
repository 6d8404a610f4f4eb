"""The 8-bit KV cache on the GPU against its definition in 64 bits (fp8_util)."""
import numpy as np
import pytest
import torch

from fp8_util import EMPTY, F8, RefCache, attend, check, gather, random_cache, tables
from gpu_util import say
from infurnace_amd.kernels import DeviceArray, evict_pages, paged_attention_fp8, store_kv_fp8, store_kv_fp8_and_decode

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.as_tensor(np.asarray(x, np.int32)).to(dev)


def rows(gen, t, hkv, d, size=1.0):
    return (size * torch.randn((t, hkv, d), generator=gen)).half()


# ---- append ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("hkv,d", [(8, 128), (3, 64), (2, 256), (1, 128)])
def test_append_token_by_token(dev, hkv, d):
    """A page filled one token at a time: the scale grows with the rows, earlier codes are rounded to it."""
    say(f"append tokens hkv={hkv} d={d}")
    gen = torch.Generator().manual_seed(d + hkv)
    ref = RefCache(5, hkv, d)
    kv, sc = ref.to(dev)
    for t in range(40):  # page 3, then 1, then 3 anew
        slot = (3, 1, 3)[t // 16] * 16 + t % 16
        k, v = rows(gen, 1, hkv, d, 2.0 ** (t % 7 - 3)), rows(gen, 1, hkv, d, 4.0 ** (t % 5))
        store_kv_fp8(kv, sc, i32([slot], dev), None, k.to(dev), v.to(dev))
        ref.store([slot], k, v)
    ref.same(kv, sc)


@pytest.mark.parametrize("hkv,d", [(8, 128), (4, 64), (2, 256)])
@pytest.mark.parametrize("t,start", [(1, 0), (2, 15), (33, 7), (333, 727), (1023, 1), (1024, 0), (1500, 9)])
def test_append_chunks(dev, hkv, d, t, start):
    say(f"append chunk hkv={hkv} d={d} t={t} start={start}")
    gen = torch.Generator().manual_seed(t * 7 + start)
    pages = -(-(start + t) // 16)
    order = torch.randperm(pages + 3, generator=gen)
    ref = random_cache(pages + 3, hkv, d, t)
    kv, sc = ref.to(dev)
    pos = torch.arange(start, start + t)
    slots = (order[pos // 16] * 16 + pos % 16).tolist()
    k, v = rows(gen, t, hkv, d, 3.0), rows(gen, t, hkv, d)
    store_kv_fp8(kv, sc, i32(slots, dev), None, k.to(dev), v.to(dev), validate=True)
    ref.store(slots, k, v)
    ref.same(kv, sc)


@pytest.mark.parametrize("n", [70, 1100])
def test_append_masks_order_and_strangers(dev, n):
    """Inactive rows, slots outside the pool, a page's tokens out of order and apart, two rows with one slot: the later."""
    say(f"append order n={n}")
    rng = np.random.default_rng(n)
    gen = torch.Generator().manual_seed(n)
    pages = 80
    ref = random_cache(pages, 2, 64, n)
    kv, sc = ref.to(dev)
    slots = np.full(n, -1, np.int64)
    for i, p in enumerate(rng.permutation(pages)[:n // 48]):  # each page's tokens within 48 entries
        at = 48 * i + rng.permutation(48)[:12]
        slots[at] = p * 16 + rng.integers(0, 16, 12)
    strange = np.flatnonzero(slots < 0)
    slots[strange] = rng.choice([-1, -2 ** 31, pages * 16, pages * 16 + 5, 2 ** 31 - 1], len(strange))
    active = rng.random(n) < 0.8
    k, v = rows(gen, n, 2, 64), rows(gen, n, 2, 64, 20.0)
    store_kv_fp8(kv, sc, i32(slots, dev), torch.as_tensor(active).to(dev), k.to(dev), v.to(dev))
    ref.store(slots.tolist(), k, v, active)
    ref.same(kv, sc)


@pytest.mark.parametrize("hkv,d", [(2, 64), (8, 128), (1, 256)])
@pytest.mark.parametrize("n,start", [(30, 0), (300, 5), (1000, 0), (3001, 11)])
def test_append_masked_chunk(dev, hkv, d, n, start):
    """A chunk in order with rows masked out of its middle."""
    say(f"append masked chunk hkv={hkv} d={d} n={n} start={start}")
    rng = np.random.default_rng(n)
    gen = torch.Generator().manual_seed(n + d)
    pages = (start + n + 15) // 16
    ref = random_cache(pages, hkv, d, n)
    kv, sc = ref.to(dev)
    slots = np.arange(start, start + n)
    active = rng.random(n) < 0.9
    k, v = rows(gen, n, hkv, d), rows(gen, n, hkv, d, 20.0)
    store_kv_fp8(kv, sc, i32(slots, dev), torch.as_tensor(active).to(dev), k.to(dev), v.to(dev), validate=True)
    ref.store(slots.tolist(), k, v, active)
    ref.same(kv, sc)


@pytest.mark.parametrize("hkv,d,seqs,each,start", [(2, 64, 65, 2, 3), (2, 128, 100, 16, 0), (1, 256, 70, 5, 12),
                                                   (8, 128, 300, 20, 0), (8, 64, 513, 3, 14)])
def test_append_position_major(dev, hkv, d, seqs, each, start):
    """A step of several tokens a sequence, every sequence's first, then every sequence's second: a page's tokens are
    `seqs` entries apart."""
    say(f"append position major hkv={hkv} d={d} seqs={seqs} each={each}")
    rng = np.random.default_rng(seqs)
    gen = torch.Generator().manual_seed(seqs)
    per = (start + each + 15) // 16
    ids = rng.permutation(seqs * per).reshape(seqs, per)
    ref = random_cache(seqs * per, hkv, d, seqs)
    kv, sc = ref.to(dev)
    pos = np.arange(start, start + each)
    slots = (ids[:, pos // 16] * 16 + pos % 16).T.reshape(-1)
    n = seqs * each
    k, v = rows(gen, n, hkv, d), rows(gen, n, hkv, d, 20.0)
    store_kv_fp8(kv, sc, i32(slots, dev), None, k.to(dev), v.to(dev), validate=True)
    ref.store(slots.tolist(), k, v)
    ref.same(kv, sc)


@pytest.mark.parametrize("n", [200, 2500])
def test_append_any_order(dev, n):
    """Slots of a few pages in a random order over the whole call, inactive rows among them."""
    say(f"append any order n={n}")
    rng = np.random.default_rng(n)
    gen = torch.Generator().manual_seed(n)
    pages = 200
    ref = random_cache(pages, 4, 128, n)
    kv, sc = ref.to(dev)
    slots = rng.permutation(pages * 16)[:n]
    active = rng.random(n) < 0.7
    k, v = rows(gen, n, 4, 128, 20.0), rows(gen, n, 4, 128)
    store_kv_fp8(kv, sc, i32(slots, dev), torch.as_tensor(active).to(dev), k.to(dev), v.to(dev), validate=True)
    ref.store(slots.tolist(), k, v, active)
    ref.same(kv, sc)


def test_append_extremes(dev):
    """fp16's smallest and largest numbers, zeros, and the borders of a scale (448, and the next number)."""
    say("append extremes")
    d = 64
    ref = RefCache(12, 1, d)
    kv, sc = ref.to(dev)
    tops = [0.0, 2.0 ** -24, 2.0 ** -14, 448.0, 448.25, 449.0, 65504.0, 57344.0, 57376.0, 1.75, 1.7509765625]
    k = torch.zeros((len(tops), 1, d)).half()
    for i, x in enumerate(tops):
        k[i, 0, 3], k[i, 0, 7], k[i, 0, 9], k[i, 0, 11] = x, -x / 3, x / 1000, 2.0 ** -24
    v = -k
    slots = [16 * i for i in range(len(tops))]
    store_kv_fp8(kv, sc, i32(slots, dev), None, k.to(dev), v.to(dev))
    ref.store(slots, k, v)
    ref.same(kv, sc)
    assert float(sc[0, 0, 0]) == EMPTY and float(sc[0, 3, 0]) == 1.0 and float(sc[0, 4, 0]) == 2.0


def test_append_leaves_other_layers_and_pages(dev):
    say("append layers")
    gen = torch.Generator().manual_seed(1)
    kv = torch.zeros((3, 2, 4, 2, 16, 128), dtype=F8, device=dev)
    sc = torch.full((3, 2, 4, 2), EMPTY, device=dev)
    k, v = rows(gen, 5, 2, 128), rows(gen, 5, 2, 128)
    store_kv_fp8(kv, sc, i32([32, 33, 34, 35, 36], dev), None, k.to(dev), v.to(dev), layer=1)
    ref = RefCache(4, 2, 128)
    ref.store([32, 33, 34, 35, 36], k, v)
    ref.same(kv[1], sc[1])
    assert not kv[0].float().any() and not kv[2].float().any() and bool((sc[0] == EMPTY).all())


# ---- decode ---------------------------------------------------------------------------------------

LENS = [1, 2, 15, 16, 17, 31, 32, 33, 47, 0, 64, 65, 100, 255, 257, 600, 1025]


def ref_decode(ref, table, lens, q, scale=None):
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    hkv = ref.c.shape[2]
    w, wt = torch.zeros((len(lens), hkv, table.shape[1]), dtype=torch.float64), 0.0
    vals = ref.values()
    for b, n in enumerate(lens):
        if n:
            k, v = gather(vals, table[b], int(n))
            o, t, wk, r = attend(q[b:b + 1], k, v, [int(n)], scale)
            out[b], tol[b], wt = o[0], t[0], max(wt, r)
            pad = torch.zeros((hkv, -(-int(n) // 16) * 16), dtype=torch.float64)
            pad[:, :int(n)] = wk
            w[b, :, :pad.shape[1] // 16] = pad.unflatten(-1, (-1, 16)).sum(-1)
    return out, tol, w, wt


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (32, 8, 128), (8, 8, 64), (10, 2, 128), (16, 1, 64), (16, 1, 128),
                                      (3, 1, 128), (16, 2, 256), (7, 7, 256), (12, 3, 64)])
@pytest.mark.parametrize("weights", [False, True])
def test_decode_ragged(dev, hq, hkv, d, weights):
    say(f"decode fp8 hq={hq} hkv={hkv} d={d} weights={weights}")
    rng = np.random.default_rng(hq * 100 + d)
    gen = torch.Generator().manual_seed(hq)
    table, pages = tables(rng, LENS)
    ref = random_cache(pages, hkv, d, hq + d, tail=0.02)
    kv, sc = ref.to(dev)
    q = (1.5 * torch.randn((len(LENS), hq, d), generator=gen)).half()
    out, tol, w, wt = ref_decode(ref, table, LENS, q)
    start = torch.rand(w.shape, generator=gen)
    pw = start.to(dev) if weights else None
    got = paged_attention_fp8(q.to(dev), kv, sc, i32(table, dev), i32(LENS, dev), page_weights=pw, validate=True)
    check(got, out, tol, "out")
    if weights:
        for b, n in enumerate(LENS):
            p = -(-n // 16)
            exp = start[b, :, :p].double() + w[b, :, :p]
            check(pw[b, :, :p], exp, w[b, :, :p] * wt + 2.0 ** -23 * exp + 1e-30, "weights")
            assert torch.equal(pw[b, :, p:].cpu(), start[b, :, p:])


@pytest.mark.parametrize("batch,n", [(1, 512), (1, 5000), (1, 16), (2, 9000), (300, 40), (900, 3)])
def test_decode_splits(dev, batch, n):
    """One long row over many ranges, many short rows in one."""
    say(f"decode fp8 splits {batch} x {n}")
    rng = np.random.default_rng(n)
    lens = rng.integers(max(1, n // 2), n + 1, batch)
    lens[0] = n
    table, pages = tables(rng, lens)
    ref = random_cache(pages, 2, 128, n)
    kv, sc = ref.to(dev)
    q = torch.randn((batch, 8, 128), generator=torch.Generator().manual_seed(n)).half()
    out, tol, w, wt = ref_decode(ref, table, lens, q)
    pw = torch.zeros(w.shape, device=dev)
    got = paged_attention_fp8(q.to(dev), kv, sc, i32(table, dev), i32(lens, dev), page_weights=pw)
    check(got, out, tol, "out")
    check(pw, w, w * wt + 1e-30, "weights")
    again = paged_attention_fp8(q.to(dev), kv, sc, i32(table, dev), i32(lens, dev))
    assert torch.equal(got, again)


@pytest.mark.parametrize("batch,d,weights", [(6, 256, True), (2500, 256, True), (4096, 256, False), (4096, 128, True)])
def test_decode_largest_groups(dev, batch, d, weights):
    """16 query heads on one kv head and many rows: the most shared memory a call takes."""
    say(f"decode fp8 largest groups batch={batch} d={d} weights={weights}")
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 40, batch)
    lens[:3] = [1000, 0, 333]
    table, pages = tables(rng, lens)
    ref = random_cache(pages, 1, d, batch)
    kv, sc = ref.to(dev)
    q = torch.randn((batch, 16, d), generator=torch.Generator().manual_seed(batch)).half()
    out, tol, w, wt = ref_decode(ref, table, lens, q)
    pw = torch.zeros(w.shape, device=dev) if weights else None
    got = paged_attention_fp8(q.to(dev), kv, sc, i32(table, dev), i32(lens, dev), page_weights=pw)
    check(got, out, tol, "out")
    if weights:
        check(pw, w, w * wt + 1e-30, "weights")


def test_decode_masks_caps_and_strange_pages(dev):
    """Inactive rows keep their output; lengths are capped; ids outside the pool hold no keys; a row with no key is
    zero; what lies behind a row's end (NaN codes, any scale) is not seen."""
    say("decode fp8 masks")
    rng = np.random.default_rng(3)
    lens = np.array([40, 100, 33, 64, 77, 20, 90], np.int32)
    table, pages = tables(rng, lens)
    ref = random_cache(pages, 2, 128, 5)
    kv, sc = ref.to(dev)
    raw = kv.view(torch.uint8)
    for b, n in enumerate(lens):  # NaN behind the rows' ends
        if n % 16:
            raw[:, int(table[b, n // 16]), :, int(n) % 16:] = 0x7f
    spare = [p for p in range(pages) if p not in set(table[b, j] for b in range(7) for j in range(-(-int(lens[b]) // 16)))]
    raw[:, spare] = 0xff
    sc[:, spare] = float("nan")
    q = torch.randn((7, 6, 128), generator=torch.Generator().manual_seed(4)).half()
    active = np.array([1, 1, 0, 1, 1, 1, 1], np.uint8)
    holes = {1: [0, 3], 3: [1], 5: [0, 1]}  # row 5 has no key left
    bad = table.copy()
    for b, js in holes.items():
        for j in js:
            bad[b, j] = [-1, pages, 2 ** 31 - 1][j % 3]
    out, tol = torch.full(q.shape, 7.0, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    vals = ref.values()
    for b, n in enumerate(lens):
        if active[b]:
            n = min(int(n), 80)
            k, v = gather(vals, table[b], n)
            live = torch.tensor([j // 16 not in holes.get(b, []) for j in range(n)])
            o, t, _, _ = attend(q[b:b + 1], k[live], v[live], [int(live.sum())])
            out[b], tol[b] = o[0], t[0]
    got = torch.full(q.shape, 7.0, dtype=torch.float16, device=dev)
    pw = torch.zeros((7, 2, table.shape[1]), device=dev)
    paged_attention_fp8(q.to(dev), kv, sc, i32(bad, dev), i32(lens, dev), torch.as_tensor(active).to(dev), out=got,
                        max_seq_len=80, page_weights=pw)
    check(got, out, tol, "out")
    assert torch.equal(got[2].cpu(), torch.full((6, 128), 7.0).half()) and not got[5].any()
    total = pw.sum(-1).cpu()
    assert torch.allclose(total, torch.tensor([3., 3, 0, 3, 3, 0, 3])[:, None].expand(7, 2), atol=1e-4)
    assert not pw[1, :, [0, 3]].any() and not pw[2].any() and not pw[5].any() and not pw[1, :, 5:].any()


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (8, 2, 64), (16, 2, 256), (5, 1, 128)])
def test_append_and_decode_is_the_two_calls(dev, hq, hkv, d):
    """The fused step leaves the cache of ``store_kv_fp8`` and the output of ``paged_attention_fp8``, bit for bit."""
    say(f"append+decode fp8 hq={hq} hkv={hkv} d={d}")
    rng = np.random.default_rng(d)
    gen = torch.Generator().manual_seed(d)
    lens = np.array(LENS + [48, 500, 16], np.int32)
    B = len(lens)
    table, pages = tables(rng, lens)
    table[-1, 0] = pages + 3  # this row's last page is outside the pool: nothing is stored
    active = np.ones(B, bool)
    active[4] = False
    ref = random_cache(pages, hkv, d, d)
    kv, sc = ref.to(dev)
    for big in (0.1, 1.0, 50.0):  # (50: scales grow)
        k, v = rows(gen, B, hkv, d, big), rows(gen, B, hkv, d, big)
        q = torch.randn((B, hq, d), generator=gen).half().to(dev)
        last = np.maximum(lens - 1, 0)
        slots = table[np.arange(B), last // 16].astype(np.int64) * 16 + last % 16
        slots[(lens == 0) | (lens > 520)] = -1
        slots[-1] = -1
        kv2, sc2 = kv.clone(), sc.clone()
        act = torch.as_tensor(active).to(dev)
        store_kv_fp8(kv2, sc2, i32(slots, dev), act, k.to(dev), v.to(dev))
        pw2 = torch.zeros((B, hkv, table.shape[1]), device=dev)
        pw = pw2.clone()
        want = paged_attention_fp8(q, kv2, sc2, i32(table, dev), i32(lens, dev), act, max_seq_len=520, page_weights=pw2)
        got = store_kv_fp8_and_decode(q, kv, sc, i32(table, dev), i32(lens, dev), act, k.to(dev), v.to(dev),
                                      max_seq_len=520, page_weights=pw)
        assert torch.equal(kv.view(torch.uint8), kv2.view(torch.uint8)) and torch.equal(sc, sc2)
        assert torch.equal(got, want) and torch.equal(pw, pw2)
        ref.store(slots.tolist(), k, v, active)
        ref.same(kv, sc)


def test_decode_far_pages(dev):
    """Page offsets past 2^31 bytes (and 2^32), in the append too."""
    say("decode fp8 far pages")
    hkv, d, pages = 8, 128, 300000
    kv = torch.zeros((2, pages, hkv, 16, d), dtype=F8, device=dev)
    sc = torch.full((2, pages, hkv), EMPTY, device=dev)
    gen = torch.Generator().manual_seed(8)
    ids = [299999, 131072, 262144, 7]
    pos = np.arange(50)
    slots = np.asarray(ids)[pos // 16] * 16 + pos % 16
    k, v = rows(gen, 50, hkv, d), rows(gen, 50, hkv, d)
    store_kv_fp8(kv, sc, i32(slots, dev), None, k.to(dev), v.to(dev))
    ref = RefCache(4, hkv, d)
    ref.store(pos.tolist(), k, v)
    ref.same(kv[:, ids], sc[:, ids])
    q = torch.randn((1, 16, d), generator=gen).half()
    out, tol, _, _ = ref_decode(ref, np.arange(4)[None], [50], q)
    check(paged_attention_fp8(q.to(dev), kv, sc, i32([ids], dev), i32([50], dev)), out, tol)
    o = paged_attention_fp8(q.to(dev), kv, sc, i32(ids, dev), None, query_start=49)
    check(o, out, tol)


# ---- prefill --------------------------------------------------------------------------------------


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (32, 8, 128), (4, 4, 64), (5, 1, 128), (16, 1, 64), (24, 1, 128)])
@pytest.mark.parametrize("t,start", [(1, 0), (1, 16), (1, 530), (7, 0), (16, 16), (33, 5), (64, 0), (100, 720), (200, 31)])
def test_prefill(dev, hq, hkv, d, t, start):
    say(f"prefill fp8 hq={hq} hkv={hkv} d={d} t={t} start={start}")
    rng = np.random.default_rng(t)
    gen = torch.Generator().manual_seed(t + start)
    table, pages = tables(rng, [start + t])
    ref = random_cache(pages, hkv, d, start, tail=0.02)
    kv, sc = ref.to(dev)
    if (start + t) % 16:  # behind the sequence's end: anything
        kv.view(torch.uint8)[:, int(table[0, (start + t) // 16]), :, (start + t) % 16:] = 0x7f
    q = (1.5 * torch.randn((t, hq, d), generator=gen)).half()
    k, v = gather(ref.values(), table[0], start + t)
    out, tol, _, _ = attend(q, k, v, start + 1 + torch.arange(t))
    got = paged_attention_fp8(q.to(dev), kv, sc, i32(table[0], dev), None, query_start=start, validate=True)
    check(got, out, tol)


@pytest.mark.parametrize("hq,hkv,d,t,start", [(16, 8, 128, 512, 1024), (32, 8, 128, 333, 720), (16, 8, 64, 1500, 3),
                                              (8, 2, 128, 2048, 0), (40, 8, 128, 300, 2500)])
def test_prefill_large(dev, hq, hkv, d, t, start):
    say(f"prefill fp8 large hq={hq} hkv={hkv} d={d} t={t} start={start}")
    rng = np.random.default_rng(t)
    gen = torch.Generator().manual_seed(t + start)
    table, pages = tables(rng, [start + t])
    ref = random_cache(pages, hkv, d, start)
    kv, sc = ref.to(dev)
    q = torch.randn((t, hq, d), generator=gen).half()
    k, v = gather(ref.values(), table[0], start + t)
    out, tol, _, _ = attend(q, k, v, start + 1 + torch.arange(t))
    check(paged_attention_fp8(q.to(dev), kv, sc, i32(table, dev), None, query_start=start), out, tol)


@pytest.mark.parametrize("hq,hkv,d,t,start", [(32, 8, 128, 1101, 0), (32, 8, 128, 600, 1500), (16, 8, 128, 2103, 2),
                                              (32, 8, 64, 1101, 3400), (36, 2, 128, 1901, 6)])
def test_prefill_blocks(dev, hq, hkv, d, t, start):
    """Calls that fill the chip, one and two key groups: NaN behind the sequence's end, a page outside the pool."""
    say(f"prefill fp8 blocks hq={hq} hkv={hkv} d={d} t={t} start={start}")
    rng = np.random.default_rng(t)
    gen = torch.Generator().manual_seed(t + start)
    total = start + t
    table, pages = tables(rng, [total])
    ref = random_cache(pages, hkv, d, start)
    kv, sc = ref.to(dev)
    assert total % 16
    kv.view(torch.uint8)[:, int(table[0, total // 16]), :, total % 16:] = 0x7f
    bad = table[0].copy()
    bad[total // 32] = -5
    live = torch.tensor([j // 16 != total // 32 for j in range(total)])
    q = torch.randn((t, hq, d), generator=gen).half()
    k, v = gather(ref.values(), table[0], total)
    out, tol, _, _ = attend(q, k[live], v[live], torch.cumsum(live.long(), 0)[start:])
    check(paged_attention_fp8(q.to(dev), kv, sc, i32(bad, dev), None, query_start=start), out, tol)


def test_prefill_strange_pages(dev):
    say("prefill fp8 strange pages")
    rng = np.random.default_rng(2)
    t, start = 90, 75
    table, pages = tables(rng, [start + t])
    ref = random_cache(pages, 2, 128, 6)
    kv, sc = ref.to(dev)
    bad = table[0].copy()
    bad[[0, 3, 9]] = [-1, pages, -2 ** 31]
    q = torch.randn((t, 4, 128), generator=torch.Generator().manual_seed(1)).half()
    k, v = gather(ref.values(), table[0], start + t)
    live = torch.tensor([j // 16 not in (0, 3, 9) for j in range(start + t)])
    limit = torch.cumsum(live.long(), 0)[start:]
    out, tol, _, _ = attend(q, k[live], v[live], limit)
    check(paged_attention_fp8(q.to(dev), kv, sc, i32(bad, dev), None, query_start=start), out, tol)


# ---- streams and graphs ---------------------------------------------------------------------------


def test_streams_and_graphs(dev):
    """Two streams at once, and two captured graphs replayed between eager calls, each with scratch of its own."""
    say("fp8 streams and graphs")
    rng = np.random.default_rng(9)
    gen = torch.Generator().manual_seed(9)
    sets = []
    for i, n in enumerate((700, 333)):
        lens = rng.integers(n // 2, n, 9)
        table, pages = tables(rng, lens)
        ref = random_cache(pages, 2, 128, n)
        kv, sc = ref.to(dev)
        q = torch.randn((9, 8, 128), generator=gen).half().to(dev)
        k, v = rows(gen, 9, 2, 128).to(dev), rows(gen, 9, 2, 128).to(dev)
        a = [q, kv, sc, i32(table, dev), i32(lens, dev), None, k, v]
        want = store_kv_fp8_and_decode(*a)  # (storing the same token again changes nothing)
        sets.append((a, want))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for (a, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(store_kv_fp8_and_decode(*a))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, (_, w) in zip(got, sets))
    graphs = []
    for a, _ in sets:
        pw = torch.zeros((9, 2, a[3].shape[1]), device=dev)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = store_kv_fp8_and_decode(*a, page_weights=pw)
            o2 = paged_attention_fp8(*a[:5])
        graphs.append((g, o, o2, pw))
    for rep in range(4):
        for (g, o, o2, _), (a, w) in zip(graphs, sets):
            o.zero_()
            o2.zero_()
            g.replay()
            paged_attention_fp8(*a[:5])
        torch.cuda.synchronize()
        for (g, o, o2, pw), (a, w) in zip(graphs, sets):
            assert torch.equal(o, w) and torch.equal(o2, w)
            assert torch.allclose(pw.sum(-1), torch.full((9, 2), 4.0 * (rep + 1), device=dev), rtol=1e-4)


def test_graph_of_a_run(dev):
    """Append of a chunk, prefill with split keys, decode with weights and eviction in one captured graph, replayed
    between eager calls of other sizes."""
    say("fp8 graph of a run")
    gen = torch.Generator().manual_seed(21)
    hkv, hq, d, n, start = 2, 8, 128, 40, 2000
    pages = (start + n) // 16 + 1
    table = torch.randperm(pages, generator=gen).to(torch.int32).to(dev)
    pos = torch.arange(start, start + n, device=dev)
    slots = (table[pos // 16] * 16 + pos % 16).int()
    ref = random_cache(pages, hkv, d, 5)
    kv, sc = ref.to(dev)
    q = torch.randn((n, hq, d), generator=gen).half().to(dev)
    k, v = rows(gen, n, hkv, d).to(dev), rows(gen, n, hkv, d).to(dev)
    lens = i32([start + n], dev)

    def run(weights):
        store_kv_fp8(kv, sc, slots, None, k, v)
        a = paged_attention_fp8(q, kv, sc, table, None, query_start=start)
        b = paged_attention_fp8(q[-1:], kv, sc, table[None], lens, page_weights=weights)
        return (a, b, *evict_pages(table[None], lens, weights, 50, sink_pages=2, recent_pages=3))

    want = run(torch.zeros((1, hkv, pages), device=dev))
    weights = torch.zeros((1, hkv, pages), device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        weights.zero_()
        got = run(weights)
    for _ in range(4):
        for t in got:
            t.zero_()
        g.replay()
        paged_attention_fp8(q[:7], kv, sc, table, None, query_start=1500)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        run(torch.zeros((1, hkv, pages), device=dev))


def test_carriers(dev):
    """Arrays that are no torch tensors, the codes as bytes: the same results as with tensors."""
    say("fp8 carriers")

    def raw(t):
        names = {torch.float16: "float16", torch.int32: "int32", torch.float32: "float32", torch.uint8: "uint8"}
        return DeviceArray(t.data_ptr(), t.shape, names[t.dtype], device=t.device.index, owner=t)

    gen = torch.Generator().manual_seed(3)
    hkv, hq, d, n = 2, 4, 64, 75
    table, pages = tables(np.random.default_rng(3), [n])
    slots = i32(table[0][np.arange(n) // 16] * 16 + np.arange(n) % 16, dev)
    tab, lens = i32(table, dev), i32([n], dev)
    q = torch.randn((n, hq, d), generator=gen).half().to(dev)
    k, v = rows(gen, n, hkv, d).to(dev), rows(gen, n, hkv, d).to(dev)
    results = []
    for wrap, kind in ((lambda t: t, F8), (raw, torch.uint8), (lambda t: t, torch.uint8)):
        codes = torch.zeros((2, pages, hkv, 16, d), dtype=torch.uint8, device=dev)
        scales = torch.full((2, pages, hkv), EMPTY, device=dev)
        kv, sc = wrap(codes.view(kind)), wrap(scales)
        w = torch.zeros((1, hkv, tab.shape[1]), device=dev)
        store_kv_fp8(kv, sc, wrap(slots), None, wrap(k), wrap(v))
        a = paged_attention_fp8(wrap(q), kv, sc, wrap(tab), None, query_start=0)
        b = store_kv_fp8_and_decode(wrap(q[-1:]), kv, sc, wrap(tab), wrap(lens), None, wrap(k[-1:]), wrap(v[-1:]),
                                    page_weights=wrap(w))
        e = evict_pages(wrap(tab), wrap(lens), wrap(w), 3)
        results.append((codes, scales, a, b, w, *e))
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))


def test_native_and_python_calls_agree(dev):
    """The native argument checks and the Python ones lead to the same calls; what the native ones leave to Python."""
    say("fp8 native calls")
    gen = torch.Generator().manual_seed(4)
    hkv, hq, d = 2, 8, 128
    lens = [33, 700, 0, 16]
    table, pages = tables(np.random.default_rng(4), lens)
    ref = random_cache(pages, hkv, d, 4)
    q = torch.randn((4, hq, d), generator=gen).half().to(dev)
    k, v = rows(gen, 4, hkv, d).to(dev), rows(gen, 4, hkv, d).to(dev)
    tab, ln = i32(table, dev), i32(lens, dev)
    act = torch.tensor([1, 1, 1, 0], dtype=torch.uint8, device=dev)
    got = []
    for validate in (False, True):
        kv, sc = ref.to(dev)
        w = torch.zeros((4, hkv, tab.shape[1]), device=dev)
        o = store_kv_fp8_and_decode(q, kv, sc, tab, ln, act, k, v, page_weights=w, validate=validate)
        p = paged_attention_fp8(q, kv, sc, tab[1], None, query_start=600, validate=validate)
        store_kv_fp8(kv, sc, i32([0, 1, 2, 3], dev), act, k, v, validate=validate)
        got.append((o, p, w, kv.view(torch.uint8), sc))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    kv, sc = ref.to(dev)
    for args in ((q[:, ::2], kv, sc, tab, ln), (q, kv.transpose(1, 2), sc, tab, ln), (q, kv, sc[:, :-1], tab, ln),
                 (q, kv, sc, tab.long(), ln), (q.float(), kv, sc, tab, ln), (q, kv, sc, tab, ln[:3])):
        with pytest.raises(ValueError):
            paged_attention_fp8(*args)
    for start in (-1, 16 * tab.shape[1] - 3, 2 ** 62):
        with pytest.raises(ValueError):
            paged_attention_fp8(q, kv, sc, tab[1], None, query_start=start)
    with pytest.raises(ValueError, match="not a page"):  # a table entry outside the pool
        paged_attention_fp8(q, kv, sc, torch.where(tab == tab[1, 2], pages, tab), ln, validate=True)
    shared = tab.clone()
    shared[3, 0] = tab[0, 2]  # row 0's last page, where its token goes, is read by row 3
    store_kv_fp8_and_decode(q, kv, sc, shared, ln, act, k, v, validate=True)  # (row 3 is inactive)
    with pytest.raises(ValueError, match="another row's table"):
        store_kv_fp8_and_decode(q, kv, sc, shared, ln, None, k, v, validate=True)
    paged_attention_fp8(q, kv, sc, shared, ln, validate=True)
    sc[0, int(tab[1, 1]), 0] = 0.75
    with pytest.raises(ValueError, match="powers of two"):
        paged_attention_fp8(q, kv, sc, tab, ln, validate=True)
