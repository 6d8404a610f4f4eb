"""evict_pages on the GPU against the definition."""
import numpy as np
import pytest
import torch

from fp8_util import evict_ref
from gpu_util import say
from infurnace_amd.kernels import evict_pages

pytestmark = pytest.mark.gpu


def run(dev, table, lens, w, keep, sink, recent, active=None):
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    got = evict_pages(t(table), t(lens), t(w), keep, sink_pages=sink, recent_pages=recent,
                      active_mask=None if active is None else t(active))
    exp = evict_ref(table, lens, w, keep, sink, recent, active)
    for g, e, what in zip(got, exp, ("table", "lens", "weights", "evicted")):
        assert np.array_equal(g.cpu().numpy(), e, equal_nan=e.dtype.kind == "f"), what


@pytest.mark.parametrize("B,M,hkv,keep,sink,recent", [(1, 1, 1, 1, 0, 1), (7, 40, 8, 12, 1, 4), (5, 64, 3, 5, 4, 1),
                                                      (3, 1100, 2, 300, 2, 16), (2, 4096, 8, 256, 0, 1),
                                                      (4, 33, 1, 3, 1, 1), (2, 2500, 1, 2400, 0, 3)])
def test_rows(dev, B, M, hkv, keep, sink, recent):
    say(f"evict B={B} M={M} hkv={hkv} keep={keep}")
    rng = np.random.default_rng(B * M)
    table = rng.permutation(B * M).reshape(B, M).astype(np.int32)
    lens = rng.integers(0, M * 16 + 1, B).astype(np.int32)
    lens[0] = M * 16
    w = np.exp(2 * rng.standard_normal((B, hkv, M))).astype(np.float32)
    run(dev, table, lens, w, keep, sink, recent)


def test_ties_and_strange_weights(dev):
    """Equal weights go to the lower page; NaN is lowest, infinities and negatives order as numbers, -0 is 0."""
    say("evict ties")
    rng = np.random.default_rng(1)
    B, M = 9, 700
    table = rng.permutation(B * M).reshape(B, M).astype(np.int32)
    lens = np.full(B, M * 16 - 3, np.int32)
    w = rng.integers(0, 3, (B, 1, M)).astype(np.float32)
    w[1] = 0
    w[2] = np.where(rng.random((1, M)) < 0.5, 0.0, -0.0)
    w[3] = rng.standard_normal((1, M))
    w[4, 0, rng.permutation(M)[:300]] = np.nan
    w[5, 0, rng.permutation(M)[:200]] = np.inf
    w[6, 0, rng.permutation(M)[:500]] = -np.inf
    w[7] = np.nan
    w[8] = 1e-42 * rng.integers(0, 5, (1, M))
    for keep in (3, 50, 333, 699):
        run(dev, table, lens, w, keep, 1, 2)


def test_inactive_rows_and_lengths(dev):
    say("evict inactive")
    rng = np.random.default_rng(2)
    table = rng.permutation(6 * 20).reshape(6, 20).astype(np.int32)
    lens = np.array([320, 5000, -7, 0, 161, 320], np.int32)  # (past the table, negative, empty)
    w = rng.random((6, 4, 20)).astype(np.float32)
    run(dev, table, lens, w, 10, 2, 3, np.array([1, 1, 1, 1, 1, 0], np.uint8))
    run(dev, table, lens, w, 10, 2, 3, np.array([0, 1, 0, 1, 0, 1], bool))


@pytest.mark.parametrize("M", [16000, 32768])
def test_wide_tables(dev, M):
    say(f"evict wide {M}")
    rng = np.random.default_rng(M)
    table = rng.permutation(2 * M).reshape(2, M).astype(np.int32)
    w = rng.random((2, 2, M)).astype(np.float32)
    t = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    lens = np.array([M * 16, M * 16 - 5], np.int32)
    keep = 1000
    tb, ln, ww, gone = (x.cpu().numpy() for x in evict_pages(t(table), t(lens), t(w), keep))
    for b in range(2):
        s = w[b].astype(np.float64).sum(0).astype(np.float32)
        order = np.argsort(-s[1:M - 1], kind="stable")[:keep - 2] + 1
        kept = np.sort(np.concatenate([[0], order, [M - 1]]))
        assert np.array_equal(tb[b, :keep], table[b, kept]) and np.array_equal(ww[b, :, :keep], w[b][:, kept])
        assert np.array_equal(tb[b, keep:], np.delete(table[b], kept)) and not ww[b, :, keep:].any()
        assert ln[b] == lens[b] - 16 * (M - keep) and gone[b] == M - keep
