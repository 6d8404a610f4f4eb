"""64-bit references of the 8-bit KV cache and of page eviction (CPU; written from the definitions)."""
import math

import numpy as np
import torch

F8 = torch.float8_e4m3fn
EMPTY = 2.0 ** -32


def need_scale(amax: float) -> float:
    """The smallest power of two s >= 2^-32 with amax <= 448 s."""
    s = EMPTY
    while amax > 448.0 * s:
        s *= 2.0
    return s


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number (ties to even), for |x| <= 448, in 64 bits."""
    _, e = torch.frexp(x.double())
    step = 2.0 ** (e.double() - 4).clamp_min(-9)
    return torch.round(x.double() / step) * step


class RefCache:
    """The cache as values: codes (64-bit numbers) [2, P, H, 16, D] and scales [2, P, H]."""

    def __init__(self, pages, hkv, d):
        self.c = torch.zeros((2, pages, hkv, 16, d), dtype=torch.float64)
        self.s = torch.full((2, pages, hkv), EMPTY, dtype=torch.float64)

    def store(self, slots, k, v, active=None):
        """slots: list of ints; k, v [T, H, D] fp16 (CPU)."""
        pages = {}
        for t, slot in enumerate(slots):
            if (active is None or active[t]) and 0 <= slot < self.c.shape[1] * 16:
                pages.setdefault(slot // 16, {})[slot % 16] = t  # (of two with one slot the later)
        for p, rows in pages.items():
            for i, x in enumerate((k, v)):
                x = x.double()
                for h in range(x.shape[1]):
                    need = need_scale(max(float(x[t, h].abs().max()) for t in rows.values()))
                    if 0 in rows:
                        self.c[i, p, h] = 0.0
                        new = need
                    else:
                        new = max(float(self.s[i, p, h]), need)
                        if new != self.s[i, p, h]:
                            self.c[i, p, h] = round_e4m3(self.c[i, p, h] * (float(self.s[i, p, h]) / new))
                    self.s[i, p, h] = new
                    for o, t in rows.items():
                        self.c[i, p, h, o] = round_e4m3(x[t, h] / new)

    def values(self):
        return self.c * self.s[..., None, None]

    def to(self, dev):
        """(codes, scales) tensors of the kernels."""
        return self.c.float().to(F8).to(dev), self.s.float().to(dev)

    def same(self, codes, scales):
        assert torch.equal(scales.cpu().double(), self.s), "scales differ"
        assert torch.equal(codes.cpu().float().double(), self.c), "codes differ"


def random_cache(pages, hkv, d, seed, tail=0.0):
    """A filled cache: every page's 16 rows stored at once; keys with large channels."""
    gen = torch.Generator().manual_seed(seed)
    ref = RefCache(pages, hkv, d)
    x = torch.randn((2, pages, hkv, 16, d), generator=gen)
    x[0] *= torch.exp(0.6 * torch.randn((hkv, 1, d), generator=gen))
    if tail:
        x = torch.where(torch.rand(x.shape, generator=gen) < tail, 8.0 * x, x)
    x = x.half().double()
    amax = x.abs().amax((-1, -2))
    s = torch.full_like(amax, EMPTY)
    while bool((amax > 448 * s).any()):
        s = torch.where(amax > 448 * s, 2 * s, s)
    ref.s = s
    ref.c = round_e4m3(x / s[..., None, None])
    return ref


def gather(values, table_row, n):
    """K, V [n, H, D] of a row's first n tokens."""
    at = torch.as_tensor(np.asarray(table_row[:-(-n // 16)]), dtype=torch.long)
    x = values[:, at].permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :n]
    return x[0], x[1]


def attend(q, k, v, limit, scale=None):
    """q [n, hq, d] fp16, k and v [m, hkv, d] in 64 bits, query i sees limit[i] keys.  Returns (out, tolerance, weights
    [hkv, m], their relative tolerance).

    Tolerance of a kernel that accumulates in fp32 and rounds probabilities and outputs to fp16:
      scores: d products, each addition off by 2^-24 of the sum of magnitudes, the scale and base change by
        2^-23 of the score, exp2 by 2^-22: |dp / p| <= ds = 2 ((d + 4) 2^-24 sum |q k| scale + 2^-21)
      probabilities in fp16: 2^-11 relative, or 2^-25 absolute below 2^-14 (of a maximum of 1)
      sums over m keys in fp32, rescaled at most once for each of them: m 2^-23 relative at most, and sqrt-like in fact
      the output: 2^-11 relative, 2^-25 absolute
    """
    n, hq, d = q.shape
    m, hkv = k.shape[0], k.shape[1]
    g = hq // hkv
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros((n, hq, d), dtype=torch.float64)
    tol = torch.zeros_like(out)
    w = torch.zeros((hkv, m), dtype=torch.float64)
    wt = 0.0
    limit = torch.as_tensor(limit)
    for h in range(hq):
        qh, kh, vh = q[:, h].double(), k[:, h // g], v[:, h // g]
        s = qh @ kh.t() * scale
        ds = 2 * ((d + 4) * 2.0 ** -24 * (qh.abs() @ kh.abs().t()) * scale + 2.0 ** -21) + m * 2.0 ** -23
        hide = torch.arange(m)[None, :] >= limit[:, None]
        s = s.masked_fill(hide, -math.inf)
        top = s.amax(-1, keepdim=True) if m else torch.zeros((n, 1))
        p = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
        l = p.sum(-1, keepdim=True)
        small = ((p > 0) & (p < 2.0 ** -13)).double()
        p = p / l.clamp_min(1e-300)
        out[:, h] = p @ vh
        dp = p * (2 * ds + 2.0 ** -11) + small * 2.0 ** -25
        ds_row = (p * 2 * ds).sum(-1, keepdim=True)  # (the sum they are divided by)
        tol[:, h] = dp @ vh.abs() + (ds_row + 2.0 ** -11) * out[:, h].abs() + 2.0 ** -25
        w[h // g] += p.sum(0)
        if m:
            wt = max(wt, float((2 * ds.masked_fill(hide, 0)).max() + 4 * 2.0 ** -24 * s.masked_fill(hide, 0).abs().max()))
    return out, tol, w, 2 * wt + 2.0 ** -20


def check(got, ref, tol, what=""):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    over = (got - ref).abs() - tol
    assert not (over > 0).any(), f"{what}: {int((over > 0).sum())} of {over.numel()} outside, by up to {float(over.max()):.3g}"


def tables(rng, lens, extra=5):
    """Random distinct pages for rows of these lengths: (table [B, max_pages], pages)."""
    need = [-(-int(n) // 16) for n in lens]
    total = sum(need) + extra
    perm = rng.permutation(total).astype(np.int32)
    table = np.full((len(lens), max(1, max(need))), perm[-1], np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def evict_ref(table, lens, w, keep, sink, recent, active=None):
    """The definition, row by row."""
    table, lens, w = table.copy(), lens.copy(), w.copy()
    gone = np.zeros(len(lens), np.int32)
    M = table.shape[1]
    for b in range(len(lens)):
        n = -(-max(0, min(int(lens[b]), 16 * M)) // 16)
        kept = list(range(n))
        if n > keep and (active is None or active[b]):
            def key(j):
                s = np.float32(sum(np.float64(w[b, h, j]) for h in range(w.shape[1])))
                return (0.0, 0) if np.isnan(s) else (float(s), 1)
            mid = [(not_nan, s, -j) for j in range(sink, n - recent) for s, not_nan in [key(j)]]
            best = sorted(mid, reverse=True)[:keep - sink - recent]
            kept = sorted(set(range(sink)) | set(range(n - recent, n)) | {-j for _, _, j in best})
        out = [j for j in range(n) if j not in set(kept)]
        row, old = table[b].copy(), w[b].copy()
        table[b, :n] = row[kept + out]
        w[b] = 0
        w[b, :, :len(kept)] = old[:, kept]
        gone[b] = len(out)
        lens[b] -= 16 * len(out)
    return table, lens, w, gone
