"""The 8-bit KV cache and the eviction of its pages, as measurable cases.

A case is one layer's call of a serving engine whose K/V are held in 8 bits with a scale for each page and
head: a step's or a chunk's append, a decode step, a prefill chunk, or the eviction that follows some steps.
Head layouts are the configurations of ``infurnace_amd.workloads`` (16 query / 8 kv heads x 128 and 32 / 8 x 128),
their tensor-parallel shards and sizes around them.  ``listed`` gives the fixed cases, ``draw`` more of the same
ranges, ``run`` computes them with elementary torch operations or (``own``) with the framework's calls.

The cache of a layer: codes [2, pages, kv heads, 16 tokens, dims] in e4m3 and scales [2, pages, kv heads]
(powers of two); a value is its code times its block's scale.
"""
import math

import torch

own = False

BS = 16              # tokens per page
F8 = torch.float8_e4m3fn
F8_MAX = 448.0       # the largest e4m3 number
MIN_EXP = -32        # exponent of an empty block's scale: 448 * 2^-32 is above the smallest fp16 number


def listed():
    return [
        # The appends of one decode step: a token for each of 48 sequences, pages filled to any level.
        dict(name="append_step", kind="append", form="step", hkv=8, d=128, tokens=48, start=0),
        # A chunk of odd length behind a prefix that ends inside a page.
        dict(name="append_ragged", kind="append", form="chunk", hkv=4, d=64, tokens=333, start=727),
        # A long prompt's K/V at once.
        dict(name="append_prompt", kind="append", form="chunk", hkv=8, d=128, tokens=8192, start=0),
        # One user's decode step: the latency of a call.
        dict(name="decode_single", kind="decode", form="append", hq=16, hkv=8, d=128, batch=1, lo=512, hi=512,
             idle=False, weights=False),
        # The ordinary batch: 32 ragged contexts up to 4096 tokens.
        dict(name="decode_ragged", kind="decode", form="append", hq=16, hkv=8, d=128, batch=32, lo=128, hi=4096,
             idle=False, weights=False),
        # One of four tensor-parallel ranks, with padding rows in the batch, gathering the pages' weights.
        dict(name="decode_shard", kind="decode", form="append", hq=8, hkv=2, d=128, batch=48, lo=100, hi=4000,
             idle=True, weights=True),
        # A full server of the larger model: 128 long contexts, attention and weights.
        dict(name="decode_large", kind="decode", form="plain", hq=32, hkv=8, d=128, batch=128, lo=1023, hi=8190,
             idle=False, weights=True),
        # The rest of a prompt after a prefix-cache hit: odd length, from a page boundary that is no tile boundary.
        dict(name="prefill_ragged", kind="prefill", hq=32, hkv=8, d=128, start=720, tokens=333),
        # A chunk in the middle of a prompt.
        dict(name="prefill_chunk", kind="prefill", hq=16, hkv=8, d=128, start=1024, tokens=512),
        # A large chunk deep in a long prompt of the larger model.
        dict(name="prefill_long", kind="prefill", hq=32, hkv=8, d=128, start=6144, tokens=2048),
        # A batch of ordinary contexts, those over 128 pages cut to that.
        dict(name="evict_step", kind="evict", hkv=8, batch=32, lo=128, hi=4096, keep=128, sink=1, recent=4),
        # Long contexts cut to 4096 tokens each.
        dict(name="evict_long", kind="evict", hkv=8, batch=64, lo=20000, hi=65536, keep=256, sink=2, recent=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(16, 8, 128), (16, 8, 128), (32, 8, 128), (32, 8, 128), (8, 4, 128), (8, 2, 128), (40, 8, 128), (16, 8, 64),
         (8, 8, 64), (8, 1, 128), (16, 1, 64)]


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "prefill", "prefill", "prefill", "evict"])
    hq, hkv, d = rng.choice(HEADS)
    if kind == "append":
        hkv, d = rng.choice([(hkv, d), (2, 256)])
        if rng.random() < 0.4:
            return dict(kind=kind, form="step", hkv=hkv, d=d, tokens=_log(rng, 1, 256), start=0)
        return dict(kind=kind, form="chunk", hkv=hkv, d=d, tokens=_log(rng, 2, 8192), start=rng.randint(0, 2000))
    if kind == "decode":
        hq, hkv, d = rng.choice([(hq, hkv, d), (hq, hkv, d), (hq, hkv, d), (16, 2, 256)])
        batch = _log(rng, 1, 160)
        hi = max(16, min(_log(rng, 64, 16000), 590000 // batch))  # (the listed cases' largest: about 590,000 keys)
        return dict(kind=kind, form=rng.choice(["plain", "append"]), hq=hq, hkv=hkv, d=d, batch=batch,
                    lo=rng.randint(1, hi), hi=hi, idle=rng.random() < 0.25, weights=rng.random() < 0.4)
    if kind == "prefill":
        tokens = _log(rng, 2, 4096)
        start = rng.choice([0, BS * rng.randint(0, 256), rng.randint(0, 6000)])
        while 4 * hq * d * tokens * (start + tokens / 2) > 2.4e11:  # (no more than the listed long chunk)
            tokens = tokens * 3 // 4
        return dict(kind=kind, hq=hq, hkv=hkv, d=d, start=start, tokens=tokens)
    batch = _log(rng, 1, 128)
    hi = min(_log(rng, 100, 65536), 4000000 // batch)
    sink, recent = rng.randint(0, 4), rng.randint(1, 16)
    return dict(kind=kind, hkv=hkv, batch=batch, lo=rng.randint(1, hi), hi=hi,
                keep=sink + recent + rng.randint(0, max(1, hi // BS)), sink=sink, recent=recent)


# ---- sizes that depend on the case alone ----------------------------------------------------------


def _lens(c):
    """The rows' lengths: spread over [lo, hi] (golden-ratio steps), the first at hi; every fifth row empty if `idle`."""
    n = [c["hi"] - int((i * 0.6180339887498949 % 1.0) * (c["hi"] - c["lo"])) for i in range(c["batch"])]
    return [0 if c.get("idle") and i % 5 == 4 else x for i, x in enumerate(n)]


def _pages(n):
    return -(-n // BS)


def work(c):
    """Every code, scale, table entry, query, output and new row once; 4 hq d flops a (query, key) pair."""
    hkv = c["hkv"]
    if c["kind"] == "evict":
        lens = _lens(c)
        pages = [_pages(n) for n in lens]
        kept = [min(n, c["keep"]) for n in pages]
        return {"bytes": 4 * (hkv + 1) * (sum(pages) + sum(kept)) + 12 * len(lens), "flops": hkv * sum(pages)}
    d = c["d"]
    row = 2 * hkv * d      # a token's K and V in codes
    if c["kind"] == "append":
        t = c["tokens"]
        pages = t if c["form"] == "step" else _pages(c["start"] % BS + t)
        return {"bytes": t * (2 * row + row + 4) + 8 * hkv * pages, "flops": 0}
    hq = c["hq"]
    if c["kind"] == "decode":
        lens = _lens(c)
        live = sum(1 for n in lens if n)
        pages = sum(_pages(n) for n in lens)
        new = live * (3 * row) if c["form"] == "append" else 0
        old = sum(lens) - (live if c["form"] == "append" else 0)
        total = old * row + new + pages * (8 * hkv + 4) + len(lens) * (4 * hq * d + 4)
        if c["weights"]:
            total += 8 * hkv * pages
        return {"bytes": total, "flops": 4 * hq * d * sum(lens)}
    s, t = c["start"], c["tokens"]
    return {"bytes": (s + t) * row + _pages(s + t) * (8 * hkv + 4) + 4 * t * hq * d,
            "flops": 4 * hq * d * (t * s + t * (t + 1) // 2)}


# ---- inputs ---------------------------------------------------------------------------------------


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _need(amax):
    """2^max(MIN_EXP, ceil(log2(amax / 448))), exactly: 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(amax > 0, e.clamp_min(MIN_EXP), MIN_EXP)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)  # (2^e bit by bit: a pow() may be off by a step)


def _cache(gen, chan, pages, d):
    """A layer's cache as filled by earlier steps; chan [2, hkv, d]: the channels' sizes (keys have large ones)."""
    hkv = chan.shape[1]
    kv = torch.empty((2, pages, hkv, BS, d), dtype=F8, device="cuda")
    scales = torch.empty((2, pages, hkv), device="cuda")
    for i in range(2):
        x = (_randn(gen, pages, hkv, BS, d) * chan[i][None, :, None, :]).half().float()
        scales[i] = _need(x.abs().amax((-1, -2)))
        kv[i] = (x / scales[i][..., None, None]).to(F8)
    return kv, scales


def prepare(c, seed):
    """Queries are sized so that scores have a spread of two, as a trained model's rather than a flat softmax."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 41)
    s = {"case": c}
    hkv = c["hkv"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["kind"] == "evict":
        lens = _lens(c)
        most = max(1, _pages(max(lens)))
        s["lens"] = i32(lens)
        total = sum(_pages(n) for n in lens) + 1
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        n = (s["lens"] + BS - 1) // BS
        col = torch.arange(most, device="cuda")
        at = (torch.cumsum(n, 0) - n)[:, None] + col[None, :]
        held = col[None, :] < n[:, None]
        s["table"] = torch.where(held, order[torch.where(held, at, total - 1).long()], order[-1]).to(torch.int32)
        w = torch.exp(1.5 * _randn(gen, c["batch"], hkv, most))
        s["weights"] = torch.where(held[:, None, :], w, torch.zeros_like(w))
        return s
    d = c["d"]
    chan = torch.exp(0.6 * _randn(gen, 2, hkv, d))
    chan[1] = 1.0
    if c["kind"] == "append":
        t = c["tokens"]
        if c["form"] == "step":  # each token in a page of its own, at any offset
            pages = t + 8
            off = torch.randint(0, BS, (t,), generator=gen, device="cuda")
            page = torch.randperm(pages, generator=gen, device="cuda")[:t]
        else:
            pages = _pages(c["start"] + t) + 8
            pos = torch.arange(c["start"], c["start"] + t, device="cuda")
            page, off = torch.randperm(pages, generator=gen, device="cuda")[pos // BS], pos % BS
        s["slots"] = (page * BS + off).to(torch.int32)
        s["kv"], s["scales"] = _cache(gen, chan, pages, d)
        s["k"] = (_randn(gen, t, hkv, d) * chan[0]).half()
        s["v"] = _randn(gen, t, hkv, d).half()
        return s
    hq = c["hq"]
    spread = (2.0 / chan[0]).repeat_interleave(hq // hkv, 0)
    if c["kind"] == "prefill":
        total = c["start"] + c["tokens"]
        pages = _pages(total) + 8
        s["kv"], s["scales"] = _cache(gen, chan, pages, d)
        s["table"] = torch.randperm(pages, generator=gen, device="cuda")[:_pages(total)].to(torch.int32)
        s["q"] = (_randn(gen, c["tokens"], hq, d) * spread).half()
        return s
    lens = _lens(c)
    need = [_pages(n) for n in lens]
    pages = sum(need) + 8
    s["kv"], s["scales"] = _cache(gen, chan, pages, d)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.full((c["batch"], max(need)), int(order[-1]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s["table"], s["lens"], s["max_len"] = table.cuda(), i32(lens), max(lens)
    s["q"] = (_randn(gen, c["batch"], hq, d) * spread).half()
    if c["form"] == "append":
        s["k"] = (_randn(gen, c["batch"], hkv, d) * chan[0]).half()
        s["v"] = _randn(gen, c["batch"], hkv, d).half()
    if c["weights"]:
        s["weights"] = torch.rand((c["batch"], hkv, max(need)), generator=gen, device="cuda")
    return s


# ---- one pass -------------------------------------------------------------------------------------


def run(s):
    c = s["case"]
    if c["kind"] == "evict":
        if own:
            from infurnace_amd.kernels import evict_pages
            got = evict_pages(s["table"], s["lens"], s["weights"], c["keep"], sink_pages=c["sink"],
                              recent_pages=c["recent"])
        else:
            got = _evict(s["table"], s["lens"], s["weights"], c["keep"], c["sink"], c["recent"])
        return dict(zip(("table", "lens", "weights", "evicted"), got))
    if c["kind"] == "append":
        if own:
            from infurnace_amd.kernels import store_kv_fp8
            store_kv_fp8(s["kv"], s["scales"], s["slots"], None, s["k"], s["v"])
        else:
            slots = s["slots"].long()
            _store(s["kv"], s["scales"], slots // BS, slots % BS, s["k"], s["v"])
        return {"kv": s["kv"], "scales": s["scales"]}
    if c["kind"] == "prefill":
        if own:
            from infurnace_amd.kernels import paged_attention_fp8
            return {"out": paged_attention_fp8(s["q"], s["kv"], s["scales"], s["table"], None, query_start=c["start"])}
        t = c["tokens"]
        limit = torch.arange(c["start"] + 1, c["start"] + t + 1, device="cuda")
        k, v = _gather(s["kv"], s["scales"], s["table"][None])
        return {"out": _attend(s["q"][None], k, v, limit[None])[0][0]}
    w = s.get("weights")
    if own:
        from infurnace_amd.kernels import paged_attention_fp8, store_kv_fp8_and_decode
        if c["form"] == "append":
            out = store_kv_fp8_and_decode(s["q"], s["kv"], s["scales"], s["table"], s["lens"], None, s["k"], s["v"],
                                          max_seq_len=s["max_len"], page_weights=w)
        else:
            out = paged_attention_fp8(s["q"], s["kv"], s["scales"], s["table"], s["lens"], max_seq_len=s["max_len"],
                                      page_weights=w)
    else:
        lens = s["lens"].long()
        if c["form"] == "append":
            _store_last(s["kv"], s["scales"], s["table"], lens, s["k"], s["v"], c["idle"])
        k, v = _gather(s["kv"], s["scales"], s["table"])
        out, p = _attend(s["q"][:, None], k, v, lens[:, None])
        out = out[:, 0]
        if w is not None:  # p [batch, hkv, 1 * group, keys]
            w += p.sum(2).unflatten(-1, (-1, BS)).sum(-1)
    got = {"out": out}
    if c["form"] == "append":
        got.update(kv=s["kv"], scales=s["scales"])
    if w is not None:
        got["weights"] = w
    return got


# ---- the plain forms ------------------------------------------------------------------------------


def _store(kv, scales, page, off, k, v):
    """Append row t at (page[t], off[t]); rows of one page share its block's new scale."""
    x = torch.stack((k, v)).float()  # [2, T, hkv, d]
    amax = torch.zeros_like(scales).scatter_reduce_(1, page[None, :, None].expand(2, -1, scales.shape[2]),
                                                    x.abs().amax(-1), "amax")[:, page]
    first = torch.full((scales.shape[1],), BS, device=page.device).scatter_reduce_(0, page, off, "amin")[page]
    begins = (first == 0)[None, :, None]
    before = scales[:, page]
    after = torch.where(begins, _need(amax), torch.maximum(before, _need(amax)))
    codes = kv.view(torch.uint8)
    kept = codes[:, page].view(F8).float() * (before / after)[..., None, None]
    kept = torch.where(begins[..., None, None], 0.0, kept)
    codes[:, page] = kept.to(F8).view(torch.uint8)  # (rows of one page write the same block)
    codes[:, page, :, off] = (x / after[..., None]).to(F8).view(torch.uint8).transpose(0, 1)
    scales[:, page] = after


def _store_last(kv, scales, table, lens, k, v, idle):
    """Append row b's token at position lens[b] - 1 of its table; an empty row appends nothing (its writes go to a page
    behind the others, which is dropped)."""
    last = (lens - 1).clamp_min(0)
    page = table.gather(1, (last // BS)[:, None])[:, 0].long()
    if not idle:
        return _store(kv, scales, page, last % BS, k, v)
    most = kv.shape[1]
    more = torch.cat((kv.view(torch.uint8), kv[:, :1].view(torch.uint8)), 1).view(F8)
    more_s = torch.cat((scales, scales[:, :1]), 1)
    _store(more, more_s, torch.where(lens > 0, page, most), last % BS, k, v)
    kv.copy_(more[:, :most])
    scales.copy_(more_s[:, :most])


def _gather(kv, scales, table):
    """K and V [batch, hkv, keys, d] in 32 bits of the tables' pages."""
    t = table.long()
    x = kv.view(torch.uint8)[:, t].view(F8).float() * scales[:, t][..., None, None]  # [2, B, pages, hkv, BS, d]
    x = x.transpose(2, 3).flatten(3, 4)
    return x[0], x[1]


def _attend(q, k, v, limit):
    """q [batch, n, hq, d], k and v [batch, hkv, keys, d]; query i sees keys [0, limit[:, i]).  Outputs in fp16, and the
    weights [batch, hkv, n * group, keys]."""
    b, n, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    qh = q.float().unflatten(2, (hkv, g)).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, d)
    s = torch.matmul(qh, k.transpose(-1, -2).contiguous()) / math.sqrt(d)
    hide = torch.arange(k.shape[2], device=q.device) >= limit.repeat_interleave(g, 1)[:, None, :, None]
    s = s.masked_fill_(hide, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    p /= p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p, v).reshape(b, hkv, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, hq, d)
    return o.half(), p


def _evict(table, lens, w, keep, sink, recent):
    n = ((lens + BS - 1) // BS)[:, None]
    j = torch.arange(table.shape[1], device=table.device)[None, :]
    key = w.double().sum(1).float()
    key = torch.where(torch.isnan(key), -math.inf, key).clamp(max=torch.finfo(torch.float32).max)
    key = torch.where((j < sink) | (j >= n - recent), math.inf, key)
    key = torch.where(j < n, key, -math.inf)
    rank = torch.argsort(torch.argsort(key, dim=1, descending=True, stable=True), dim=1)
    kept = (j < n) & ((n <= keep) | (rank < keep))
    order = torch.argsort(torch.where(kept, 0, torch.where(j < n, 1, 2)), dim=1, stable=True)
    left = kept.sum(1, keepdim=True)
    out_w = w.gather(2, order[:, None, :].expand_as(w))
    out_w = torch.where((j < left)[:, None, :], out_w, torch.zeros_like(out_w))
    evicted = (n - left)[:, 0].to(torch.int32)
    return table.gather(1, order), lens - BS * evicted, out_w, evicted


# ---- the same in 64 bits, from the definitions ----------------------------------------------------


def _round8(x):
    """The nearest multiple of e4m3's spacing at x (ties to even), in 64 bits: 4 significant bits, at least 2^-9 apart."""
    _, e = torch.frexp(x)
    step = (((e.long() - 4).clamp_min(-9) + 1023) << 52).view(torch.float64)
    return torch.round(x / step) * step


def _pow64(a):
    """The smallest power of two that takes a to 448 or below."""
    e = MIN_EXP
    while a > F8_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def _append64(kv, scales, writes, k, v):
    """writes: {page: [(offset, row of k and v)]}; kv and scales in 64 bits, changed in place."""
    page = torch.tensor(list(writes), device="cuda")
    for i, x in enumerate((k.double(), v.double())):
        tops = x.abs().amax(-1).cpu().tolist()
        for at, rows in writes.items():
            new = [_pow64(max(tops[r][h] for _, r in rows)) for h in range(x.shape[1])]
            new = torch.tensor(new, dtype=torch.float64, device="cuda")
            if min(o for o, _ in rows) == 0:
                kv[i, at] = 0.0
            else:
                new = torch.maximum(new, scales[i, at])
                kv[i, at] = _round8(kv[i, at] * (scales[i, at] / new)[:, None, None])
            scales[i, at] = new
            where = torch.tensor([o for o, _ in rows], device="cuda")
            kv[i, at][:, where] = _round8(x[[r for _, r in rows]] / new[None, :, None]).transpose(0, 1)
    return page


def _attend64(q, k, v, first):
    """q [n, hq, d], k and v [hkv, keys, d] in 64 bits; query i sees first + i keys."""
    n, hq, d = q.shape
    g = hq // k.shape[0]
    out, weights = torch.empty_like(q), []
    for h in range(k.shape[0]):
        total = torch.zeros(k.shape[1], dtype=torch.float64, device="cuda")
        for at in range(0, n, 512):
            part = q[at:at + 512, h * g:(h + 1) * g]
            s = torch.matmul(part, k[h].t()) / math.sqrt(d)
            seen = first + at + torch.arange(part.shape[0], device="cuda")
            s = s.masked_fill(torch.arange(k.shape[1], device="cuda")[None, None, :] >= seen[:, None, None], -math.inf)
            p = torch.softmax(s, -1)
            out[at:at + 512, h * g:(h + 1) * g] = torch.matmul(p, v[h])
            total += p.sum((0, 1))
        weights.append(total)
    return out, torch.stack(weights)


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "evict":  # (whole numbers are compared as they are)
        w = s["weights"].double()
        total, out = w.sum(1).cpu(), torch.zeros_like(w)
        for b, n in enumerate(_lens(c)):
            pages = list(range(_pages(n)))
            if len(pages) > c["keep"]:
                mid = sorted(pages[c["sink"]:len(pages) - c["recent"]], key=lambda j: -float(total[b, j]))
                mid = mid[:c["keep"] - c["sink"] - c["recent"]]
                pages = sorted(pages[:c["sink"]] + mid + pages[len(pages) - c["recent"]:])
            out[b, :, :len(pages)] = w[b][:, pages]
        return {"table": None, "lens": None, "weights": out, "evicted": None}
    if c["kind"] in ("append", "decode"):
        kv, scales = s["kv"].double(), s["scales"].double()
    if c["kind"] == "append":
        writes = {}
        for t, slot in enumerate(s["slots"].tolist()):
            writes.setdefault(slot // BS, []).append((slot % BS, t))
        _append64(kv, scales, writes, s["k"], s["v"])
        return {"kv": kv, "scales": scales}
    if c["kind"] == "prefill":
        at = s["table"].long()
        x = s["kv"].view(torch.uint8)[:, at].view(F8).double() * s["scales"][:, at].double()[..., None, None]
        x = x.transpose(1, 2).flatten(2, 3)[:, :, :c["start"] + c["tokens"]]
        return {"out": _attend64(s["q"].double(), x[0], x[1], c["start"] + 1)[0]}
    table, lens = s["table"].tolist(), _lens(c)
    if c["form"] == "append":
        writes = {table[b][(n - 1) // BS]: [((n - 1) % BS, b)] for b, n in enumerate(lens) if n}
        _append64(kv, scales, writes, s["k"], s["v"])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    w = s["weights"].double() if c["weights"] else None
    for b, n in enumerate(lens):
        if not n:
            continue
        at = s["table"][b, :_pages(n)].long()
        x = (kv[:, at] * scales[:, at][..., None, None]).transpose(1, 2).flatten(2, 3)[:, :, :n]
        o, total = _attend64(s["q"][b:b + 1].double(), x[0], x[1], n)
        out[b] = o[0]
        if w is not None:
            full = torch.zeros((total.shape[0], _pages(n) * BS), dtype=torch.float64, device="cuda")
            full[:, :n] = total
            w[b, :, :_pages(n)] += full.unflatten(-1, (-1, BS)).sum(-1)
    got = {"out": out}
    if c["form"] == "append":
        got.update(kv=kv, scales=scales)
    if w is not None:
        got["weights"] = w
    return got
