"""Refusals of the 8-bit cache's and the eviction's calls, on the host: nothing is launched."""
import pytest
import torch

from fp8_util import F8
from infurnace_amd import _capi
from infurnace_amd.kernels import (KVStoreError, PagedAttentionError, evict_pages, paged_attention_fp8, store_kv_fp8,
                                   store_kv_fp8_and_decode)
from infurnace_amd.kernels.kv_fp8 import _validate_slots

A = 0x10000  # a 16-byte-aligned fake device address; never dereferenced (validation fails first)


def test_store_entry_point():
    L = _capi.lib()
    ok = dict(c=A, s=A, P=64, sm=A, am=None, k=A, v=A, T=4, hkv=8, d=128, bs=16)

    def call(**kw):
        a = {**ok, **kw}
        return L.ifn_store_kv_fp8(a["c"], a["s"], a["P"], a["sm"], a["am"], a["k"], a["v"], a["T"], a["hkv"], a["d"],
                                  a["bs"], None)
    for name in ("c", "s", "sm", "k", "v"):
        assert call(**{name: None}) == _capi.IFN_ERR_INVALID_ARGUMENT
    for kw in (dict(P=0), dict(T=-1), dict(hkv=0), dict(d=0), dict(bs=0)):
        assert call(**kw) == _capi.IFN_ERR_INVALID_ARGUMENT
    for kw in (dict(d=96), dict(d=512), dict(bs=32), dict(P=1 << 28)):
        assert call(**kw) == _capi.IFN_ERR_UNSUPPORTED
    for name in ("c", "k", "v"):
        assert call(**{name: A + 8}) == _capi.IFN_ERR_ALIGNMENT
    assert call(T=0) == _capi.IFN_OK


@pytest.mark.parametrize("append", [False, True])
def test_decode_entry_points(append):
    L = _capi.lib()
    ok = dict(out=A, q=A, c=A, s=A, P=64, bt=A, W=32, sl=A, am=None, k=A, v=A, pw=None, B=4, hq=16, hkv=8, d=128, bs=16,
              msl=512, scale=0.0, ws=None, wsb=0)

    def call(**kw):
        a = {**ok, **kw}
        head = [a[x] for x in ("out", "q", "c", "s", "P", "bt", "W", "sl", "am")]
        tail = [a[x] for x in ("pw", "B", "hq", "hkv", "d", "bs", "msl", "scale", "ws", "wsb")]
        if append:
            return L.ifn_paged_decode_append_fp8(*head, a["k"], a["v"], *tail, None)
        return L.ifn_paged_decode_fp8(*head, *tail, None)
    for name in ("out", "q", "c", "s", "bt", "sl") + (("k", "v") if append else ()):
        assert call(**{name: None}) == _capi.IFN_ERR_INVALID_ARGUMENT
    for kw in (dict(B=-1), dict(hq=12), dict(hq=0), dict(P=0), dict(W=0), dict(msl=-1)):
        assert call(**kw) == _capi.IFN_ERR_INVALID_ARGUMENT
    for kw in (dict(d=96), dict(bs=32), dict(hq=17, hkv=1), dict(B=5000), dict(B=4096, hq=32, hkv=32)):
        assert call(**kw) == _capi.IFN_ERR_UNSUPPORTED
    # (states, offsets and page sums that shared memory does not hold)
    assert call(B=4096, hq=16, hkv=1, d=256, pw=A) == _capi.IFN_ERR_UNSUPPORTED
    assert call(B=4096, hq=16, hkv=1, d=256) == _capi.IFN_ERR_WORKSPACE
    for name in ("out", "q", "c") + (("k", "v") if append else ()):
        assert call(**{name: A + 8}) == _capi.IFN_ERR_ALIGNMENT
    assert call(B=0) == _capi.IFN_OK
    assert call() == _capi.IFN_ERR_WORKSPACE
    need = L.ifn_paged_decode_fp8_workspace_bytes(4, 16, 8, 128, 16, 32, 512, 0)
    with_weights = L.ifn_paged_decode_fp8_workspace_bytes(4, 16, 8, 128, 16, 32, 512, 1)
    assert with_weights > need > 0
    assert call(ws=A, wsb=need - 1) == _capi.IFN_ERR_WORKSPACE
    assert call(ws=A, wsb=need, pw=A) == _capi.IFN_ERR_WORKSPACE
    assert L.ifn_paged_decode_fp8_workspace_bytes(-1, 16, 8, 128, 16, 32, 512, 0) == 0


def test_prefill_entry_point():
    L = _capi.lib()
    ok = dict(out=A, q=A, c=A, s=A, P=64, bt=A, W=32, qs=0, T=16, hq=16, hkv=8, d=128, bs=16, scale=0.0,
              ws=A, wsb=1 << 40)

    def call(**kw):
        a = {**ok, **kw}
        return L.ifn_paged_prefill_fp8(*[a[x] for x in ok], None)
    for name in ("out", "q", "c", "s", "bt"):
        assert call(**{name: None}) == _capi.IFN_ERR_INVALID_ARGUMENT
    for kw in (dict(T=-1), dict(qs=-1), dict(hq=12), dict(qs=500), dict(P=0)):
        assert call(**kw) == _capi.IFN_ERR_INVALID_ARGUMENT
    for kw in (dict(d=256), dict(bs=8)):
        assert call(**kw) == _capi.IFN_ERR_UNSUPPORTED
    assert call(out=A + 2) == _capi.IFN_ERR_ALIGNMENT
    assert call(T=0) == _capi.IFN_OK
    assert call(ws=None) == _capi.IFN_ERR_WORKSPACE and call(wsb=64) == _capi.IFN_ERR_WORKSPACE
    assert L.ifn_paged_prefill_fp8_workspace_bytes(16, -1, 16, 8, 128, 16) == 0


def test_evict_entry_point():
    L = _capi.lib()
    names = ("ot", "ol", "ow", "ne", "bt", "W", "sl", "am", "pw", "B", "hkv", "bs", "keep", "sink", "recent")
    ok = dict(zip(names, (A, A, A, A, A, 32, A, None, A, 4, 8, 16, 8, 1, 1)))

    def call(**kw):
        a = {**ok, **kw}
        return L.ifn_evict_pages(*[a[x] for x in names], None)
    for name in ("ot", "ol", "ow", "ne", "bt", "sl", "pw"):
        assert call(**{name: None}) == _capi.IFN_ERR_INVALID_ARGUMENT
    for kw in (dict(B=-1), dict(W=0), dict(hkv=0), dict(recent=0), dict(sink=-1), dict(keep=1), dict(sink=2 ** 31 - 1)):
        assert call(**kw) == _capi.IFN_ERR_INVALID_ARGUMENT
    for kw in (dict(bs=32), dict(W=32769)):
        assert call(**kw) == _capi.IFN_ERR_UNSUPPORTED
    assert call(B=0) == _capi.IFN_OK


def _cache(**kw):
    return (torch.zeros((2, 8, 2, 16, 64), dtype=kw.get("dtype", F8)), torch.ones((2, 8, 2)))


def test_wrappers_refuse():
    """The wrappers' own checks come first, on any device (these tensors are on the host)."""
    kv, sc = _cache()
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    h = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    with pytest.raises(KVStoreError, match="GPU tensor"):
        store_kv_fp8(kv, sc, i(3), None, h(3, 2, 64), h(3, 2, 64))
    with pytest.raises(KVStoreError, match="float8"):
        store_kv_fp8(*_cache(dtype=torch.float16), i(3), None, h(3, 2, 64), h(3, 2, 64))
    with pytest.raises(KVStoreError, match="scales shape"):
        store_kv_fp8(kv, sc[:, :4], i(3), None, h(3, 2, 64), h(3, 2, 64))
    with pytest.raises(KVStoreError, match="rank"):
        store_kv_fp8(kv[0], sc[0], i(3), None, h(3, 2, 64), h(3, 2, 64))
    with pytest.raises(KVStoreError, match="scales dtype"):
        store_kv_fp8(kv, sc.half(), i(3), None, h(3, 2, 64), h(3, 2, 64))
    with pytest.raises(KVStoreError, match="contiguous"):
        store_kv_fp8(kv.transpose(1, 2), sc.transpose(1, 2), i(3), None, h(3, 2, 64), h(3, 2, 64))
    with pytest.raises(PagedAttentionError, match="GPU tensor"):
        paged_attention_fp8(h(1, 4, 64), kv, sc, i(1, 4), i(1))
    with pytest.raises(PagedAttentionError, match="GPU tensor"):
        paged_attention_fp8(h(1, 4, 64), kv, sc, i(4), None, query_start=0)
    with pytest.raises(PagedAttentionError, match="GPU tensor"):
        store_kv_fp8_and_decode(h(1, 4, 64), kv, sc, i(1, 4), i(1), None, h(1, 2, 64), h(1, 2, 64))
    with pytest.raises(PagedAttentionError, match="GPU tensor"):
        evict_pages(i(1, 4), i(1), torch.zeros((1, 2, 4)), 2)


def test_validate_slots():
    s = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    _validate_slots(s([0, 1, 2, 40]), None, 64)
    _validate_slots(s([-1, 500, 2]), torch.tensor([0, 0, 1]), 64)
    with pytest.raises(KVStoreError, match="outside"):
        _validate_slots(s([0, 64]), None, 64)
    with pytest.raises(KVStoreError, match="same slot"):
        _validate_slots(s([3, 5, 3]), None, 64)
    _validate_slots(s([0] + list(range(16, 200)) + [1]), None, 256)  # (a page's tokens may be any distance apart)
