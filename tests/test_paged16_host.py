"""Refusals of the 16-bit paged layer's entry points that need no GPU: the C
ABI's host validation and the Python layer's argument checks."""
import ctypes

import numpy as np
import pytest
import torch

from oscar_b200 import _native, kernels

I32 = ctypes.c_int32
FAKE = 1 << 20  # a 16-byte aligned address that validation never follows


@pytest.fixture(scope="module")
def lib():
    from oscar_b200 import build

    build.build()
    return _native.lib()


def ints(*values):
    return (I32 * len(values))(*values)


def rope(lib, **kw):
    a = dict(q=FAKE, qt=6144, qh=256, k=FAKE, kt=1024, kh=256, v=FAKE, vt=1024, vh=256, dtype=1, n=4, hq=24, hk=4, d=256,
             wq=FAKE, wk=FAKE, wdt=1, eps=1e-6, offset=0.0, cs=FAKE, csdt=0, css=64, maxpos=10, rot=64, inter=0, pos=FAKE,
             oq=FAKE, oqt=6144, oqh=256, ok=None, okt=0, okh=0, kc=FAKE, vc=FAKE, nb=2, bs=16, kb=16384, kk=1024, kkh=256,
             vb=16384, vv=1024, vvh=256, slots=FAKE)
    a.update(kw)
    return lib.oscar_qk_norm_rope(*a.values(), None)


def attention(lib, qsl=(0, 3), seqs=(5,), **kw):
    a = dict(q=FAKE, qt=6144, qh=256, dtype=1, n=3, hq=24, hk=4, d=256, kc=FAKE, vc=FAKE, nb=2, bs=16, kb=16384, kt=1024,
             kh=256, vb=16384, vt=1024, vh=256, bt=FAKE, rows=1, cols=1, stride=1, qsl=ints(*qsl), seqs=ints(*seqs),
             num=len(seqs), scale=0.1, w=None, observe=1, out=FAKE, lse=FAKE, ws=FAKE, wsb=0)
    a.update(kw)
    return lib.oscar_paged_attention(*a.values(), None)


def evict(lib, seqs=(5,), **kw):
    a = dict(kc=FAKE, vc=FAKE, d=256, nb=2, bs=16, hk=4, kb=16384, kt=1024, kh=256, vb=16384, vt=1024, vh=256, w=FAKE,
             bt=FAKE, rows=1, cols=1, stride=1, dst=None, drows=0, dcols=0, dstride=0, seqs=ints(*seqs), num=len(seqs),
             keep=3, sink=1, recent=1, kept=FAKE, kcols=3)
    a.update(kw)
    return lib.oscar_evict_cache(*a.values(), None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=0), 2, b"bf16 or fp16"), (dict(d=96), 2, b"64, 128, 256"), (dict(rot=24), 1, b"multiple of 16"),
    (dict(rot=272), 1, b"multiple of 16"), (dict(wdt=2), 2, b"fp32 or of the heads' type"), (dict(eps=-1.0), 1, b"eps"),
    (dict(eps=float("nan")), 1, b"eps"), (dict(vc=None), 1, b"come together"), (dict(slots=None), 1, b"come together"),
    (dict(kc=None, vc=None, slots=None), 1, b"no destination"), (dict(q=FAKE + 2), 1, b"16-byte"),
    (dict(qt=6145), 1, b"16-byte"), (dict(kk=1028), 1, b"16-byte"), (dict(kkh=64), 1, b"overlap"), (dict(pos=None), 1, b"null"),
    (dict(n=-1), 1, b"geometry"), (dict(v=None), 1, b"null"), (dict(css=48), 1, b"16-byte"),
])
def test_qk_norm_rope_refusals(lib, kw, status, text):
    assert rope(lib, **kw) == status
    assert text in lib.oscar_last_error()
    with pytest.raises(ValueError):
        _native.check(status)


@pytest.mark.parametrize("kw", [
    dict(oqh=128), dict(oqt=256), dict(oqt=0), dict(oqh=0), dict(oqt=23 * 256 + 248), dict(ok=FAKE, okt=0, okh=256),
    dict(ok=FAKE, okt=1024, okh=248), dict(oqt=256, oqh=768),
])
def test_overlapping_outputs_are_refused(lib, kw):
    assert rope(lib, **kw) == 1 and b"output rows overlap" in lib.oscar_last_error()


def test_outputs_in_any_order_are_accepted(lib):
    n = 2**31  # refused before anything is launched, but only after the outputs
    for kw in (dict(oqt=6144), dict(oqt=256, oqh=256 * n), dict(hq=1, hk=1, oqt=256, oqh=0, kkh=0),
               dict(ok=FAKE, okt=256, okh=256 * n)):
        assert rope(lib, n=n, **kw) == 2 and b"too many tokens" in lib.oscar_last_error()


def test_nothing_to_do_is_accepted(lib):
    assert rope(lib, n=0) == 0
    assert attention(lib, qsl=(0, 0), n=0) == 0
    assert evict(lib, seqs=(0, 0), rows=2) == 0
    assert lib.oscar_paged_attention_workspace(ints(0), None, 0, 24, 4, 256, 0) == 0


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=0), 2, b"bf16 or fp16"), (dict(d=80), 2, b"64, 128, 256"), (dict(hq=23), 1, b"multiple of Hk"),
    (dict(hq=520), 2, b"group 130 > 128"),
    (dict(qsl=(0, 2)), 1, b"query layout"), (dict(qsl=(1, 3)), 1, b"query layout"), (dict(qsl=(0, 4, 3), seqs=(5, 5)), 1, b"fall"),
    (dict(seqs=(-1,)), 1, b"negative"), (dict(scale=0.0), 1, b"scale"), (dict(scale=float("inf")), 1, b"scale"),
    (dict(seqs=(17,)), 1, b"cannot cover"), (dict(rows=0), 1, b"block-table rows"), (dict(bt=None), 1, b"block table"),
    (dict(w=FAKE, observe=0), 1, b"observe"), (dict(q=None), 1, b"null"), (dict(kt=1001), 1, b"16-byte"),
    (dict(vb=128), 1, b"overlap"), (dict(nb=0), 1, b"caches"), (dict(bs=0), 1, b"geometry"), (dict(out=FAKE + 8), 1, b"16-byte"),
])
def test_paged_attention_refusals(lib, kw, status, text):
    assert attention(lib, **kw) == status
    assert text in lib.oscar_last_error()


def test_lengths_that_32_bits_of_positions_do_not_hold(lib):
    top = 2**31 - 1
    wide = dict(cols=2**27, stride=2**27)
    assert evict(lib, seqs=(5, top), rows=2, **wide) == 2 and b"request 1 too long" in lib.oscar_last_error()
    assert evict(lib, seqs=(2**30 + 1,), **wide) == 2
    for seqs in ((top,), (2**30 + 1,)):
        assert attention(lib, seqs=seqs, **wide) == 2 and b"too long" in lib.oscar_last_error()
        assert lib.oscar_paged_attention_workspace(ints(0, 3), ints(*seqs), 1, 24, 4, 256, 0) < 0
    # a prompt of 2^26 tokens; one of 2^20 fits
    assert lib.oscar_paged_attention_workspace(ints(0, 2**26), ints(2**26), 1, 24, 4, 256, 0) < 0
    assert lib.oscar_paged_attention_workspace(ints(0, 2**20), ints(2**20), 1, 24, 4, 256, 0) > 0
    # many heads
    assert lib.oscar_paged_attention_workspace(ints(0, 1), ints(2**29), 1, 512, 256, 64, 0) < 0


def test_wait_limit(lib):
    assert lib.oscar_set_wait_limit(-2) == 1
    assert b"wait limit" in lib.oscar_last_error()
    assert lib.oscar_set_wait_limit(5) == 0 and lib.oscar_set_wait_limit(-1) == 0


def test_out_over_the_queries_where_keys_are_weighed(lib):
    long = dict(qsl=(0, 9), seqs=(16,), n=9, wsb=0)
    for out in (FAKE, FAKE + 9 * 6144 * 2 - 32, FAKE - 9 * 6144 * 2 + 32):
        assert attention(lib, out=out, w=FAKE, **long) == 1 and b"overlap q" in lib.oscar_last_error()
    for kw in (dict(out=FAKE, w=None), dict(out=FAKE + 9 * 6144 * 2, w=FAKE), dict(out=FAKE - 9 * 6144 * 2, w=FAKE)):
        attention(lib, **kw, **long)  # (goes on to what needs a GPU)
        assert b"overlap q" not in lib.oscar_last_error()


@pytest.mark.parametrize("lens,seqs,hq,hk,d", [
    ([4] * 64, [32768] * 64, 24, 4, 256), ([4] * 256, [24580] * 256, 24, 4, 256), ([1, 4] * 200, [100000] * 400, 32, 8, 128),
    ([4], [2**22], 24, 4, 256), ([1] * 3, [2**23, 100, 2**20], 64, 16, 64), ([8192, 4, 70], [17448, 10**6, 10**6], 24, 4, 256),
])
def test_workspace_is_bounded(lib, lens, seqs, hq, hk, d):
    qsl = np.concatenate([[0], np.cumsum(lens)])
    need = [lib.oscar_paged_attention_workspace(ints(*qsl), ints(*seqs), len(seqs), hq, hk, d, weighted) for weighted in (0, 1)]
    assert 0 < need[0] < need[1] <= (320 << 20) + 8 * hq * int(qsl[-1])


def test_workspace_of_invalid_lists(lib):
    assert lib.oscar_paged_attention_workspace(ints(0, 4, 3), ints(1, 1), 2, 24, 4, 256, 0) < 0
    assert lib.oscar_paged_attention_workspace(ints(0, 4), ints(9), 1, 24, 5, 256, 0) < 0
    plain = lib.oscar_paged_attention_workspace(ints(0, 4), ints(900), 1, 24, 4, 256, 0)
    assert 0 < plain < lib.oscar_paged_attention_workspace(ints(0, 4), ints(900), 1, 24, 4, 256, 1)


@pytest.mark.parametrize("kw,status,text", [
    (dict(d=32), 2, b"64, 128, 256"), (dict(keep=0), 1, b"keep"), (dict(sink=3), 1, b"keep"), (dict(recent=-1), 1, b"keep"),
    (dict(seqs=(-2,)), 1, b"negative"), (dict(seqs=(17,)), 1, b"cannot cover"), (dict(kcols=2), 1, b"places"),
    (dict(dst=FAKE, drows=1, dcols=0, dstride=0), 1, b"destination"), (dict(rows=0), 1, b"block-table rows"),
    (dict(w=None), 1, b"null"), (dict(kept=None), 1, b"null"), (dict(vt=1004), 1, b"16-byte"), (dict(hk=0), 1, b"geometry"),
])
def test_evict_refusals(lib, kw, status, text):
    assert evict(lib, **kw) == status
    assert text in lib.oscar_last_error()


def test_python_layer_refusals():
    q, k = torch.zeros(2, 24, 256, dtype=torch.bfloat16), torch.zeros(2, 4, 256, dtype=torch.bfloat16)
    cache = torch.zeros(2, 16, 4, 256, dtype=torch.bfloat16)
    w = torch.ones(256)
    table = torch.zeros(1, 1, dtype=torch.int32)
    weights = torch.zeros(2, 4, 16)
    pos = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.qk_norm_rope(q, k, None, w, w, 1e-6, torch.zeros(4, 64), pos)
    with pytest.raises(ValueError, match="one type"):
        kernels.qk_norm_rope(q, k.half(), None, w, w, 1e-6, torch.zeros(4, 64), pos)
    with pytest.raises(ValueError, match="come together"):
        kernels.qk_norm_rope(q, k, None, w, w, 1e-6, torch.zeros(4, 64), pos, k_cache=cache, v_cache=cache, slot_mapping=pos)
    with pytest.raises(ValueError, match="unsupported type"):
        kernels.qk_norm_rope(q.float(), k.float(), None, w, w, 1e-6, torch.zeros(4, 64), pos)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.paged_attention(q, cache, cache, table, [0, 2], [5], 0.1)
    with pytest.raises(ValueError, match="multiple"):
        kernels.paged_attention(q[:, :23], cache, cache, table, [0, 2], [5], 0.1)
    with pytest.raises(ValueError, match="unsupported query type"):
        kernels.paged_attention(q.float(), cache, cache, table, [0, 2], [5], 0.1)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.evict_cache(cache, cache, weights, table, [5], 3)
    with pytest.raises(ValueError, match="unsupported cache type"):
        kernels.evict_cache(cache.float(), cache.float(), weights, table, [5], 3)


@pytest.mark.gpu
def test_python_layer_refusals_on_device():
    dev = torch.device("cuda", 0)
    q = torch.zeros(2, 24, 256, dtype=torch.bfloat16, device=dev)
    cache = torch.zeros(2, 16, 4, 256, dtype=torch.bfloat16, device=dev)
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    call = lambda **kw: kernels.paged_attention(  # noqa: E731
        **{**dict(q=q, k_cache=cache, v_cache=cache, table=table, qsl=[0, 2], seqs=[5], scale=0.1), **kw})
    with pytest.raises(ValueError, match="heads' type"):
        call(k_cache=cache.half(), v_cache=cache.half())
    with pytest.raises(ValueError, match="alike"):
        call(v_cache=cache[:1])
    with pytest.raises(ValueError, match="query layout"):
        call(qsl=[0, 1])
    with pytest.raises(ValueError, match="cannot cover"):
        call(seqs=[17])
    with pytest.raises(ValueError, match="weights must be"):
        call(weights=torch.zeros(2, 16, 4, device=dev))
    with pytest.raises(ValueError, match="observe"):
        call(observe=4)
    with pytest.raises(ValueError, match="out must be"):
        call(out=q.float())
    with pytest.raises(ValueError, match="fall"):
        call(qsl=np.array([0, 3, 2], np.int32), seqs=[5, 5], table=table.repeat(2, 1))
    with pytest.raises(ValueError, match="keep"):
        kernels.evict_cache(cache, cache, torch.zeros(2, 4, 16, device=dev), table, [5], 3, sink=2, recent=2)
    with pytest.raises(ValueError, match="weights must be"):
        kernels.evict_cache(cache, cache, torch.zeros(2, 16, 4, device=dev), table, [5], 3)
    with pytest.raises(ValueError, match="multiple of 16"):
        kernels.qk_norm_rope(q, q[:, :4], None, torch.ones(256, device=dev), torch.ones(256, device=dev), 1e-6,
                             torch.zeros(4, 24, device=dev), torch.zeros(2, dtype=torch.int64, device=dev))
