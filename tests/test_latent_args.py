"""The C ABI of rope, kv_write / kv_read and mla_attend on the CPU: what is
refused, before anything of a device is needed, and the rotation table."""
import copy
import ctypes
import math

import pytest

from flash_deepseek_amd import _lib

INVAL, STATE = _lib.FDM_E_INVAL, _lib.FDM_E_STATE
P = 1 << 20  # an aligned address that is never read


def table(dim=64, layout=0, scaling=0, orig=4096, base=10000.0, factor=1.0, fast=32.0, slow=1.0, mul=1.0):
    t = _lib.RopeTable()
    rc = _lib.lib.fdm_rope_table_init(ctypes.byref(_lib.RopeParams(dim, layout, scaling, orig, base, factor, fast, slow, mul)), ctypes.byref(t))
    return rc, t


@pytest.mark.parametrize("scaling,factor", [(0, 1.0), (1, 4.0), (2, 40.0), (2, 8.0)])
@pytest.mark.parametrize("dim", [2, 18, 64, 128, 256])
def test_table_holds_the_frequencies(dim, scaling, factor):
    from tests.latent_case import frequencies
    rc, t = table(dim, scaling=scaling, factor=factor)
    assert rc == 0 and t.dim == dim and t.mul == 1.0
    want = frequencies(dim, scaling=("none", "linear", "yarn")[scaling], factor=factor)
    for i in range(dim // 2):
        got = t.turns[i] / 2.0 ** 64 * 2.0 * math.pi
        # the double reference: a few of its roundings; the table: cut to 2^-64 of a turn
        assert abs(got - float(want[i])) < 2.0 ** -48 * float(want[i]) + 2.0 ** -64 * 2.0 * math.pi


@pytest.mark.parametrize("bad", [dict(dim=0), dict(dim=3), dict(dim=258), dict(layout=2), dict(layout=-1), dict(scaling=3),
                                 dict(base=1.0), dict(base=math.nan), dict(base=math.inf), dict(scaling=1, factor=0.5),
                                 dict(scaling=2, factor=math.nan), dict(scaling=2, orig=0), dict(scaling=2, slow=0.0),
                                 dict(scaling=2, fast=math.inf), dict(mul=math.nan)])
def test_table_refusals(bad):
    assert table(**bad)[0] == INVAL


ROPE = dict(table=None, pos=P, T=2, H=4, D=64, offset=0, x=P, xt=0, x0=256, x1=64, y=2 * P, yt=0, y0=256, y1=64, stream=None)


def rope(**kw):
    a = {**ROPE, **kw}
    if a["table"] is None:
        a["table"] = table()[1]
    return _lib.lib.fdm_rope(ctypes.byref(a.pop("table")), *a.values())


@pytest.mark.parametrize("bad", [dict(T=-1), dict(H=0), dict(H=4097), dict(D=0), dict(D=4097), dict(D=63), dict(offset=-1), dict(offset=1),
                                 dict(xt=2), dict(yt=12), dict(pos=None), dict(x=None), dict(y=None), dict(x=P + 2), dict(pos=P + 1),
                                 dict(y=P, y0=512), dict(y=P, yt=1), dict(y0=64), dict(y1=63), dict(y0=0, y1=64), dict(y1=32),
                                 dict(table=_lib.RopeTable(63, 0)), dict(table=_lib.RopeTable(64, 2))])
def test_rope_refusals(bad):
    assert rope(**bad) == INVAL


CACHE = dict(latent=P, rope=P, scale=None, format=1, n_pages=4, page_size=16)
BAD_CACHES = [dict(latent=None), dict(rope=None), dict(latent=P + 8), dict(rope=P + 8), dict(format=3), dict(format=-1), dict(n_pages=0),
              dict(page_size=0), dict(page_size=24), dict(n_pages=1 << 27), dict(format=2), dict(format=2, scale=P + 2)]


def cache(**kw):
    return ctypes.byref(_lib.KvCacheDesc(*{**CACHE, **kw}.values()))


def write(c=None, x=P, xt=0, stride=576, w=None, t=None, pos=None, slots=P, T=2):
    return _lib.lib.fdm_kv_write(cache() if c is None else c, x, xt, stride, w, t, pos, slots, T, None)


def read(c=None, slots=P, T=2, y=P, yt=0, stride=576):
    return _lib.lib.fdm_kv_read(cache() if c is None else c, slots, T, y, yt, stride, None)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_cache_refusals(bad):
    assert write(cache(**bad)) == INVAL and read(cache(**bad)) == INVAL
    assert attend(c=cache(**bad)) == INVAL


def test_write_and_read_refusals():
    t = ctypes.byref(table()[1])
    for bad in (dict(x=None), dict(slots=None), dict(xt=12), dict(T=-1), dict(T=(1 << 25) + 1), dict(x=P + 1), dict(slots=P + 2), dict(t=t), dict(w=P + 2),
                dict(t=t, pos=P + 2), dict(t=ctypes.byref(table(32)[1]), pos=P)):
        assert write(**bad) == INVAL, bad
    for bad in (dict(y=None), dict(slots=None), dict(yt=12), dict(T=-1), dict(T=(1 << 25) + 1), dict(y=P + 2), dict(stride=575), dict(stride=0)):
        assert read(**bad) == INVAL, bad
    assert _lib.lib.fdm_kv_write(None, P, 0, 576, None, None, None, P, 2, None) == INVAL


BATCH = dict(B=2, N=3, H=4, q_start=P, kv_len=P, pages=P, pages_stride=4, mask=None, mask_words=0)
CALL = dict(ql=P, ql0=2048, ql1=512, qr=P, qr0=256, qr1=64, scale=0.1, out=2 * P, o0=2048, o1=512, lse=None, ws=P, size=1 << 40, stream=None)


def attend(c=None, **kw):
    batch = _lib.MlaBatch(*{k: kw.pop(k, v) for k, v in BATCH.items()}.values())
    return _lib.lib.fdm_mla_attend(cache() if c is None else c, ctypes.byref(batch), *{**CALL, **kw}.values())


@pytest.mark.parametrize("bad", [dict(B=0), dict(B=513), dict(N=-1), dict(N=(1 << 20) + 1), dict(H=0), dict(H=129), dict(pages_stride=0),
                                 dict(mask=P), dict(mask_words=1), dict(mask=P, mask_words=-1), dict(mask=P + 4, mask_words=1),
                                 dict(q_start=None), dict(kv_len=None), dict(pages=None), dict(ql=None), dict(qr=None), dict(out=None),
                                 dict(ws=None), dict(ws=P + 128), dict(ql=P + 8), dict(qr=P + 8), dict(out=P + 8), dict(ql0=2052),
                                 dict(ql1=516), dict(qr0=260), dict(qr1=4), dict(o0=2044), dict(o1=511), dict(o1=504), dict(o0=512),
                                 dict(scale=math.nan), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(lse=P + 2)])
def test_attend_refusals(bad):
    assert attend(**bad) == INVAL


def test_good_arguments_get_as_far_as_the_device():
    if _lib.lib.fdm_available():
        pytest.skip("library already initialised in this process")
    assert rope() == STATE and write() == STATE and read() == STATE and attend() == STATE
    assert write(t=ctypes.byref(table()[1]), pos=P, w=P) == STATE
    assert rope(y=P) == STATE and rope(T=0, x=None) == STATE and attend(N=0, ql=None) == STATE
    assert _lib.lib.fdm_mla_workspace(4, 128, ctypes.byref(ctypes.c_size_t())) == STATE
    assert _lib.lib.fdm_mla_workspace(4, 129, ctypes.byref(ctypes.c_size_t())) == INVAL
    assert copy.copy(table()[1]).dim == 64


def test_a_cache_of_another_device(monkeypatch):
    """The planes' device is the one that they were given with, whatever the library's is now."""
    import types

    import torch

    import flash_deepseek_amd as fdm
    elsewhere = types.SimpleNamespace(device=1, half=torch.bfloat16)
    monkeypatch.setattr(fdm, "_device", 0)
    x, q, r = torch.zeros(2, 576), torch.zeros(2, 4, 512, dtype=torch.bfloat16), torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: fdm.kv_write(elsewhere, x, i), lambda: fdm.kv_read(elsewhere, i, x),
                 lambda: fdm.mla_attend(elsewhere, q, r, i, i[:1], i[None], 1.0, q)):
        with pytest.raises(fdm.FdmError, match="the cache is on device 1"):
            call()
