"""The C ABI of kv_grow / kv_trim, add_rms_norm and project on the CPU: what is
refused, before anything of a device is needed."""
import ctypes
import math

import pytest

from flash_deepseek_amd import _lib

INVAL, STATE = _lib.FDM_E_INVAL, _lib.FDM_E_STATE
P = 1 << 20  # an aligned address that is never read
F32, F16, BF16, E4M3 = _lib.GGML_F32, _lib.GGML_F16, _lib.GGML_BF16, _lib.E4M3

PAGES = dict(pages=P, kv_len=P, free=P, n_free=P, turn=P, B=4, pages_stride=8, n_pages=40, page_size=16)


def pages(**kw):
    return ctypes.byref(_lib.KvPagesDesc(*{**PAGES, **kw}.values()))


def grow(p=None, new=P, N=10, q=P, pos=P, slots=P, refused=None):
    return _lib.lib.fdm_kv_grow(pages() if p is None else p, new, N, q, pos, slots, refused, None)


def trim(p=None, keep=P):
    return _lib.lib.fdm_kv_trim(pages() if p is None else p, keep, None)


@pytest.mark.parametrize("bad", [dict(pages=None), dict(kv_len=None), dict(free=None), dict(n_free=None), dict(turn=None), dict(pages=P + 2),
                                 dict(n_free=P + 1), dict(B=0), dict(B=4097), dict(pages_stride=0), dict(B=4096, pages_stride=1 << 19),
                                 dict(n_pages=0), dict(page_size=0), dict(page_size=24), dict(n_pages=1 << 27)])
def test_pages_refusals(bad):
    assert grow(pages(**bad)) == INVAL and trim(pages(**bad)) == INVAL


def test_grow_and_trim_refusals():
    for bad in (dict(new=None), dict(q=None), dict(pos=None), dict(slots=None), dict(N=-1), dict(N=(1 << 25) + 1), dict(new=P + 2), dict(q=P + 1),
                dict(pos=P + 2), dict(slots=P + 3), dict(refused=P + 2)):
        assert grow(**bad) == INVAL, bad
    assert trim(keep=None) == INVAL and trim(keep=P + 2) == INVAL
    assert _lib.lib.fdm_kv_grow(None, P, 1, P, P, P, None, None) == INVAL and _lib.lib.fdm_kv_trim(None, P, None) == INVAL


NORM = dict(x=P, xt=F32, xs=256, add=2 * P, at=F32, as_=256, sum=3 * P, ss=256, w=P, eps=1e-6, y=4 * P, yt=BF16, ys=256, scale=None, cs=0, T=3, d=256, stream=None)


def norm(**kw):
    return _lib.lib.fdm_add_rms_norm(*{**NORM, **kw}.values())


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(y=None), dict(xt=12), dict(at=12), dict(yt=12), dict(T=-1), dict(d=0), dict(d=32769), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
    dict(x=P + 2), dict(add=P + 1), dict(sum=P + 2), dict(y=P + 1), dict(w=P + 2), dict(scale=P), dict(yt=E4M3), dict(yt=E4M3, scale=P, cs=1), dict(ys=255),
    dict(ss=255), dict(ys=0), dict(sum=P, xs=256, ss=512), dict(sum=4 * P), dict(sum=2 * P, at=BF16), dict(sum=2 * P, as_=512), dict(y=P), dict(y=P, yt=F32, ys=512),
    dict(y=2 * P), dict(y=2 * P, yt=F32, as_=300), dict(xs=1 << 61), dict(as_=-(1 << 62)), dict(cs=1 << 62)])
def test_norm_refusals(bad):
    assert norm(**bad) == INVAL


PROJ = dict(type=BF16, T=3, in_dim=256, out_dim=64, x=P, x_stride=256, x_scale=None, x_scale_stride=0, w=P, w_stride=256, w_scale=None, y=2 * P,
            y_stride=64, y_type=BF16, n_adapters=0, rank=0, B=0, a=None, b=None, times=None, q_start=None, adapter=None)
WITH = dict(n_adapters=2, rank=16, B=2, a=P, b=P, times=P, q_start=P, adapter=P)
FP8 = dict(type=E4M3, x_scale=P, x_scale_stride=2, w_scale=P)


def project(ws=P, size=1 << 40, **kw):
    return _lib.lib.fdm_project(ctypes.byref(_lib.Projection(*{**PROJ, **kw}.values())), ws, size, None)


@pytest.mark.parametrize("bad", [
    dict(type=F32), dict(type=12), dict(y_type=12), dict(y_type=E4M3), dict(T=-1), dict(T=(1 << 20) + 1), dict(in_dim=0), dict(in_dim=252), dict(in_dim=1 << 19),
    dict(out_dim=0), dict(out_dim=1 << 19), dict(x=None), dict(w=None), dict(y=None), dict(ws=None), dict(ws=P + 128), dict(x=P + 8), dict(w=P + 8), dict(y=P + 1),
    dict(x_stride=252), dict(w_stride=4), dict(x_stride=1 << 23), dict(w_stride=-(1 << 23)), dict(y_stride=63), dict(y_stride=0), dict(y_stride=1 << 23),
    dict(x_scale=P), dict(w_scale=P), dict(FP8, x_scale=None), dict(FP8, w_scale=None), dict(FP8, in_dim=264), dict(FP8, x_stride=264), dict(FP8, x_scale_stride=1 << 23),
    dict(WITH, n_adapters=-1), dict(WITH, n_adapters=1025), dict(WITH, rank=0), dict(WITH, rank=12), dict(WITH, rank=136), dict(WITH, rank=-8), dict(WITH, B=0),
    dict(WITH, B=4097), dict(WITH, a=None), dict(WITH, b=None), dict(WITH, q_start=None), dict(WITH, adapter=None), dict(WITH, a=P + 8), dict(WITH, b=P + 2),
    dict(WITH, times=P + 2), dict(WITH, q_start=P + 1), dict(WITH, adapter=P + 2)])
def test_project_refusals(bad):
    assert project(**bad) == INVAL
    assert _lib.lib.fdm_project(None, P, 1 << 40, None) == INVAL


def test_good_arguments_get_as_far_as_the_device():
    if _lib.lib.fdm_available():
        pytest.skip("library already initialised in this process")
    assert grow() == STATE and grow(refused=P, N=0, pos=None, slots=None) == STATE and trim() == STATE
    assert norm() == STATE and norm(T=0, x=None) == STATE and norm(sum=P) == STATE and norm(add=None, sum=None, w=None) == STATE
    assert norm(y=P, yt=F32) == STATE and norm(y=2 * P, yt=F32) == STATE and norm(yt=E4M3, scale=P, cs=2) == STATE and norm(sum=2 * P) == STATE
    assert norm(T=1, xs=3, as_=1, ss=0, ys=0, sum=P) == STATE and norm(xs=0, as_=0) == STATE
    assert project() == STATE and project(T=0, x=None) == STATE and project(**WITH) == STATE and project(**FP8) == STATE
    assert project(T=1, x_stride=1, y_stride=3) == STATE and project(out_dim=1, w_stride=5, y_stride=1) == STATE and project(x_stride=0) == STATE
    n = ctypes.byref(ctypes.c_size_t())
    assert _lib.lib.fdm_project_workspace(4, 256, 64, 16, n) == STATE
    for bad in ((-1, 256, 64, 0), (4, 255, 64, 0), (4, 256, 0, 0), (4, 256, 64, 4), (4, 256, 64, 136)):
        assert _lib.lib.fdm_project_workspace(*bad, n) == INVAL
    assert _lib.lib.fdm_project_workspace(4, 256, 64, 16, None) == INVAL


LEAST = -(1 << 63)


def test_strides_and_rows_past_every_bound():
    for k in ("xs", "as_", "ss", "ys", "cs"):
        assert norm(**{k: LEAST}) == INVAL and norm(**{k: (1 << 63) - 1}) == INVAL, k
    for k in ("x_stride", "w_stride", "y_stride"):
        assert project(**{k: LEAST}) == INVAL and project(**{k: (1 << 63) - 16}) == INVAL, k
    assert project(**{**FP8, "x_scale_stride": LEAST}) == INVAL
    assert norm(T=(1 << 21) + 1) == INVAL
