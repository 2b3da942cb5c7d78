"""What the Python entry points of the step's operators hand on and what they
refuse, on the CPU: the library's call is replaced by one that keeps its arguments."""
import types

import pytest
import torch

import flash_deepseek_amd as fdm
from flash_deepseek_amd import _lib

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(fdm, "_on_device", lambda *a: None)
    monkeypatch.setattr(fdm, "_call_stream", lambda s: 0)
    monkeypatch.setattr(fdm, "call", lambda name, *a: made.append((name, a)))
    return made


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def books(**kw):
    a = dict(pages=i32(3, 8), kv_len=i32(3), free=i32(40), n_free=i32(1), page_size=16)
    a.update(kw)
    return fdm.KvPages(**a)


@pytest.mark.parametrize("bad", [dict(pages=i32(24)), dict(pages=i32(8, 3).t()), dict(pages=torch.zeros(3, 8, dtype=torch.int64)), dict(kv_len=i32(4)),
                                 dict(free=torch.zeros(40)), dict(n_free=i32(2)), dict(page_size=0), dict(page_size=24)])
def test_pages_that_do_not_fit(calls, bad):
    with pytest.raises(fdm.FdmError):
        books(**bad)


def test_grow_and_trim_hand_on(calls):
    p = books()
    fdm.kv_grow(p, i32(3), i32(4), i32(10), i32(10))
    fdm.kv_trim(p, i32(3))
    (n0, a), (n1, b) = calls
    assert n0 == "fdm_kv_grow" and n1 == "fdm_kv_trim" and a[2] == 10 and a[6] is None
    d = a[0]._obj
    assert (d.B, d.pages_stride, d.n_pages, d.page_size) == (3, 8, 40, 16) and p._turn.data_ptr() == d.turn
    for bad in ((i32(4), i32(4), i32(10), i32(10)), (i32(3), i32(3), i32(10), i32(10)), (i32(3), i32(4), i32(9), i32(10)),
                (i32(3), i32(4), i32(10), torch.zeros(10, dtype=torch.int64)), (i32(3), i32(4), i32(20)[::2], i32(10))):
        with pytest.raises(fdm.FdmError):
            fdm.kv_grow(p, *bad)
    with pytest.raises(fdm.FdmError):
        fdm.kv_grow(p, i32(3), i32(4), i32(10), i32(10), refused=i32(2))
    with pytest.raises(fdm.FdmError):
        fdm.kv_trim(p, i32(2))
    assert len(calls) == 2


def norm(T=3, d=256, **kw):
    a = dict(x=torch.zeros(T, d), add=torch.zeros(T, d, dtype=BF), norm_w=torch.ones(d), out=torch.zeros(T, d, dtype=BF))
    a.update(kw)
    fdm.add_rms_norm(**a)


@pytest.mark.parametrize("bad", [dict(x=torch.zeros(768)), dict(x=torch.zeros(3, 256, dtype=torch.float64)), dict(add=torch.zeros(3, 255)), dict(add=torch.zeros(256, 3).t()),
                                 dict(norm_w=torch.ones(255)), dict(norm_w=torch.ones(256, dtype=BF)), dict(out=torch.zeros(2, 256)), dict(sum=torch.zeros(3, 256, dtype=BF)),
                                 dict(out=torch.zeros(3, 256).to(F8)), dict(scale=torch.zeros(3, 2, dtype=torch.uint8)),
                                 dict(out=torch.zeros(3, 256).to(F8), scale=torch.zeros(3, 1, dtype=torch.uint8)), dict(out=torch.zeros(3, 256).to(F8), scale=torch.zeros(3, 2))])
def test_norm_refusals(calls, bad):
    with pytest.raises(fdm.FdmError):
        norm(**bad)
    assert calls == []


def test_norm_hands_on(calls):
    norm()
    norm(add=None, norm_w=None, out=torch.zeros(3, 256).to(F8), scale=torch.zeros(3, 2, dtype=torch.uint8), sum=torch.zeros(3, 256))
    (_, a), (_, b) = calls
    assert a[1] == _lib.GGML_F32 and a[4] == _lib.GGML_BF16 and a[11] == _lib.GGML_BF16 and a[13] is None and a[15:17] == (3, 256)
    assert b[3] is None and b[8] is None and b[11] == _lib.E4M3 and b[14] == 2 and b[6]


def project(T=3, inner=256, n_out=64, dtype=BF, n=2, rank=16, **kw):
    half = torch.float16 if dtype is torch.float16 else BF
    a = dict(x=torch.zeros(T, inner).to(dtype), w=torch.zeros(n_out, inner).to(dtype), out=torch.zeros(T, n_out, dtype=half), workspace=torch.zeros(1024, dtype=torch.uint8))
    if dtype is F8:
        a.update(x_scale=torch.zeros(T, 2, dtype=torch.uint8), w_scale=torch.zeros(1, 2, dtype=torch.uint8))
    if n:
        a.update(adapters=fdm.Adapters(torch.zeros(n, rank, inner, dtype=half), torch.zeros(n, n_out, rank, dtype=half)), q_start=i32(3), adapter=i32(2))
    a.update(kw)
    fdm.project(**a)


@pytest.mark.parametrize("bad", [
    dict(x=torch.zeros(3, 256)), dict(x=torch.zeros(3, 256, dtype=torch.float16)), dict(x=torch.zeros(256, dtype=BF)), dict(x=torch.zeros(256, 3, dtype=BF).t()),
    dict(w=torch.zeros(64, 255, dtype=BF)), dict(out=torch.zeros(3, 63)), dict(out=torch.zeros(3, 64, dtype=torch.float64)), dict(x_scale=torch.zeros(3, 2, dtype=torch.uint8)),
    dict(q_start=None), dict(adapter=None), dict(q_start=i32(4)), dict(adapter=torch.zeros(2, dtype=torch.int64)), dict(workspace=torch.zeros(2048, dtype=torch.uint8)[::2]),
    dict(workspace=torch.zeros(1, dtype=torch.uint8).expand(1 << 40)), dict(dtype=F8, x_scale=None), dict(dtype=F8, w_scale=None),
    dict(dtype=F8, x_scale=torch.zeros(3, 3, dtype=torch.uint8)), dict(dtype=F8, x_scale=torch.zeros(3, 2)), dict(dtype=F8, w_scale=torch.zeros(2, 2, dtype=torch.uint8)),
    dict(dtype=F8, w_scale=torch.zeros(1, 4, dtype=torch.uint8)[:, ::2])])
def test_project_refusals(calls, bad):
    with pytest.raises(fdm.FdmError):
        project(**bad)
    assert calls == []


def test_adapters_that_do_not_fit(calls):
    z = lambda *s, t=BF: torch.zeros(*s, dtype=t)
    for a, b, times in ((z(2, 16, 256), z(2, 64, 8), None), (z(2, 16, 256), z(3, 64, 16), None), (z(16, 256), z(64, 16), None), (z(2, 16, 256), z(2, 64, 16, t=torch.float16), None),
                        (z(2, 16, 256, t=torch.float32), z(2, 64, 16, t=torch.float32), None), (z(2, 256, 16).transpose(1, 2), z(2, 64, 16), None),
                        (z(2, 16, 256), z(2, 64, 16), torch.ones(3)), (z(2, 16, 256), z(2, 64, 16), z(2)), (z(0, 16, 256), z(0, 64, 16), None)):
        with pytest.raises(fdm.FdmError):
            fdm.Adapters(a, b, times)
    other = fdm.Adapters(z(2, 16, 512), z(2, 64, 16))
    half = fdm.Adapters(z(2, 16, 256, t=torch.float16), z(2, 64, 16, t=torch.float16))
    for ad in (other, half):
        with pytest.raises(fdm.FdmError):
            project(adapters=ad)
    assert calls == []


def test_project_hands_on(calls):
    project()
    project(dtype=F8, n=0, n_out=100, w_scale=torch.zeros(1, 2, dtype=torch.uint8))
    project(dtype=torch.float16)
    a, b, c = (k[1][0]._obj for k in calls)
    assert (a.type, a.T, a.in_dim, a.out_dim, a.n_adapters, a.rank, a.B) == (_lib.GGML_BF16, 3, 256, 64, 2, 16, 2) and not a.x_scale and not a.times and a.q_start
    assert b.type == _lib.E4M3 and b.x_scale_stride == 2 and b.n_adapters == 0 and not b.a and b.y_stride == 100
    assert c.type == _lib.GGML_F16 and c.y_type == _lib.GGML_F16
    assert calls[0][1][2] == 1024


def test_things_of_another_device(monkeypatch):
    """The tensors that a handle keeps are on the device that they were given on."""
    monkeypatch.setattr(fdm, "_device", 0)
    p = types.SimpleNamespace(device=1, desc=_lib.KvPagesDesc(B=2))
    for call in (lambda: fdm.kv_grow(p, i32(2), i32(3), i32(4), i32(4)), lambda: fdm.kv_trim(p, i32(2))):
        with pytest.raises(fdm.FdmError, match="the pages are on device 1"):
            call()
    with pytest.raises(fdm.FdmError, match="a tensor is on"):
        norm()
    monkeypatch.setattr(fdm, "_on_device", lambda *a: None)
    ad = types.SimpleNamespace(device=1, in_dim=256, out_dim=64, dtype=BF)
    with pytest.raises(fdm.FdmError, match="the adapters are on device 1"):
        project(n=0, adapters=ad, q_start=i32(3), adapter=i32(2))
