"""What the Python entry points of the latent operators hand on and what they refuse, on
the CPU: the library's call is replaced by one that keeps its arguments."""
import types

import pytest
import torch

import flash_deepseek_amd as fdm

BF = torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(fdm, "_on_device", lambda *a: None)
    monkeypatch.setattr(fdm, "_call_stream", lambda s: 0)
    monkeypatch.setattr(fdm, "call", lambda name, *a: made.append((name, a)))
    return made


def attend(N=3, H=4, B=2, **kw):
    from flash_deepseek_amd import _lib
    cache = types.SimpleNamespace(device=0, half=BF, desc=_lib.KvCacheDesc())
    i = torch.zeros(B + 1, dtype=torch.int32)
    a = dict(workspace=torch.zeros(1024, dtype=torch.uint8))
    a.update(kw)
    fdm.mla_attend(cache, torch.zeros(N, H, 512, dtype=BF), torch.zeros(N, H, 64, dtype=BF), i, i[:B], torch.zeros(B, 4, dtype=torch.int32), 1.0,
                   torch.zeros(N, H, 512, dtype=BF), **a)


def test_a_mask_without_words_is_refused(calls):
    with pytest.raises(fdm.FdmError, match="a word at least"):
        attend(mask=torch.zeros(3, 0, dtype=torch.int64))
    assert calls == []
    attend(mask=torch.zeros(3, 1, dtype=torch.int64))
    attend()
    batch = [a[1]._obj for _, a in calls]
    assert batch[0].mask_words == 1 and batch[0].mask and batch[1].mask_words == 0 and not batch[1].mask


@pytest.mark.parametrize("workspace", [torch.zeros(1, dtype=torch.uint8).expand(1 << 40), torch.zeros(2048, dtype=torch.uint8)[::2],
                                       torch.zeros(32, 64, dtype=torch.uint8).t()])
def test_a_workspace_that_is_not_contiguous_is_refused(calls, workspace):
    """A size in elements says how many bytes lie behind the address only then."""
    with pytest.raises(fdm.FdmError, match="contiguous"):
        attend(workspace=workspace)
    assert calls == []
    attend(workspace=torch.zeros(64, 32, dtype=torch.float32))
    assert calls[0][1][-2] == 64 * 32 * 4


def test_a_step_without_tokens_may_have_a_mask(calls):
    attend(N=0, mask=torch.zeros(0, 2, dtype=torch.int64))
    batch = calls[0][1][1]._obj
    assert batch.N == 0 and batch.mask_words == 0 and not batch.mask
    # what the library takes that for
    from flash_deepseek_amd import _lib
    from tests.test_latent_args import INVAL, attend as c_attend
    assert c_attend(N=0, ql=None) in (_lib.FDM_E_STATE, _lib.FDM_OK) and c_attend(N=0, ql=None, mask_words=2) == INVAL


def test_strides_of_a_single_token_or_head_are_free():
    """A tensor's stride along an axis of one element may be anything (a column turned into a row has 1)."""
    from flash_deepseek_amd import _lib
    from tests.test_latent_args import INVAL, STATE, attend as c_attend
    if _lib.lib.fdm_available():
        pytest.skip("library already initialised in this process")
    row = torch.zeros(512, 1).t()[:, None]
    assert row.shape == (1, 1, 512) and row.stride()[0] == 1
    assert c_attend(N=1, ql0=1, qr0=3, o0=1) == STATE
    assert c_attend(H=1, ql1=1, qr1=3, o1=1) == STATE
    for bad in (dict(ql0=1), dict(qr0=3), dict(o0=2049), dict(ql1=1), dict(qr1=3), dict(o1=513)):
        assert c_attend(**bad) == INVAL, bad
