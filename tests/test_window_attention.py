"""What attention with a window refuses, and how its backward deals its shares, without a GPU."""
import ctypes

import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native
from hipkittens_b200.attention import HipCrossAttention, HipSelfAttention

LL3 = ctypes.c_longlong * 3
ST = LL3(512, 128, 64)


def fwd(native_built, **change):
    a = dict(q=4096, k=4096, v=4096, o=4096, lse=4096, b=1, n=4, nk=4, h=2, hkv=2, d=64, qs=ST, ks=ST, vs=ST, lens=None, window=2, sinks=0,
             scale=0.0) | change
    return _native.capi().hk_attn_fwd_window(*a.values(), 0, None)


def paged(native_built, **change):
    a = dict(q=4096, k=4096, v=4096, table=4096, lens=4096, o=4096, lse=4096, s=1, t=4, h=2, hkv=2, d=64, page=16, max_pages=4, pool=4,
             window=2, sinks=0, scale=0.0) | change
    return _native.capi().hk_attn_fwd_paged_window(*a.values(), 0, None)


def bwd(native_built, **change):
    a = dict(q=4096, k=4096, v=4096, o=4096, d_o=4096, lse=4096, delta=4096, dq=4096, dk=4096, dv=4096, b=1, n=4, nk=4, h=2, hkv=2, d=64,
             qs=ST, ks=ST, vs=ST, dqs=ST, dks=ST, dvs=ST, lens=None, window=2, sinks=0, scale=0.0, ws=None, ws_bytes=0) | change
    return _native.capi().hk_attn_bwd_window(*a.values(), 0, None)


BAD = [(dict(q=None), "EINVAL"), (dict(k=4100), "EINVAL"), (dict(window=0), "EINVAL"), (dict(window=-4), "EINVAL"), (dict(sinks=-1), "EINVAL"),
       (dict(d=96), "EUNSUPPORTED"), (dict(h=3), "EINVAL"), (dict(lse=4098), "EINVAL"), (dict(lse=None), "EINVAL")]


@pytest.mark.parametrize("change,code", BAD + [(dict(nk=0), "EINVAL"), (dict(qs=LL3(512, 128, 4)), "EINVAL"), (dict(vs=None), "EINVAL")])
def test_forward_refuses(native_built, change, code):
    assert fwd(native_built, **change) == getattr(_native, "HK_" + code)


@pytest.mark.parametrize("change,code", BAD + [(dict(table=None), "EINVAL"), (dict(t=0), "EINVAL"), (dict(page=8), "EUNSUPPORTED")])
def test_paged_forward_refuses(native_built, change, code):
    assert paged(native_built, **change) == getattr(_native, "HK_" + code)


@pytest.mark.parametrize("change,code", BAD + [
    (dict(dq=None), "EINVAL"), (dict(dks=LL3(0, 64, 64)), "EINVAL"), (dict(dvs=None), "EINVAL"), (dict(delta=4097), "EINVAL"),
    (dict(n=4000, nk=4000, sinks=4), "EWORKSPACE"), (dict(n=4000, nk=4000, sinks=4, ws=4096, ws_bytes=100), "EWORKSPACE"),
    (dict(n=4000, nk=4000, sinks=4, ws=4112, ws_bytes=1 << 30), "EWORKSPACE"),
])
def test_backward_refuses(native_built, change, code):
    assert bwd(native_built, **change) == getattr(_native, "HK_" + code)


def test_workspace_of_the_backward(native_built):
    of = _native.capi().hk_attn_bwd_window_workspace_bytes
    share = 2 * 128 * 128 * 4
    assert of(1, 129, 129, 8, 2, 128, 129, 0) == 0                    # nothing hidden
    assert of(16, 8192, 8192, 32, 8, 128, 1024, 0) == 0               # no sinks, blocks for every SM
    n = of(2, 8192, 8192, 32, 8, 128, 1024, 4)
    assert n > 0 and n % (16 * share) == 0 and n // (16 * share) <= 32  # one block of each unit shared
    assert of(2, 8192, 8192, 32, 8, 64, 1024, 4) % (16 * share // 2) == 0
    assert of(1, 384, 384, 8, 2, 128, 128, 2) % (6 * share) == 0 < of(1, 384, 384, 8, 2, 128, 128, 2)  # all six blocks
    assert of(1, 1000, 100, 8, 2, 128, 500, 0) == of(1, 1000, 100, 8, 2, 128, 100, 0)  # a longer window is no longer one
    assert of(1, 2 ** 30, 2 ** 30, 1, 1, 128, 1, 2 ** 30 - 1) >= 0
    for bad in ((0, 8, 8, 2, 2, 64, 4, 0), (1, 8, 8, 3, 2, 64, 4, 0), (1, 8, 8, 2, 2, 96, 4, 0), (1, 8, 8, 2, 2, 64, 0, 0), (1, 8, 8, 2, 2, 64, 4, -1)):
        assert of(*bad) == 0


@pytest.mark.parametrize("make", [HipSelfAttention, HipCrossAttention])
def test_modules_refuse_windows_that_are_none(make):
    for bad, text in ((dict(window=0), "positive int"), (dict(window="8"), "positive int"), (dict(sinks=3), "sinks need a window"),
                      (dict(window=8, sinks=-2), "sinks must be")):
        with pytest.raises(RuntimeError, match=text):
            make(causal=True, **bad)
    assert make(causal=True, window=8, sinks=1).window == 8 and make().window is None


def test_python_refuses(native_built):
    t = torch.zeros(1)
    with pytest.raises(RuntimeError, match="a window needs causal"):
        hk.attn_fwd(t, t, t, window=8)
    with pytest.raises(RuntimeError, match="sinks need a window"):
        hk.attn_fwd(t, t, t, causal=True, sinks=2)
    with pytest.raises(RuntimeError, match="a window needs causal"):
        hk.attn_fwd_paged(t, t, t, t, t, causal=False, window=8)
    with pytest.raises(RuntimeError, match="a window needs causal"):
        _native.attn_bwd_strided(*[t] * 9, causal=False, window=8)
