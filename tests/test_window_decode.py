"""What the decode with a window refuses, and how many pages it counts on, without a GPU."""
import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native


def call(native_built, **change):
    a = dict(q=4096, k=4096, v=4096, table=4096, lens=4096, o=4096, lse=4096, s=1, h=8, hkv=2, d=128, page=16, max_pages=8, pool=8,
             window=16, sinks=1, scale=0.0, ws=4096, ws_bytes=1 << 30) | change
    return _native.capi().hk_attn_paged_decode_window(*a.values(), 0, None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), "EINVAL"), (dict(k=None), "EINVAL"), (dict(table=None), "EINVAL"), (dict(lens=None), "EINVAL"), (dict(o=None), "EINVAL"),
    (dict(lse=None), "EINVAL"), (dict(q=4100), "EINVAL"), (dict(v=4104), "EINVAL"), (dict(table=4098), "EINVAL"), (dict(lens=4097), "EINVAL"),
    (dict(lse=4098), "EINVAL"), (dict(s=0), "EINVAL"), (dict(h=0), "EINVAL"), (dict(hkv=3), "EINVAL"), (dict(max_pages=0), "EINVAL"),
    (dict(pool=0), "EINVAL"), (dict(window=0), "EINVAL"), (dict(window=-1), "EINVAL"), (dict(sinks=-1), "EINVAL"),
    (dict(max_pages=2**27), "EINVAL"), (dict(d=96), "EUNSUPPORTED"), (dict(d=256), "EUNSUPPORTED"), (dict(page=32), "EUNSUPPORTED"),
    (dict(h=18), "EUNSUPPORTED"), (dict(s=65536), "EUNSUPPORTED"), (dict(max_pages=10000, window=8192 * 16 + 2), "EUNSUPPORTED"),
    (dict(ws=None), "EWORKSPACE"), (dict(ws=4112), "EWORKSPACE"), (dict(ws_bytes=100), "EWORKSPACE"),
])
def test_refusals(native_built, change, code):
    assert call(native_built, **change) == getattr(_native, "HK_" + code)


def test_workspace_follows_the_window_and_not_the_table(native_built):
    full = hk.paged_decode_workspace_bytes(4, 8, 128, 8192)
    assert hk.paged_decode_workspace_bytes(4, 8, 128, 8192, window=100000000) == full
    small = hk.paged_decode_workspace_bytes(4, 8, 128, 8192, window=500, sinks=4)
    assert 0 < small < full and hk.paged_decode_workspace_bytes(4, 8, 128, 100000, window=500, sinks=4) == small
    assert 0 < hk.paged_decode_workspace_bytes(4, 8, 64, 8192, window=500, sinks=4) < small
    for bad in (dict(d=96), dict(page_size=8)):
        assert hk.paged_decode_workspace_bytes(**(dict(s=4, h=8, d=128, max_pages=8, page_size=16, window=5) | bad)) == 0
    assert hk.paged_decode_workspace_bytes(4, 8, 64, 8192) == 0  # without a window, D = 128 only


def test_python_refuses_windows_that_are_none(native_built):
    t = torch.zeros(1)
    for bad, text in ((dict(window=0), "positive int"), (dict(window=-3), "positive int"), (dict(window=2.0), "positive int"),
                      (dict(window=True), "positive int"), (dict(window=2**31), "positive int"), (dict(sinks=4), "sinks need a window"),
                      (dict(window=4, sinks=-1), "sinks must be"), (dict(window=4, sinks=1.5), "sinks must be")):
        with pytest.raises(RuntimeError, match=text):
            hk.paged_decode(t, t, t, t, t, **bad)
