"""What the norm and rotation of q and k refuses, without a GPU."""
import ctypes

import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native

LL3 = ctypes.c_longlong * 3


def fwd(native_built, **change):
    a = dict(q=4096, k=4096, wq=4096, wk=4096, cos=4096, sin=4096, qo=4096, ko=4096, b=1, n=4, h=2, hkv=1, d=64, rot=64, rows=4,
             qs=LL3(512, 128, 64), ks=LL3(256, 64, 64), pos=None, off=0, eps=1e-6, flags=0) | change
    return _native.capi().hk_qk_norm_rotary(*a.values(), 0, None)


def bwd(native_built, **change):
    a = dict(q=4096, k=4096, wq=4096, wk=4096, cos=4096, sin=4096, dqo=4096, dko=4096, dq=4096, dk=4096, dwq=4096, dwk=4096, b=1, n=4,
             h=2, hkv=1, d=64, rot=64, rows=4, qs=LL3(512, 128, 64), ks=LL3(256, 64, 64), pos=None, off=0, eps=1e-6, flags=0, ws=4096,
             ws_bytes=1 << 30) | change
    return _native.capi().hk_qk_norm_rotary_bwd(*a.values(), 0, None)


SHARED = [
    (dict(q=None), "EINVAL"), (dict(k=None), "EINVAL"), (dict(cos=None), "EINVAL"), (dict(sin=None), "EINVAL"),
    (dict(q=4104), "EINVAL"), (dict(wq=4104), "EINVAL"), (dict(cos=4104), "EINVAL"), (dict(pos=4098), "EINVAL"),
    (dict(b=0), "EINVAL"), (dict(n=0), "EINVAL"), (dict(h=0), "EINVAL"), (dict(hkv=-1), "EINVAL"), (dict(rows=0), "EINVAL"),
    (dict(rows=3), "EINVAL"), (dict(off=1), "EINVAL"), (dict(off=-1), "EINVAL"), (dict(off=2**31 - 1), "EINVAL"),
    (dict(eps=-1.0), "EINVAL"), (dict(eps=float("nan")), "EINVAL"), (dict(flags=8), "EINVAL"),
    (dict(qs=LL3(512, 128, 4)), "EINVAL"), (dict(ks=LL3(0, 64, 64)), "EINVAL"), (dict(qs=LL3(-512, 128, 64)), "EINVAL"),
    (dict(d=72), "EUNSUPPORTED"), (dict(d=272), "EUNSUPPORTED"), (dict(rot=24), "EUNSUPPORTED"), (dict(rot=80), "EUNSUPPORTED"),
    (dict(b=2**15, n=2**15, rows=2**15, h=2), "EINVAL"),
]


@pytest.mark.parametrize("change,code", SHARED + [(dict(qo=None), "EINVAL"), (dict(ko=4100), "EINVAL")])
def test_forward_refuses(native_built, change, code):
    assert fwd(native_built, **change) == getattr(_native, "HK_" + code)


@pytest.mark.parametrize("change,code", SHARED + [
    (dict(dq=None), "EINVAL"), (dict(dk=4100), "EINVAL"), (dict(dqo=None), "EINVAL"), (dict(dwq=4097), "EINVAL"),
    (dict(wq=None), "EINVAL"), (dict(ws=None), "EWORKSPACE"), (dict(ws_bytes=100), "EWORKSPACE"), (dict(ws=4100), "EWORKSPACE"),
])
def test_backward_refuses(native_built, change, code):
    assert bwd(native_built, **change) == getattr(_native, "HK_" + code)


def test_workspace_bytes(native_built):
    bytes_of = _native.capi().hk_qk_norm_rotary_bwd_workspace_bytes
    assert bytes_of(128) > 0 and bytes_of(128) == 2 * bytes_of(64)
    assert bytes_of(0) == bytes_of(8) == bytes_of(272) == bytes_of(-16) == 0


def test_the_python_front_end_says_what_is_wrong(native_built):
    q, k = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    cos = torch.zeros(4, 32)
    with pytest.raises(RuntimeError, match="q must be a 4-D CUDA tensor"):
        hk.qk_norm_rotary(q, k, None, None, cos, cos)
    with pytest.raises(RuntimeError, match="q must be a 4-D CUDA tensor"):
        hk.qk_norm_rotary_bwd(q, k, None, None, cos, cos, q, k)


def test_the_code_has_a_text(native_built):
    assert b"position" in _native.capi().hk_strerror(_native.HK_EBADPOS)
