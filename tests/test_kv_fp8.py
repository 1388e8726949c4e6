"""What the 8-bit paged cache's entries refuse, and the reference that its GPU tests use, without a GPU."""
import math

import pytest
import torch

import hipkittens_b200 as hk
import kv_fp8_reference as ref
from hipkittens_b200 import _native


def test_the_reference_rounds_as_torch_does():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[codes.isfinite()].unique()
    middles = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, middles, middles * (1 + 2.0 ** -20), middles * (1 - 2.0 ** -20), torch.randn(4000).double() * 100])
    x = x[x.abs() <= 448].float()
    assert torch.equal(ref.e4m3(x), x.to(torch.float8_e4m3fn).double())
    assert ref.e4m3(torch.tensor(math.inf)) == 448 and ref.e4m3(torch.tensor(math.nan)).isnan()
    for amax, s in ((448.0, 1.0), (449.0, 2.0), (224.0, 0.5), (0.0, 2.0 ** -120), (math.inf, 2.0 ** 119), (3.0e38, 2.0 ** 119)):
        assert ref.scale_for(amax) == s


def strides(*v):
    return (_native.ctypes.c_longlong * 3)(*v)


def append(**change):
    a = dict(k=4096, v=4096, kp=4096, vp=4096, ks=4096, vs=4096, table=4096, start=4096, cu=None, sin=4096, cos=4096, s=2, t=5, hkv=2,
             d=128, k_st=strides(1280, 256, 128), v_st=strides(1280, 256, 128), rot=128, rows=100, flags=0, page=16, max_pages=8,
             pool=8) | change
    return _native.capi().hk_paged_kv_append_fp8(*a.values(), 0, None)


def read(**change):
    a = dict(kp=4096, vp=4096, ks=4096, vs=4096, table=4096, lens=4096, cu=None, k=4096, v=4096, s=2, rows=5, hkv=2, d=128, tail=0,
             page=16, max_pages=8, pool=8) | change
    return _native.capi().hk_paged_kv_read_fp8(*a.values(), 0, None)


def decode(**change):
    a = dict(q=4096, kp=4096, vp=4096, ks=4096, vs=4096, table=4096, lens=4096, o=4096, lse=4096, s=1, h=8, hkv=2, d=128, page=16,
             max_pages=8, pool=8, window=0, sinks=0, scale=0.0, ws=4096, ws_bytes=1 << 30) | change
    return _native.capi().hk_attn_paged_decode_fp8(*a.values(), 0, None)


CACHE = [(dict(kp=None), "EINVAL"), (dict(vp=None), "EINVAL"), (dict(ks=None), "EINVAL"), (dict(vs=None), "EINVAL"),
         (dict(table=None), "EINVAL"), (dict(kp=4104), "EINVAL"), (dict(vp=4097), "EINVAL"), (dict(ks=4098), "EINVAL"),
         (dict(vs=4097), "EINVAL"), (dict(table=4098), "EINVAL"), (dict(s=0), "EINVAL"), (dict(hkv=0), "EINVAL"), (dict(max_pages=0), "EINVAL"),
         (dict(pool=0), "EINVAL"), (dict(s=65536), "EINVAL"), (dict(max_pages=2 ** 27), "EINVAL"), (dict(pool=2 ** 27), "EINVAL"), (dict(d=96), "EUNSUPPORTED"),
         (dict(d=256), "EUNSUPPORTED"), (dict(page=32), "EUNSUPPORTED")]


@pytest.mark.parametrize("change,code", CACHE + [
    (dict(k=None), "EINVAL"), (dict(v=None), "EINVAL"), (dict(start=None), "EINVAL"), (dict(sin=None), "EINVAL"), (dict(cos=None), "EINVAL"),
    (dict(k=4104), "EINVAL"), (dict(cos=4104), "EINVAL"), (dict(start=4098), "EINVAL"), (dict(cu=4098), "EINVAL"), (dict(t=0), "EINVAL"),
    (dict(flags=2), "EINVAL"), (dict(k_st=None), "EINVAL"), (dict(k_st=strides(1280, 256, 100)), "EINVAL"),
    (dict(v_st=strides(1280, -256, 128)), "EINVAL"), (dict(k_st=strides(0, 256, 128)), "EINVAL"), (dict(rows=0), "EINVAL"),
    (dict(s=65535, t=2 ** 31 - 1), "EINVAL"), (dict(rot=24), "EUNSUPPORTED"), (dict(rot=144), "EUNSUPPORTED"),
])
def test_append_refusals(native_built, change, code):
    assert append(**change) == getattr(_native, "HK_" + code)


@pytest.mark.parametrize("change,code", CACHE + [
    (dict(k=None), "EINVAL"), (dict(v=4104), "EINVAL"), (dict(lens=None), "EINVAL"), (dict(cu=4096), "EINVAL"), (dict(lens=4098), "EINVAL"),
    (dict(rows=0), "EINVAL"), (dict(s=65535, rows=2 ** 31 - 1, hkv=64), "EINVAL"),
])
def test_read_refusals(native_built, change, code):
    assert read(**change) == getattr(_native, "HK_" + code)


@pytest.mark.parametrize("change,code", CACHE + [
    (dict(q=None), "EINVAL"), (dict(lens=None), "EINVAL"), (dict(o=None), "EINVAL"), (dict(lse=None), "EINVAL"), (dict(q=4100), "EINVAL"),
    (dict(o=4104), "EINVAL"), (dict(lens=4097), "EINVAL"), (dict(lse=4098), "EINVAL"), (dict(h=0), "EINVAL"), (dict(hkv=3), "EINVAL"),
    (dict(window=-1), "EINVAL"), (dict(sinks=-1, window=5), "EINVAL"), (dict(sinks=1), "EINVAL"), (dict(h=18), "EUNSUPPORTED"),
    (dict(s=65535, h=65535, hkv=65535), "EINVAL"),
    (dict(ws=None), "EWORKSPACE"), (dict(ws=4112), "EWORKSPACE"), (dict(ws_bytes=100), "EWORKSPACE"),
])
def test_decode_refusals(native_built, change, code):
    assert decode(**change) == getattr(_native, "HK_" + code)


def test_workspace(native_built):
    # two parts of up to 8 heads for each warp of the GPU, in fp32
    assert 0 < hk.paged_decode_fp8_workspace_bytes(4, 8, 64) < hk.paged_decode_fp8_workspace_bytes(4, 8, 128) < 1 << 25
    for bad in (dict(d=96), dict(hkv=0), dict(s=0), dict(s=65536)):
        assert hk.paged_decode_fp8_workspace_bytes(**(dict(s=4, hkv=8, d=128) | bad)) == 0


def test_python_refuses_what_is_not_on_the_gpu(native_built):
    codes, scales = torch.zeros(4, 16, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(4, 2)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: hk.paged_decode_fp8(q, codes, codes, scales, scales, table, lens),
                 lambda: hk.paged_kv_read_fp8(codes, codes, scales, scales, table, 4, ctx_lens=lens),
                 lambda: hk.paged_kv_append_fp8(q, q, codes, codes, scales, scales, table, lens)):
        with pytest.raises(RuntimeError, match="on CUDA device"):
            call()
    with pytest.raises(RuntimeError, match="sinks need a window"):
        hk.paged_decode_fp8(q, codes, codes, scales, scales, table, lens, sinks=4)
