"""What attention over ragged batches refuses, without a GPU."""
import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native
from hipkittens_b200.attention import HipRaggedAttention


def strides(*v):
    return (_native.ctypes.c_longlong * 3)(*v)


def forward(**change):
    a = dict(q=4096, k=4096, v=4096, o=4096, lse=4096, cu_q=4096, cu_k=4096, s=2, tq=300, tk=300, h=8, hkv=2, d=128,
             q_st=strides(1024, 128), k_st=strides(256, 128), v_st=strides(256, 128), causal=1, scale=0.0, fill=1, ws=4096,
             ws_bytes=1 << 30) | change
    return _native.capi().hk_attn_fwd_ragged(*a.values(), 0, None)


def backward(**change):
    a = dict(q=4096, k=4096, v=4096, o=4096, d_o=4096, lse=4096, delta=4096, dq=4096, dk=4096, dv=4096, cu_q=4096, cu_k=4096, s=2, tq=300,
             tk=300, h=8, hkv=2, d=128, q_st=strides(1024, 128), k_st=strides(256, 128), v_st=strides(256, 128),
             dq_st=strides(1024, 128), dk_st=strides(256, 128), dv_st=strides(256, 128), causal=1, scale=0.0, fill=1, ws=4096,
             ws_bytes=1 << 30) | change
    return _native.capi().hk_attn_bwd_ragged(*a.values(), 0, None)


BOTH = [(dict(q=None), "EINVAL"), (dict(k=None), "EINVAL"), (dict(v=None), "EINVAL"), (dict(o=None), "EINVAL"), (dict(lse=None), "EINVAL"),
        (dict(cu_q=None), "EINVAL"), (dict(cu_k=None), "EINVAL"), (dict(q=4104), "EINVAL"), (dict(v=4100), "EINVAL"), (dict(o=4104), "EINVAL"),
        (dict(lse=4097), "EINVAL"), (dict(cu_q=4098), "EINVAL"), (dict(s=0), "EINVAL"), (dict(s=65536), "EINVAL"), (dict(tq=-1), "EINVAL"),
        (dict(tk=2 ** 30 + 1), "EINVAL"), (dict(h=0), "EINVAL"), (dict(hkv=3), "EINVAL"), (dict(tq=2 ** 30, h=1024), "EINVAL"),
        (dict(q_st=None), "EINVAL"), (dict(k_st=strides(256, 100)), "EINVAL"), (dict(v_st=strides(-256, 128)), "EINVAL"),
        (dict(q_st=strides(1 << 39, 128)), "EINVAL"), (dict(d=96), "EUNSUPPORTED"), (dict(d=256), "EUNSUPPORTED"),
        (dict(ws=None), "EWORKSPACE"), (dict(ws=4112), "EWORKSPACE"), (dict(ws_bytes=300), "EWORKSPACE")]


@pytest.mark.parametrize("change,code", BOTH)
def test_forward_refusals(native_built, change, code):
    assert forward(**change) == getattr(_native, "HK_" + code)


@pytest.mark.parametrize("change,code", BOTH + [
    (dict(d_o=None), "EINVAL"), (dict(delta=None), "EINVAL"), (dict(dq=4104), "EINVAL"), (dict(dk=None), "EINVAL"), (dict(delta=4098), "EINVAL"),
    (dict(dv_st=strides(256, 4)), "EINVAL"), (dict(dq_st=None), "EINVAL")])
def test_backward_refusals(native_built, change, code):
    assert backward(**change) == getattr(_native, "HK_" + code)


def test_workspace(native_built):
    lib = _native.capi()
    assert lib.hk_attn_fwd_ragged_workspace_bytes(0, 10) == 0 and lib.hk_attn_bwd_ragged_workspace_bytes(1, -1, 5) == 0
    # a place for each tile that sequences of so many rows can have, 32 bytes each
    assert lib.hk_attn_fwd_ragged_workspace_bytes(7, 1000) >= (1000 // 128 + 7) * 32
    assert lib.hk_attn_bwd_ragged_workspace_bytes(7, 1000, 2000) >= (1000 // 128 + 2000 // 128 + 14) * 32


def test_python_refuses_what_is_not_on_the_gpu(native_built):
    q, kv = torch.zeros(10, 4, 64, dtype=torch.bfloat16), torch.zeros(10, 2, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32)
    for call in (lambda: hk.attn_fwd_ragged(q, *kv.unbind(1), cu), lambda: HipRaggedAttention()(q, kv, cu),
                 lambda: hk.attn_bwd_ragged(q, *kv.unbind(1), q, q, torch.zeros(4, 10), cu)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
