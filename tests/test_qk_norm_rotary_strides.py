"""The norm and rotation of q and k through strides that do not fit 32 bits once a few heads are passed."""
import os
import re

import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipkittens_b200", "csrc")


def test_products_with_a_stride_are_formed_in_64_bits():
    """A head's stride may be 2^30 units of 8 values, and a warp steps over up to 8 heads at a time."""
    with open(os.path.join(CSRC, "qk_norm_rotary_sm100.cuh")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    products = re.findall(r"[^;{}]*\*\s*s\.stride_[nh]\b[^;{}]*", code)
    assert products
    for text in products:
        for factor in re.findall(r"([\w)(>.<: ]*?)\s*\*\s*s\.stride_[nh]\b", text):
            assert re.search(r"static_cast<long long>\([\w.]+\)$", factor.strip()), text


@pytest.mark.gpu
@pytest.mark.parametrize("d,heads,apart", [(64, 9, 1 << 31), (128, 5, 1 << 32), (64, 17, (1 << 30) + 8)])
def test_heads_far_apart(d, heads, apart):
    """A head-major tensor of B N D values a head: as many heads as a warp steps over, and one more. Bit by bit what packed heads give."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("a tensor of 35 GB needs more memory than is free")
    gen = torch.Generator().manual_seed(d)
    b, n = 2, 21
    q, k, dq, dk = (torch.randn(b, n, h, d, generator=gen).to(torch.bfloat16).cuda() for h in (heads, 2, heads, 2))
    w = (1 + torch.randn(d, generator=gen) / 4).cuda()
    angle = torch.arange(n)[:, None] / 100.0 ** (torch.arange(0, d, 2) / d)
    cos, sin = angle.cos().cuda(), angle.sin().cuda()
    far = torch.empty((heads - 1) * apart + b * n * d, dtype=torch.bfloat16, device="cuda")
    view = far.as_strided((b, n, heads, d), (n * d, d, apart, 1))
    view.copy_(q)
    want = hk.qk_norm_rotary(q, k, w, w, cos, sin), hk.qk_norm_rotary_bwd(q, k, w, w, cos, sin, dq, dk)
    got = hk.qk_norm_rotary(view, k, w, w, cos, sin), hk.qk_norm_rotary_bwd(view, k, w, w, cos, sin, dq, dk)
    as_k = hk.qk_norm_rotary(k, view, w, w, cos, sin)
    assert _native.device_status(0) == 0
    for x, y in zip((*want[0], *want[1], *want[0][::-1]), (*got[0], *got[1], *as_k)):
        assert torch.equal(x, y)
    del far, view
    torch.cuda.empty_cache()
