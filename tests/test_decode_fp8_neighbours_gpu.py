"""Decode over 8-bit pages: what scales a sequence's neighbours in a batch have does not reach it, and of its own they may be far apart."""
import math

import pytest
import torch

import hipkittens_b200 as hk
import kv_fp8_reference as ref
from hipkittens_b200 import _native
from test_decode_fp8_gpu import check, dev, make  # noqa: F401
from test_decode_fp8_nan_codes_gpu import wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hkv,d", [(2, 128), (1, 64)])
@pytest.mark.parametrize("huge", [2.0 ** 119, 3.0e38, math.inf, math.nan])
def test_scales_of_neighbours(dev, hkv, d, huge):  # noqa: F811
    """60 sequences of a few pages each, so that a warp works on several, with small values; three of them get huge scales."""
    gen = torch.Generator().manual_seed(d)
    lens = torch.randint(1, 70, (60,), generator=gen).tolist()
    a = make(dev, lens, 4 * hkv, hkv, d, pow2=False, seed=9)
    a[4].mul_(2.0 ** -20)
    a = wide(a, 2100)
    want = hk.paged_decode_fp8(*a)
    check(a, want)
    of = (0, 23, 41)
    for i in of:
        a[4][a[5][i, :-(-lens[i] // 16)].long()] = huge
    got = hk.paged_decode_fp8(*a)
    others = [i for i in range(60) if i not in of]
    assert all(torch.equal(x[others], y[others]) for x, y in zip(got, want))
    assert torch.equal(got[1], want[1])


@pytest.mark.parametrize("row", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("huge,small", [(2.0 ** 100, 2.0 ** -38), (1.37 * 2.0 ** 100, 1.1 * 2.0 ** -38), (2.0 ** 20, 2.0 ** -118), (2.0 ** -100, 2.0 ** -119)])
def test_scales_of_one_sequence(dev, d, row, huge, small):  # noqa: F811
    """One page of V with a scale far above the others', and no weight at all."""
    a = make(dev, [300, 40], 4, 2, d, seed=6)
    big = a[5][0, 7].long()
    a[0].abs_()
    a[1][big] = torch.full_like(a[1][big].float(), -300).to(torch.float8_e4m3fn)
    a[3][big] = 2.0  # scores a thousand below the others'
    a[4].fill_(small)
    a[4][big] = huge
    if row:
        a = wide(a, 2100)
    check(a, hk.paged_decode_fp8(*a))
    assert (ref.decode(*a)[0][0].abs() > 0).any()
    assert _native.device_status(0) == _native.HK_OK
