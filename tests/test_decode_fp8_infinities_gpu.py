"""Decode over 8-bit pages whose values come near the end of fp32, as the block of an infinity does that was appended: 448 x 2^119."""
import pytest
import torch

import hipkittens_b200 as hk
import kv_fp8_reference as ref
from test_decode_fp8_gpu import check, dev, make  # noqa: F401
from test_decode_fp8_nan_codes_gpu import wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("row", [False, True])
@pytest.mark.parametrize("d,lens", [(64, [300, 40]), (128, [300, 40]), (128, [3000, 17])])
def test_an_infinity_of_v_without_weight(dev, d, lens, row):  # noqa: F811
    a = make(dev, lens, 4, 2, d, seed=6)
    big = a[5][0, 7].long()
    a[0].abs_()
    a[1][big] = torch.full_like(a[1][big].float(), -300).to(torch.float8_e4m3fn)
    a[2][big] = torch.full_like(a[1][big].float(), 448).to(torch.float8_e4m3fn)
    a[3][big] = 2.0  # scores a thousand below the others'
    a[4][big] = 2.0 ** 119
    if row:
        a = wide(a, 3100)
    check(a, hk.paged_decode_fp8(*a))


@pytest.mark.parametrize("row", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_an_infinity_of_v_with_weight(dev, d, row):  # noqa: F811
    """O is a mean of values: as long as these are fp32 numbers, it is."""
    a = make(dev, [300, 700, 16], 8, 2, d, seed=7)
    for i, page in ((0, 3), (1, 40), (2, 0)):
        at = a[5][i, page].long()
        a[2][at] = 0.0
        a[2][at, 5, :, 9] = 448.0
        a[4][at] = 2.0 ** 119
    if row:
        a = wide(a, 2100)
    o, _ = hk.paged_decode_fp8(*a)
    wo, bo, _, _ = ref.decode(*a)
    assert (wo[:, :, :, 9].abs() > 1e30).all()
    # the fp32 sums' smallest step, 2^-147 of the largest scale, 50 times: less than 2^-8 of any other column's
    assert ((o.cpu().double() - wo).abs() <= bo).all()


def test_values_of_another_quantiser_s_scales(dev):  # noqa: F811
    """A scale of 2^126, where codes of 1 and 2 are fp32 numbers."""
    a = make(dev, [33, 500], 4, 2, 128, seed=8)
    a[2].copy_(torch.randint(-1, 2, a[2].shape, generator=torch.Generator().manual_seed(1)).float())
    a[4].fill_(2.0 ** 126)
    for b in (a, wide(a, 2100)):
        check(b, hk.paged_decode_fp8(*b))


@pytest.mark.parametrize("row", [False, True])
def test_an_infinity_of_k(dev, row):  # noqa: F811
    """In a column where q is zero: its page's scores are those of a page of zeros, also where q's largest value times the page's scale is
    above fp32."""
    a = make(dev, [100, 50], 4, 2, 128, seed=9)
    at = a[5][0, 2].long()
    a[0][0, 0, :, 7] = 0.0
    a[0][0, 0, :, 1] = 1024.0
    a[1][:, :, :, 1] = 0.0
    a[1][at] = 0.0
    zeros = [t.clone() for t in a]
    a[1][at, 3, :, 7] = 448.0
    a[3][at] = 2.0 ** 119
    if row:
        a = wide(a, 2100)
    check(zeros, hk.paged_decode_fp8(*a))
