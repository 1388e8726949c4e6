"""Codes that are NaN, 0x7f and 0xff, in an 8-bit cache of another quantiser: one that the query sees makes NaN of what it is part of, as it
does of what is read back, and one that it does not see of nothing. O of a column is a sum over V's values in that column alone, scores and L
take all of K's."""
import pytest
import torch

import hipkittens_b200 as hk
import kv_fp8_reference as ref
from hipkittens_b200 import _native
from test_decode_fp8_gpu import dev, make  # noqa: F401

pytestmark = pytest.mark.gpu


def wide(a, width):
    """The same call with room in the table that nothing uses: with much of it, all pages are one row of work."""
    s, have = a[5].shape
    return a[:5] + [torch.cat([a[5], torch.full((s, width - have), -1, dtype=torch.int32, device=a[5].device)], 1)] + a[6:]


def plant(t, table, seq, token, head, col, code):
    t.view(torch.uint8)[table[seq, token // 16].long(), token % 16, head, col] = code


def check(a, **kw):
    o, l = (t.cpu().double() for t in hk.paged_decode_fp8(*a, **kw))
    wo, bo, wl, bl = ref.decode(*a, **kw)
    assert torch.equal(o.isnan(), wo.isnan()) and torch.equal(l.isnan(), wl.isnan())
    assert ((o - wo).abs() <= bo)[~wo.isnan()].all()
    assert ((l - wl).abs() <= bl)[~wl.isnan()].all()
    assert _native.device_status(0) == _native.HK_OK
    return o, l


@pytest.mark.parametrize("row", [False, True])
@pytest.mark.parametrize("h,hkv,d", [(8, 2, 128), (15, 3, 64), (8, 1, 64), (4, 4, 128)])
def test_codes_of_nan(dev, h, hkv, d, row):  # noqa: F811
    a = make(dev, [40, 700, 33, 16, 1], h, hkv, d, seed=h + d)
    table = a[5]
    if row:
        a = wide(a, 2100)
    clean, _ = check(a)
    assert clean.isfinite().all()
    for t in a[1:3]:  # behind the contexts' ends
        for seq, page, first in ((0, 2, 8), (2, 2, 1), (4, 0, 1)):
            t.view(torch.uint8)[table[seq, page].long(), first:] = 127
    assert torch.equal(check(a)[0], clean)
    for seq, token, head, col, code in ((0, 3, hkv - 1, 5, 127), (0, 39, 0, d - 1, 255), (1, 350, 0, 0, 127), (1, 351, 0, 17, 255), (1, 699, hkv - 1, 30, 127),
                                        (2, 32, 0, 8, 255), (4, 0, 0, d // 2 + 1, 127)):
        plant(a[2], table, seq, token, head, col, code)
    o, _ = check(a)
    assert int(o.isnan().sum()) == 7 * (h // hkv) and o[3].isfinite().all()
    _, v = hk.paged_kv_read_fp8(*a[1:6], 700, ctx_lens=a[6])
    assert torch.equal(v.isnan().any(1).repeat_interleave(h // hkv, 1).cpu(), o[:, 0].isnan())
    plant(a[1], table, 1, 500, 0, 2, 255)
    _, l = check(a)
    assert int(l.isnan().sum()) == h // hkv


def test_a_window_hides_them(dev):  # noqa: F811
    """Seen by one query as a sink and by none between the sinks and the window; of more units than have a CTA each, and of few."""
    for s in (3, 160):
        a = make(dev, [900 - i for i in range(s)], 8, 4, 128, seed=s)
        for i, token, col in ((0, 2, 9), (1, 400, 9), (2, 820, 9)):
            plant(a[2], a[5], i, token, 1, col, 127)
        o, _ = check(a, window=100, sinks=5)
        assert torch.equal(o.isnan().flatten(1).any(1), torch.tensor([True, False, True] + [False] * (s - 3)))


def test_a_page_of_nothing_else(dev):  # noqa: F811
    for d in (64, 128):
        a = make(dev, [50, 50], 8, 1, d, seed=3)
        a[2].view(torch.uint8)[a[5][1, 1].long()] = 255
        o, l = check(a)
        assert o[1].isnan().all() and o[0].isfinite().all() and l.isfinite().all()
