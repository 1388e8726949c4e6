"""Ragged sequences whose first does not begin at row 0, read back and appended: the rows in front of it are no sequence's."""
import pytest
import torch

import hipkittens_b200 as hk
import kv_fp8_reference as ref
from hipkittens_b200 import _native
from test_kv_fp8_gpu import Cache, dev, int32  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hkv,d", [(3, 64), (2, 128)])
@pytest.mark.parametrize("front", [1, 15, 16, 17, 100, 160])
@pytest.mark.parametrize("lens", [[40, 1], [0, 33, 0], [0]])
def test_rows_in_front(dev, hkv, d, front, lens):  # noqa: F811
    s, behind = len(lens), 19
    cache = Cache(dev, s * 3, hkv, d, s, 3, seed=front)
    cu = [front + sum(lens[:i]) for i in range(s + 1)]
    rows = cu[-1] + behind
    spoiled = torch.full((2, rows, hkv, d), 7.0, dtype=torch.bfloat16, device=dev)  # what the allocator gives back next
    del spoiled
    new = hk.paged_kv_read_fp8(*cache.gpu, rows, cu_seqlens=int32(dev, cu))
    given = [torch.full((rows, hkv, d), 5.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    hk.paged_kv_read_fp8(*cache.gpu, rows, cu_seqlens=int32(dev, cu), k_out=given[0], v_out=given[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    there = hk.paged_kv_read_fp8(*cache.gpu, rows, cu_seqlens=int32(dev, cu), stream=side)
    torch.cuda.current_stream().wait_stream(side)
    for j in (0, 1):
        assert not new[j][:front].any() and not new[j][cu[-1]:].any() and torch.equal(there[j], new[j])
        assert (given[j][:front] == 5).all() and (given[j][cu[-1]:] == 5).all()
        for i, n in enumerate(lens):
            if n:
                want = ref.tokens(cache.ref[j], cache.ref[2 + j], cache.table[i], n).to(torch.bfloat16)
                assert torch.equal(new[j][cu[i]:cu[i + 1]].cpu(), want) and torch.equal(given[j][cu[i]:cu[i + 1]].cpu(), want)
    assert _native.device_status(0) == _native.HK_OK


@pytest.mark.parametrize("front", [1, 16, 37])
def test_an_append_from_a_later_row_on(dev, front):  # noqa: F811
    hkv, d, lens, start = 2, 64, [20, 0, 33], [3, 0, 17]
    cache = Cache(dev, 12, hkv, d, 3, 4, seed=front)
    cu = [front + sum(lens[:i]) for i in range(4)]
    x = torch.randn(cu[-1] + 11, hkv, d, generator=torch.Generator().manual_seed(front)).to(torch.bfloat16)
    x[:front], x[cu[-1]:] = float("nan"), 1e30
    hk.paged_kv_append_fp8(x.to(dev), x.to(dev), *cache.gpu, int32(dev, start), cu_seqlens=int32(dev, cu))
    for i, n in enumerate(lens):
        if n:
            for j in (0, 1):
                ref.append(cache.ref[j], cache.ref[2 + j], cache.table[i], start[i], x[cu[i]:cu[i + 1]])
    for got, want in zip(cache.values(), cache.ref):
        assert torch.equal(got, want)
    assert _native.device_status(0) == _native.HK_OK
