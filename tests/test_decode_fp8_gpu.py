"""Decode against the paged cache in 8 bits, against the definition in 64 bits (the bounds are the reference's)."""
import math

import pytest
import torch

import hipkittens_b200 as hk
import kv_fp8_reference as ref
from hipkittens_b200 import _native

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need a B200"
    return torch.device("cuda:0")


def make(dev, lens, h, hkv, d, pow2=True, seed=0, width=None, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    s = len(lens)
    width = width or max(1, -(-max(lens) // 16))
    pool = s * width + 2
    x = torch.randn(2, pool, 16, hkv, d, generator=gen)
    scales = torch.exp2(torch.round(spread * torch.randn(2, pool, hkv, generator=gen)) - 7)
    if not pow2:
        scales = scales * (1 + torch.rand(2, pool, hkv, generator=gen))
    codes = (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    table = torch.randperm(pool, generator=gen)[:s * width].reshape(s, width).to(torch.int32)
    q = torch.randn(s, 1, h, d, generator=gen).to(torch.bfloat16)
    return [t.to(dev) for t in (q, codes[0], codes[1], scales[0], scales[1], table, torch.tensor(lens, dtype=torch.int32))]


def check(a, got, **kw):
    o, l = got
    wo, bo, wl, bl = ref.decode(*a, **kw)
    assert o.shape == a[0].shape and l.shape == wl.shape
    empty = wl == -math.inf
    assert torch.equal(l.cpu().double()[empty], wl[empty]) and not o[:, 0][empty[:, :, 0, 0].to(o.device)].any()
    assert ((o.cpu().double() - wo).abs() <= bo).all(), float(((o.cpu().double() - wo).abs() / bo.clamp(min=1e-30)).max())
    assert ((l.cpu().double() - wl).abs()[~empty] <= bl[~empty]).all()
    assert _native.device_status(0) == _native.HK_OK


@pytest.mark.parametrize("h,hkv,d", [(8, 1, 128), (6, 2, 64), (8, 8, 128), (16, 2, 64), (15, 3, 128), (7, 1, 64), (20, 5, 128), (4, 4, 64)])
@pytest.mark.parametrize("lens", [[1], [0, 16, 17], [15, 130, 1, 700], [2500], [33] * 40])
def test_decode(dev, h, hkv, d, lens):
    a = make(dev, lens, h, hkv, d, pow2=len(lens) % 2 == 0, seed=h + d + len(lens))
    check(a, hk.paged_decode_fp8(*a))


@pytest.mark.parametrize("h,hkv,d,lens,window,sinks", [
    (8, 2, 128, [1, 100, 5, 1000], 64, 4), (6, 1, 64, [500, 3000], 333, 20), (8, 1, 128, [2000], 1, 0), (8, 8, 64, [77, 16, 15], 16, 1),
    (4, 2, 128, [900, 0, 30], 10000, 0), (4, 2, 64, [900, 40], 17, 200), (8, 2, 128, [6000], 4096, 64)])
def test_decode_with_a_window(dev, h, hkv, d, lens, window, sinks):
    a = make(dev, lens, h, hkv, d, pow2=False, seed=window)
    check(a, hk.paged_decode_fp8(*a, window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("s,hkv,width,n", [(1, 1, 8192, 9000), (2, 8, 600, 9600), (64, 8, 40, 640), (3, 1, 8000, 20000), (200, 2, 30, 470),
                                           (1, 8, 2000, 100), (30, 8, 300, 4800)])
def test_every_way_to_spread_a_context(dev, s, hkv, width, n):
    lens = [max(0, n - 37 * i) for i in range(s)]
    a = make(dev, lens, 2 * hkv, hkv, 128, seed=s, width=-(-n // 16))
    if width > a[5].shape[1]:  # room in the table that nothing uses
        a[5] = torch.cat([a[5], torch.full((s, width - a[5].shape[1]), -1, dtype=torch.int32, device=dev)], 1)
    check(a, hk.paged_decode_fp8(*a))


def test_scales_far_apart(dev):
    """Pages of V 2^80 apart, the largest of them with next to no weight, and of K 2^10; no scale at all, one page without weight."""
    a = make(dev, [700, 64, 2000], 8, 2, 128, seed=5)
    a[4].copy_(torch.exp2(torch.randint(-40, 41, a[4].shape, generator=torch.Generator().manual_seed(1)).float()))
    a[3].mul_(torch.exp2(torch.randint(-5, 6, a[3].shape, generator=torch.Generator().manual_seed(2)).float()).to(dev))
    check(a, hk.paged_decode_fp8(*a))
    a = make(dev, [300], 4, 2, 64, seed=6)
    big = a[5][0, 7].long()
    a[1][big] = torch.full_like(a[1][big].float(), -300).to(torch.float8_e4m3fn)  # far below the others for a positive q
    a[0].abs_()
    a[4][big] = 2.0 ** 20
    check(a, hk.paged_decode_fp8(*a))
    a[4].zero_()
    o, _ = hk.paged_decode_fp8(*a)
    assert not o.any()


def test_codes_of_every_value(dev):
    """Subnormal codes among them, alone in a page of K and of V."""
    a = make(dev, [256 + 16], 8, 1, 128, seed=7)
    raw = torch.arange(256, dtype=torch.uint8)
    raw[(raw & 127) == 127] = 0
    gen = torch.Generator().manual_seed(3)
    for t in (a[1], a[2]):
        flat = t.view(torch.uint8)
        for i in range(17):
            flat[a[5][0, i].long()] = raw[torch.randint(0, 256, flat.shape[1:], generator=gen)].to(dev)
        flat[a[5][0, 4].long()] = torch.randint(0, 8, flat.shape[1:], generator=gen, dtype=torch.uint8).to(dev)
    a[3].fill_(2.0 ** -7), a[4].fill_(1.0)
    check(a, hk.paged_decode_fp8(*a))
    for t in (a[1], a[2]):
        t.view(torch.uint8)[:] = torch.randint(0, 8, t.shape, generator=gen, dtype=torch.uint8).to(dev)
    check(a, hk.paged_decode_fp8(*a))


def test_what_is_not_seen_is_not_looked_at(dev):
    """NaN codes and scales behind a context's end and between the sinks and a window, and pages there that do not exist."""
    a = make(dev, [40, 700], 8, 2, 128, seed=8)
    want = hk.paged_decode_fp8(*a)
    windowed = hk.paged_decode_fp8(*a, window=100, sinks=5)
    a[1].view(torch.uint8)[a[5][0, 2].long(), 8:] = 127
    a[2].view(torch.uint8)[a[5][0, 2].long(), 8:] = 255
    a[5][0, 3:] = -1
    got = hk.paged_decode_fp8(*a)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    a[3][a[5][1, 20].long()] = math.nan
    a[4][a[5][1, 21].long()] = math.nan
    a[5][1, 10:20] = 10 ** 9
    got = hk.paged_decode_fp8(*a, window=100, sinks=5)
    assert all(torch.equal(x, y) for x, y in zip(got, windowed))
    assert _native.device_status(0) == _native.HK_OK
    # a block of NaN that is seen is not lost
    a[4][a[5][1, 43].long(), 1] = math.nan
    o, _ = hk.paged_decode_fp8(*a, window=100, sinks=5)
    assert o[1, 0, 4:].isnan().all() and o[1, 0, :4].isfinite().all() and o[0].isfinite().all()


def test_values_of_q_far_apart(dev):
    a = make(dev, [100, 50], 8, 2, 128, seed=9)
    a[0][0] *= 1e-30
    a[0][1, :, 1] *= 2.0 ** 60
    a[0][1, :, 2] = 0
    a[3][a[5][1].long()] *= 2.0 ** -60
    a[0][1, :, 0] *= torch.exp2(-torch.arange(128.0)).to(torch.bfloat16).to(dev)
    check(a, hk.paged_decode_fp8(*a))
    a[0][0, 0, 3, 7] = math.nan
    o, l = hk.paged_decode_fp8(*a)
    assert o[0, 0, 3].isnan().all() and l[0, 3].isnan().all() and o[0, 0, :3].isfinite().all()


def test_bad_pages_and_lengths(dev):
    a = make(dev, [40, 33], 8, 2, 128, seed=10)
    a[6][1] = 1000
    o, _ = hk.paged_decode_fp8(*a)
    assert _native.device_status(0) == _native.HK_EBADLEN and o.isfinite().all()
    a[5][0, 1] = 99
    hk.paged_decode_fp8(*a)
    assert _native.device_status(0) in (_native.HK_EBADPAGE, _native.HK_EBADLEN)
    a[6][:] = -5
    o, l = hk.paged_decode_fp8(*a)
    assert not o.any() and (l == -math.inf).all()
    assert _native.device_status(0) == _native.HK_OK


def test_graphs_streams_and_given_outputs(dev):
    """Two graphs with a workspace each, replayed in turn and from two streams; the same numbers each time."""
    a, b = make(dev, [9000, 300], 8, 1, 128, seed=11, width=8000), make(dev, [500], 8, 2, 64, seed=12)
    want = hk.paged_decode_fp8(*a), hk.paged_decode_fp8(*b)
    graphs, outs = [], []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(hk.paged_decode_fp8(*x))
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(got, w))
    need = hk.paged_decode_fp8_workspace_bytes(2, 1, 128)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    out, lse = torch.empty_like(a[0]), torch.empty(2, 8, 1, 1, device=dev)
    r = hk.paged_decode_fp8(*a, out=out, lse=lse, workspace=ws)
    assert r[0] is out and torch.equal(out, want[0][0]) and torch.equal(lse, want[0][1])
    side.wait_stream(torch.cuda.current_stream())
    o, l = hk.paged_decode_fp8(*a, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want[0][0])
    with pytest.raises(_native.HkError):
        hk.paged_decode_fp8(*a, workspace=ws[:1024])
    with pytest.raises(RuntimeError, match="lse must be"):
        hk.paged_decode_fp8(*a, lse=lse[:1])
    with pytest.raises(RuntimeError, match="q must be torch.bfloat16"):
        hk.paged_decode_fp8(a[0].half(), *a[1:])
    with pytest.raises(_native.HkError):
        hk.paged_decode_fp8(a[0].repeat(1, 1, 2, 1), *a[1:])  # 16 heads to a K/V head
    with pytest.raises(RuntimeError):
        hk.paged_decode(a[0], *a[1:3], *a[5:])  # bf16 pages only


def test_softmax_scale(dev):
    a = make(dev, [123], 4, 2, 64, seed=13)
    check(a, hk.paged_decode_fp8(*a, softmax_scale=0.02), scale=0.02)
