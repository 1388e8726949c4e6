"""The paged cache in 8 bits on the GPU: what appends leave in it, and what reads bring back. Without a rotation everything is exact: codes,
scales and the bf16 of their products with powers of two. With one, x cos - y sin is two products and a sum in fp32, good to 2^-22 of the sum
of their sizes, which can move a value across the border between two codes, or a block's largest across that between two scales."""
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


def status():
    return _native.device_status(0)


class Cache:
    """A pool of random blocks on the GPU, and the same in 64 bits on the CPU."""

    def __init__(self, dev, pool, hkv, d, s, width, seed=0, pow2=True):
        gen = torch.Generator().manual_seed(seed)
        raw = torch.randint(0, 256, (2, pool, 16, hkv, d), generator=gen, dtype=torch.uint8)
        raw[(raw & 127) == 127] = 0
        scales = torch.exp2(torch.randint(-9, 3, (2, pool, hkv), generator=gen).float())
        if not pow2:
            scales = scales * (1 + torch.rand(2, pool, hkv, generator=gen))
        codes = raw.view(torch.float8_e4m3fn)
        self.ref = [codes[0].double(), codes[1].double(), scales[0].double(), scales[1].double()]
        self.table = torch.randperm(pool, generator=gen)[:s * width].reshape(s, width).to(torch.int32)
        self.gpu = [codes[0].to(dev), codes[1].to(dev), scales[0].to(dev), scales[1].to(dev), self.table.to(dev)]

    def values(self):
        return [t.cpu().double() for t in self.gpu[:4]]


def int32(dev, v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def check_exact(cache):
    for got, want in zip(cache.values(), cache.ref):
        assert torch.equal(got.nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("hkv,d,lens,start", [
    (2, 128, [1, 1, 1], [0, 15, 37]),
    (1, 64, [16, 16], [0, 16]),
    (3, 128, [17, 17, 17, 17], [0, 1, 15, 31]),
    (2, 64, [33, 33], [5, 16]),
    (8, 128, [100, 100], [3, 64]),
    (5, 64, [2, 2], [14, 15]),
    (4, 128, [40, 0, 1, 25, 0, 16], [0, 3, 15, 7, 2, 16]),
    (1, 64, [0, 0, 3], [0, 0, 29]),
    (2, 64, [47], [1]),
])
def test_append_is_exact(dev, hkv, d, lens, start, ragged):
    if not ragged and len(set(lens)) > 1:
        pytest.skip("one length for all without cu_seqlens")
    s, width = len(lens), 11
    cache = Cache(dev, s * width + 3, hkv, d, s, width, seed=len(lens) + d)
    gen = torch.Generator().manual_seed(5)
    total = sum(lens)
    x = (torch.randn(total, 2 * hkv + 1, d, generator=gen) * torch.exp2(4 * torch.randn(total, 1, 1, generator=gen))).to(torch.bfloat16)
    g = x.to(dev)
    k, v = g[:, :hkv], g[:, hkv:2 * hkv]  # strided views
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    if ragged:
        hk.paged_kv_append_fp8(k, v, *cache.gpu, int32(dev, start), cu_seqlens=int32(dev, cu))
    else:
        hk.paged_kv_append_fp8(k.unflatten(0, (s, -1)), v.unflatten(0, (s, -1)), *cache.gpu, int32(dev, start))
    for i in range(s):
        if lens[i]:
            rows = x[cu[i]:cu[i + 1]]
            ref.append(cache.ref[0], cache.ref[2], cache.table[i], start[i], rows[:, :hkv])
            ref.append(cache.ref[1], cache.ref[3], cache.table[i], start[i], rows[:, hkv:2 * hkv])
    check_exact(cache)
    assert status() == _native.HK_OK


def test_token_by_token_as_scales_grow(dev):
    """40 tokens, each larger than the last, into pages whose other rows are rounded anew each time the scale grows; the whole again with one
    token in a graph that is replayed."""
    hkv, d, s = 2, 128, 3
    cache = Cache(dev, 12, hkv, d, s, 4, seed=1)
    gen = torch.Generator().manual_seed(2)
    x = (torch.randn(40, s, 1, hkv, d, generator=gen) * 1.3 ** torch.arange(40)[:, None, None, None, None]).to(torch.bfloat16)
    start = int32(dev, [0, 7, 20])
    k, v = (torch.empty(s, 1, hkv, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    hk.paged_kv_append_fp8(k.zero_(), v.zero_(), *cache.gpu, int32(dev, [63, 63, 63]))  # set up outside the capture
    for i in range(s):
        for j in (0, 1):
            ref.append(cache.ref[j], cache.ref[2 + j], cache.table[i], 63, torch.zeros(1, hkv, d))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hk.paged_kv_append_fp8(k, v, *cache.gpu, start)
    for n in range(40):
        k.copy_(x[n])
        v.copy_(-x[39 - n])
        graph.replay()
        start += 1
        for i, first in enumerate((0, 7, 20)):
            ref.append(cache.ref[0], cache.ref[2], cache.table[i], first + n, x[n, i])
            ref.append(cache.ref[1], cache.ref[3], cache.table[i], first + n, -x[39 - n, i])
    check_exact(cache)
    assert status() == _native.HK_OK


def test_scales_of_another_quantiser_are_kept(dev):
    cache = Cache(dev, 4, 2, 64, 1, 4, seed=3, pow2=False)
    x = torch.randn(20, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16) * 0.001
    x[9] *= 100000  # the second block's needs a scale of its own
    before = cache.ref[2][cache.table[0, 0].long()].clone()
    hk.paged_kv_append_fp8(x.to(dev)[None], x.to(dev)[None], *cache.gpu, int32(dev, [7]))
    got = cache.values()
    assert torch.equal(got[2][cache.table[0, 0].long()], before)
    # fp32 divides by such a scale: 2^-24 beside the rounding to e4m3
    for j in (0, 1):
        page = cache.table[0, 0].long()
        want = x[:9].double() / cache.ref[2 + j][page][:, None]
        bound = want.abs() * (2 ** -4 + 2 ** -20) + 2.0 ** -10
        assert ((got[j][page, 7:] - want).abs() <= bound).all()
        assert torch.equal(got[j][page, :7], cache.ref[j][page, :7])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv,d,rot,n,start", [(2, 128, 128, 50, [0, 9]), (3, 64, 64, 7, [11, 30]), (1, 128, 48, 1, [40, 47]), (2, 64, 16, 33, [2, 0]),
                                               (4, 128, 16, 16, [16, 1])])
def test_append_rotates(dev, hkv, d, rot, n, start, dtype):
    cache = Cache(dev, 16, hkv, d, 2, 6, seed=4)
    gen = torch.Generator().manual_seed(7)
    x = torch.randn(2, n, 2 * hkv, d, generator=gen).to(torch.bfloat16)
    angle = torch.arange(90)[:, None] / 100.0 ** (torch.arange(0, rot, 2) / rot)
    cos, sin = angle.cos().to(dtype), angle.sin().to(dtype)
    g = x.to(dev)
    before = [t.clone() for t in cache.ref]
    hk.paged_kv_append_fp8(g[:, :, :hkv], g[:, :, hkv:], *cache.gpu, int32(dev, start), cos=cos.to(dev), sin=sin.to(dev))
    got = cache.values()
    for i in range(2):
        ref.append(cache.ref[1], cache.ref[3], cache.table[i], start[i], x[i, :, hkv:])
        y, size = ref.rotate(x[i, :, :hkv], start[i], cos, sin)
        off = size * 2 ** -22
        for slot in range(start[i] // 16, (start[i] + n - 1) // 16 + 1):
            r0, r1 = max(0, start[i] - slot * 16), min(16, start[i] + n - slot * 16)
            page, rows = int(cache.table[i, slot]), slice(slot * 16 + r0 - start[i], slot * 16 + r1 - start[i])
            for h in range(hkv):
                s, old = float(got[2][page, h]), float(before[2][page, h]) if r0 else 0.0
                amax, most = float(y[rows, h].abs().max()), float(off[rows, h].max())
                assert math.log2(s) % 1 == 0 and amax <= 448 * s + most and (s == old or amax >= 224 * s - most)
                assert s >= old
                want = y[rows, h] / s
                assert ((got[0][page, r0:r1, h] - want).abs() <= (want.abs() + off[rows, h] / s) * 2 ** -4 + off[rows, h] / s + 2.0 ** -10).all()
                keep = [r for r in range(16) if not r0 <= r < r1]
                other = before[0][page, keep, h]
                assert torch.equal(got[0][page, keep, h], ref.e4m3(other * old / s) if r0 else other)
    assert torch.equal(got[1], cache.ref[1]) and torch.equal(got[3], cache.ref[3])
    untouched = [p for p in range(16) if p not in cache.table.flatten().tolist()]
    assert torch.equal(got[0][untouched], before[0][untouched])
    assert status() == _native.HK_OK


@pytest.mark.parametrize("hkv,d,rot", [(13, 128, 128), (8, 64, 32), (5, 128, 0), (1, 64, 64)])
def test_many_pages_and_heads_are_as_one_sequence_at_a_time(dev, hkv, d, rot):
    """More of them than are worked on at once, where a warp takes two heads: bit for bit what a call for each sequence leaves."""
    s, width = 40, 26
    cache, other = (Cache(dev, s * width, hkv, d, s, width, seed=17) for _ in range(2))
    gen = torch.Generator().manual_seed(18)
    lens = [390, 0, 1] + torch.randint(100, 390, (s - 3,), generator=gen).tolist()
    start = torch.randint(0, 20, (s,), generator=gen).tolist()
    cu = [sum(lens[:i]) for i in range(s + 1)]
    x = torch.randn(cu[-1], 2, hkv, d, generator=gen).to(torch.bfloat16).to(dev)
    angle = torch.arange(416)[:, None] / 100.0 ** (torch.arange(0, rot, 2) / max(rot, 1))
    turn = dict(cos=angle.cos().to(dev), sin=angle.sin().to(dev)) if rot else {}
    hk.paged_kv_append_fp8(x[:, 0], x[:, 1], *cache.gpu, int32(dev, start), cu_seqlens=int32(dev, cu), **turn)
    for i in range(s):
        if lens[i]:
            rows = x[None, cu[i]:cu[i + 1]]
            hk.paged_kv_append_fp8(rows[:, :, 0], rows[:, :, 1], *other.gpu[:4], other.gpu[4][i:i + 1], int32(dev, start[i:i + 1]), **turn)
    for got, want in zip(cache.gpu, other.gpu):
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    assert status() == _native.HK_OK


def test_values_at_the_ends(dev):
    """Zeros, infinities, NaN, the smallest and largest bf16 values: each in a block of its own, beside one that it does not touch."""
    hkv, d = 2, 64
    cache = Cache(dev, 10, hkv, d, 1, 10, seed=6)
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(96, hkv, d, generator=gen).to(torch.bfloat16)
    x[0:16] = 0
    x[16, 0, 3] = math.inf
    x[20, 0, 9] = -math.inf
    x[33, 0, 5] = math.nan
    x[48:64, 0] = 2.0 ** -133  # the smallest
    x[48:64, 1] = 2.0 ** -126 * torch.randn(16, d, generator=gen)
    x[64:80, 0] = torch.finfo(torch.bfloat16).max
    x[80:96, 0, ::2] = 448
    x[80:96, 0, 1::2] = -0.0
    ref.append(cache.ref[0], cache.ref[2], cache.table[0], 0, x)
    ref.append(cache.ref[1], cache.ref[3], cache.table[0], 0, x)
    hk.paged_kv_append_fp8(x.to(dev)[None], x.to(dev)[None], *cache.gpu, int32(dev, [0]))
    check_exact(cache)
    assert cache.values()[2][cache.table[0, 2].long(), 0].isnan() and not cache.values()[2][cache.table[0, 2].long(), 1].isnan()
    k, v = hk.paged_kv_read_fp8(*cache.gpu, 96, ctx_lens=int32(dev, [96]))
    want = ref.tokens(cache.ref[0], cache.ref[2], cache.table[0], 96)
    assert torch.equal(k[0].cpu().double().nan_to_num(nan=7e30), want.to(torch.bfloat16).double().nan_to_num(nan=7e30)) and torch.equal(
        k.nan_to_num(nan=1.0), v.nan_to_num(nan=1.0))
    assert k[0, 32:48, 0].isnan().all() and not k[0, 32:48, 1].isnan().any()
    # a NaN stays with its block until that starts anew
    y = torch.ones(1, 1, hkv, d, dtype=torch.bfloat16, device=dev)
    hk.paged_kv_append_fp8(y, y, *cache.gpu, int32(dev, [40]))
    assert cache.values()[2][cache.table[0, 2].long(), 0].isnan()
    hk.paged_kv_append_fp8(y, y, *cache.gpu, int32(dev, [32]))
    assert cache.values()[2][cache.table[0, 2].long(), 0] == 2.0 ** -8
    assert status() == _native.HK_OK


def test_bad_pages_positions_and_lengths(dev):
    hkv, d = 1, 64
    cache = Cache(dev, 6, hkv, d, 2, 3, seed=9)
    cache.table[0, 1], cache.table[1, 0] = 6, -1
    cache.gpu[4].copy_(cache.table)
    x = torch.randn(2, 40, hkv, d, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    g = x.to(dev)
    assert status() == _native.HK_OK
    hk.paged_kv_append_fp8(g, g, *cache.gpu, int32(dev, [10, 10]))  # positions 48 and 49 are behind the table as well
    assert status() == _native.HK_EBADPAGE
    for j in (0, 1):
        ref.append(cache.ref[j], cache.ref[2 + j], cache.table[0], 10, x[0, :6])
        ref.append(cache.ref[j], cache.ref[2 + j], cache.table[0], 32, x[0, 22:38])
        for p in (1, 2):
            ref.append(cache.ref[j], cache.ref[2 + j], cache.table[1], 16 * p, x[1, 16 * p - 10:16 * p + 6])
    check_exact(cache)
    k, v = hk.paged_kv_read_fp8(*cache.gpu, 60, ctx_lens=int32(dev, [60, 20]))
    assert status() in (_native.HK_EBADPAGE, _native.HK_EBADLEN)
    assert not k[0, 16:32].any() and not k[0, 48:].any() and not k[1, :16].any() and not k[1, 20:].any()
    want = (cache.ref[1][cache.table[0, 2].long()] * cache.ref[3][cache.table[0, 2].long()][None, :, None]).to(torch.bfloat16)
    assert torch.equal(v[0, 32:48].cpu(), want)
    # negative and far positions
    hk.paged_kv_append_fp8(g, g, *cache.gpu, int32(dev, [-2 ** 31, 2 ** 31 - 1]))
    assert status() == _native.HK_EBADPAGE
    check_exact(cache)
    # tables that end: tokens behind them are not written
    cos = torch.ones(20, d // 2, device=dev)
    hk.paged_kv_append_fp8(g[:1, :20], g[:1, :20], *cache.gpu[:4], cache.gpu[4][1:].clone(), int32(dev, [16]), cos=cos, sin=torch.zeros_like(cos))
    assert status() == _native.HK_EBADPOS
    for j in (0, 1):
        ref.append(cache.ref[j], cache.ref[2 + j], cache.table[1], 16, x[0, :4])
    check_exact(cache)
    # offsets that fall, or lie outside
    for cu in ([0, 50, 20], [-5, 10, 20], [0, 10, 41]):
        hk.paged_kv_read_fp8(*cache.gpu, 40, cu_seqlens=int32(dev, cu))
        assert status() in (_native.HK_EBADLEN, _native.HK_EBADPAGE)
        hk.paged_kv_append_fp8(g[0], g[0], *cache.gpu, int32(dev, [1000, 1000]), cu_seqlens=int32(dev, cu))
        assert status() in (_native.HK_EBADLEN, _native.HK_EBADPAGE)
    check_exact(cache)


@pytest.mark.parametrize("pow2", [True, False])
@pytest.mark.parametrize("hkv,d,lens", [(2, 128, [100, 1, 0, 33]), (3, 64, [16, 15, 17]), (1, 128, [0, 0]), (8, 64, [48])])
def test_read(dev, hkv, d, lens, pow2):
    s, width = len(lens), 8
    cache = Cache(dev, s * width, hkv, d, s, width, seed=11, pow2=pow2)
    rows = max(max(lens), 1) + 5
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    outs = {}
    outs["padded"] = hk.paged_kv_read_fp8(*cache.gpu, rows, ctx_lens=int32(dev, lens))
    outs["ragged"] = hk.paged_kv_read_fp8(*cache.gpu, cu[-1] + 21, cu_seqlens=int32(dev, cu))
    given = [torch.full((cu[-1] + 21, hkv, d), 5.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    back = hk.paged_kv_read_fp8(*cache.gpu, cu[-1] + 21, cu_seqlens=int32(dev, cu), k_out=given[0], v_out=given[1])
    assert back[0] is given[0] and back[1] is given[1]
    for j in (0, 1):
        for i, n in enumerate(lens):
            want = ref.tokens(cache.ref[j], cache.ref[2 + j], cache.table[i], n) if n else torch.zeros(0, hkv, d).double()
            got = outs["padded"][j][i, :n].cpu()
            if pow2:
                assert torch.equal(got, want.to(torch.bfloat16))
            else:  # fp32 and then bf16
                assert ((got.double() - want).abs() <= want.abs() * (2 ** -8 + 2 ** -23)).all()
            assert not outs["padded"][j][i, n:].any()
            for t in (outs["ragged"][j], given[j]):
                assert torch.equal(t[cu[i]:cu[i + 1]].cpu(), got)
        assert not outs["ragged"][j][cu[-1]:].any() and (given[j][cu[-1]:] == 5).all()
    assert status() == _native.HK_OK


def test_nan_behind_a_length_is_not_read_back(dev):
    cache = Cache(dev, 4, 2, 64, 1, 4, seed=12)
    cache.gpu[2][cache.table[0, 1].long()] = math.nan
    cache.gpu[0].view(torch.uint8)[cache.table[0, 0].long(), 9:] = 127
    k, _ = hk.paged_kv_read_fp8(*cache.gpu, 40, ctx_lens=int32(dev, [9]))
    assert k.isfinite().all() and not k[0, 9:].any()


def test_given_streams_and_refusals(dev):
    cache = Cache(dev, 8, 2, 64, 2, 4, seed=13)
    x = torch.randn(2, 9, 2, 64, device=dev).to(torch.bfloat16)
    start = int32(dev, [0, 5])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    hk.paged_kv_append_fp8(x, x, *cache.gpu, start, stream=side)
    k, v = hk.paged_kv_read_fp8(*cache.gpu, 14, ctx_lens=int32(dev, [9, 14]), stream=side)
    torch.cuda.current_stream().wait_stream(side)
    for j in (0, 1):
        for i in (0, 1):
            ref.append(cache.ref[j], cache.ref[2 + j], cache.table[i], (0, 5)[i], x[i].cpu())
    check_exact(cache)
    assert torch.equal(k[1].cpu().double(), ref.tokens(cache.ref[0], cache.ref[2], cache.table[1], 14).to(torch.bfloat16).double())
    kp, vp, ks, vs, table = cache.gpu
    for bad, text in (((x.float(), x, kp, vp, ks, vs, table, start), "k_new must be torch.bfloat16"),
                      ((x, x[:, :8], kp, vp, ks, vs, table, start), "same shape"),
                      ((x[:1], x[:1], kp, vp, ks, vs, table, start), "must be"),
                      ((x, x, kp.view(torch.uint8), vp, ks, vs, table, start), "float8_e4m3fn"),
                      ((x, x, kp, vp, ks[:4], vs, table, start), "a scale for each page and head"),
                      ((x, x, kp, vp, ks, vs.double(), table, start), "fp32"),
                      ((x, x, kp, vp, ks, vs, table.long(), start), "int32"),
                      ((x, x, kp, vp, ks, vs, table, start.cpu()), "must be a tensor on"),
                      ((x, x, kp, vp, ks, vs, table, start[:1]), "start_pos"),
                      ((x.transpose(1, 3), x.transpose(1, 3), kp, vp, ks, vs, table, start), "must be")):
        with pytest.raises(RuntimeError, match=text):
            hk.paged_kv_append_fp8(*bad)
    with pytest.raises(RuntimeError, match="belong together"):
        hk.paged_kv_append_fp8(x, x, *cache.gpu, start, cos=torch.ones(9, 32, device=dev))
    with pytest.raises(RuntimeError, match="same shape and type"):
        hk.paged_kv_append_fp8(x, x, *cache.gpu, start, cos=torch.ones(9, 32, device=dev), sin=torch.ones(9, 32, device=dev).bfloat16())
    with pytest.raises(RuntimeError, match="either ctx_lens or cu_seqlens"):
        hk.paged_kv_read_fp8(*cache.gpu, 4)
    with pytest.raises(RuntimeError, match="rows must be"):
        hk.paged_kv_read_fp8(*cache.gpu, -1, ctx_lens=start)
    with pytest.raises(RuntimeError, match="k_out"):
        hk.paged_kv_read_fp8(*cache.gpu, 4, ctx_lens=start, k_out=x, v_out=x)
    hk.paged_kv_append_fp8(x[:, :0], x[:, :0], *cache.gpu, start)  # nothing to do
    assert hk.paged_kv_read_fp8(*cache.gpu, 0, ctx_lens=start)[0].shape == (2, 0, 2, 64)
    check_exact(cache)


def test_offsets_behind_32_bits(dev):
    """A pool whose codes, and whose bf16 rows, pass 2^32 bytes."""
    hkv, d = 8, 128
    pool = 2 ** 32 // (16 * hkv * d) + 64
    kp, vp = (torch.zeros(pool, 16, hkv, d, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros(pool, hkv, device=dev) for _ in range(2))
    table = int32(dev, [[pool - 1, 3, pool - 40], [0, pool - 7, 1]])
    x = torch.randn(2, 40, hkv, d, device=dev).to(torch.bfloat16)
    hk.paged_kv_append_fp8(x, -x, kp, vp, ks, vs, table, int32(dev, [0, 0]))
    k, v = hk.paged_kv_read_fp8(kp, vp, ks, vs, table, 40, ctx_lens=int32(dev, [40, 40]))
    assert ((k.double() - x.double()).abs() <= x.double().abs() * (2 ** -4 + 2 ** -8) + x.double().abs().max() * 2.0 ** -17).all()
    assert torch.equal(k, -v)
    used = torch.zeros(pool, dtype=torch.bool, device=dev)
    used[table.flatten().long()] = True
    assert torch.equal(ks.ne(0).all(1), used) and torch.equal(ks.ne(0).any(1), used)
    q = torch.randn(2, 1, 16, d, device=dev).to(torch.bfloat16)
    o, l = hk.paged_decode_fp8(q, kp, vp, ks, vs, table, int32(dev, [40, 33]))
    few = table.flatten().long()
    small = [t[few] for t in (kp.view(torch.uint8), vp.view(torch.uint8), ks, vs)]
    wo, bo, wl, bl = ref.decode(q, small[0].view(torch.float8_e4m3fn), small[1].view(torch.float8_e4m3fn), small[2], small[3],
                                torch.arange(6).reshape(2, 3), torch.tensor([40, 33]))
    assert ((o.cpu().double() - wo).abs() <= bo).all() and ((l.cpu().double() - wl).abs() <= bl).all()
    # rows of the output behind 2^32 bytes
    del kp, vp, k, v
    torch.cuda.empty_cache()
    cache = Cache(dev, 8, hkv, d, 1, 8, seed=1)
    rows = 2 ** 32 // (hkv * d * 2) + 128
    cu = int32(dev, [rows - 100, rows - 10])
    k, _ = hk.paged_kv_read_fp8(*cache.gpu, rows, cu_seqlens=cu)
    assert torch.equal(k[rows - 100:rows - 10].cpu().double(), ref.tokens(cache.ref[0], cache.ref[2], cache.table[0], 90).to(torch.bfloat16).double())
    assert not k[rows - 10:].any()
