"""Attention forward with a window and sinks, contiguous and paged, against the definition in 64 bits (window_reference says how far
off it may be)."""
import math

import pytest
import torch
import window_reference as ref

import hipkittens_b200 as hk
from hipkittens_b200 import _native

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need a B200"
    return torch.device("cuda:0")


def make(dev, b, n, nk, h, hkv, d, seed=0, packed=False):
    gen = torch.Generator().manual_seed(seed)
    if packed:
        qkv = torch.randn(b, n, h + 2 * hkv, d, generator=gen).to(torch.bfloat16).to(dev)
        return qkv[:, :, :h], qkv[:, :, h:h + hkv], qkv[:, :, h + hkv:]
    return [torch.randn(b, x, y, d, generator=gen).to(torch.bfloat16).to(dev) for x, y in ((n, h), (nk, hkv), (nk, hkv))]


def check(got, want):
    ref.close(got[0], want[0], want[1], "O")
    ref.close(got[1], want[2], want[3], "L")


CASES = [
    # b, n, nk, h, hkv, window, sinks, key lengths
    (1, 1, 1, 1, 1, 1, 0, None),
    (1, 1, 1, 2, 1, 5, 3, None),
    (2, 77, 77, 4, 2, 1, 0, None),
    (1, 128, 128, 2, 1, 2, 1, None),
    (1, 129, 129, 3, 1, 127, 0, None),             # pairs of query tiles
    (2, 300, 300, 4, 2, 128, 4, None),
    (1, 300, 300, 1, 1, 128, 4, None),
    (1, 513, 513, 2, 2, 129, 0, None),
    (1, 1000, 1000, 8, 2, 100, 0, None),
    (1, 1000, 1000, 6, 2, 100, 1, None),
    (1, 1000, 1000, 4, 1, 300, 127, None),
    (1, 1000, 1000, 3, 3, 300, 128, None),
    (2, 1000, 1000, 2, 1, 64, 129, None),
    (1, 1000, 1000, 2, 1, 64, 500, None),           # sinks that most windows run into
    (1, 1000, 1000, 2, 1, 999, 2, None),
    (1, 1000, 1000, 2, 1, 1000, 2, None),           # nothing hidden
    (1, 1000, 1000, 2, 1, 10, 1000, None),
    (1, 64, 1000, 4, 2, 100, 3, None),              # a chunk behind a cache
    (2, 130, 777, 3, 1, 200, 20, None),
    (1, 500, 200, 4, 2, 50, 4, None),               # more queries than keys: rows without keys
    (3, 400, 400, 4, 2, 60, 5, [400, 1, 137]),
    (3, 400, 400, 3, 1, 130, 0, [129, 399, 256]),
    (2, 257, 900, 2, 1, 150, 33, [900, 100]),
    (1, 4000, 4000, 2, 1, 1000, 4, None),
]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,n,nk,h,hkv,window,sinks,lens", CASES)
def test_against_the_definition(dev, b, n, nk, h, hkv, window, sinks, lens, d):
    q, k, v = make(dev, b, n, nk, h, hkv, d, seed=n + window)
    kv_lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device=dev)
    lse = torch.full((b, h, 1, n), float("nan"), device=dev)
    got = hk.attn_fwd(q, k, v, causal=True, out=out, lse=lse, kv_lens=kv_lens, window=window, sinks=sinks)
    assert _native.device_status(0) == 0
    check(got, ref.forward(q, k, v, window, sinks, lens))
    again = hk.attn_fwd(q, k, v, causal=True, kv_lens=kv_lens, window=window, sinks=sinks)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("d", [64, 128])
def test_views_of_a_packed_projection_and_a_scale(dev, d):
    q, k, v = make(dev, 2, 333, 333, 6, 2, d, packed=True)
    got = hk.attn_fwd(q, k, v, causal=True, window=90, sinks=7, softmax_scale=0.3)
    same = hk.attn_fwd(q.contiguous(), k.contiguous(), v.contiguous(), causal=True, window=90, sinks=7, softmax_scale=0.3)
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
    scaled = (q.double() * 0.3 * math.sqrt(d)).requires_grad_(False)
    want = ref.forward(scaled, k, v, 90, 7)
    ref.close(got[0], want[0], want[1], "O")


def test_a_window_over_all_keys_is_causal_attention(dev):
    q, k, v = make(dev, 2, 500, 500, 8, 2, 128)
    plain = hk.attn_fwd(q, k, v, causal=True)
    for window, sinks in ((500, 0), (2 ** 31 - 1, 3), (1, 2 ** 31 - 1)):
        got = hk.attn_fwd(q, k, v, causal=True, window=window, sinks=sinks)
        assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])


@pytest.mark.parametrize("d", [64, 128])
def test_scores_far_apart(dev, d):
    """Sinks whose scores lie hundreds above or below those of the window, masked keys with NaN, infinity and the largest value, and
    rows of values that overflow an exponential against the first tile's maximum."""
    q, k, v = make(dev, 1, 700, 700, 2, 1, d, seed=3)
    base = ref.forward(q, k, v, 100, 2)
    for factor in (30.0, -30.0, 200.0):
        k2 = k.clone()
        k2[:, 0] = (q[0, :, 0].float().mean(0) * 0 + 1).to(torch.bfloat16) * factor / math.sqrt(d)
        check(hk.attn_fwd(q, k2, v, causal=True, window=100, sinks=2), ref.forward(q, k2, v, 100, 2))
        k2 = k.clone()
        k2[:, 400:420] *= factor
        check(hk.attn_fwd(q, k2, v, causal=True, window=100, sinks=2), ref.forward(q, k2, v, 100, 2))
    # a key that only the last rows see, as no number: the rows before it do not notice
    for bad in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).max):
        k2 = k.clone()
        k2[:, 600] = bad
        got = hk.attn_fwd(q, k2, v, causal=True, window=100, sinks=2)
        ref.close(got[0][:, :600], base[0][:, :600], base[1][:, :600], "O")
        ref.close(got[1][..., :600], base[2][..., :600], base[3][..., :600], "L")


def paged(dev, s, t, lens, h, hkv, d, seed=0):
    gen = torch.Generator().manual_seed(seed)
    width = -(-max(lens) // 16)
    q = torch.randn(s, t, h, d, generator=gen).to(torch.bfloat16)
    kp, vp = (torch.randn(s * width + 5, 16, hkv, d, generator=gen).to(torch.bfloat16) for _ in range(2))
    table = torch.randperm(s * width + 5, generator=gen)[:s * width].reshape(s, width).to(torch.int32)
    return [x.to(dev) for x in (q, kp, vp, table, torch.tensor(lens, dtype=torch.int32))]


def gathered(kp, table):
    return kp[table.long()].flatten(1, 2)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t,lens,h,hkv,window,sinks", [
    (1, [500, 3], 4, 2, 100, 2), (64, [1000, 64, 777], 8, 2, 200, 4), (130, [2000, 131], 3, 1, 333, 20), (300, [300, 1500], 2, 2, 17, 0),
    (200, [100, 700], 4, 4, 50, 150),
])
def test_paged_is_the_contiguous_call_on_the_gathered_keys(dev, t, lens, h, hkv, window, sinks, d):
    q, kp, vp, table, cl = paged(dev, len(lens), t, lens, h, hkv, d, seed=t)
    k, v = gathered(kp, table), gathered(vp, table)
    got = hk.attn_fwd_paged(q, kp, vp, table, cl, window=window, sinks=sinks)
    assert _native.device_status(0) == 0
    want = hk.attn_fwd(q, k, v, causal=True, kv_lens=cl, window=window, sinks=sinks)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check(got, ref.forward(q, k, v, window, sinks, lens))


@pytest.mark.parametrize("h,hkv", [(4, 2), (3, 1)])
def test_pages_that_no_row_sees_are_not_looked_up(dev, h, hkv):
    t, window, sinks = 40, 100, 20
    lens = [1000, 515]
    q, kp, vp, table, cl = paged(dev, 2, t, lens, h, hkv, 128, seed=8)
    want = hk.attn_fwd_paged(q, kp, vp, table, cl, window=window, sinks=sinks)
    gone = table.clone()
    for i, n in enumerate(lens):
        first = n - t - window + 1
        gone[i, 2:first // 16] = -7
        gone[i, -(-n // 16):] = 2 ** 31 - 1
    got = hk.attn_fwd_paged(q, kp, vp, gone, cl, window=window, sinks=sinks)
    assert _native.device_status(0) == 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    gone[0, 1] = -1
    hk.attn_fwd_paged(q, kp, vp, gone, cl, window=window, sinks=sinks)
    assert _native.device_status(0) == _native.HK_EBADPAGE


def test_append_then_chunk_then_decode(dev):
    """What a server does with a window layer: append, attend a chunk, then token by token; the same rows as one forward."""
    s, n, h, hkv, d, window, sinks = 2, 350, 8, 2, 128, 90, 4
    q, k, v = make(dev, s, n, n, h, hkv, d, seed=11)
    full = hk.attn_fwd(q, k, v, causal=True, window=window, sinks=sinks)
    want = ref.forward(q, k, v, window, sinks)
    kp, vp = (torch.zeros(60, 16, hkv, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    table = torch.randperm(60, generator=torch.Generator().manual_seed(2))[:44].reshape(2, 22).to(torch.int32).to(dev)
    at = 0
    for t in (200, 130, 1, 1, 1, 1):
        hk.paged_kv_append(k[:, at:at + t].contiguous(), v[:, at:at + t].contiguous(), kp, vp, table,
                           torch.full((s,), at, dtype=torch.int32, device=dev))
        at += t
        lens = torch.full((s,), at, dtype=torch.int32, device=dev)
        qs = q[:, at - t:at].contiguous()
        o, l = (hk.paged_decode if t == 1 else hk.attn_fwd_paged)(qs, kp, vp, table, lens, window=window, sinks=sinks)
        rows = slice(at - t, at)
        ref.close(o, want[0][:, rows], want[1][:, rows], "O")
        ref.close(l.reshape(s, h, 1, t), want[2][..., rows], want[3][..., rows], "L")
    check(full, want)
    assert _native.device_status(0) == 0


def test_streams_and_a_graph(dev):
    sets = [make(dev, 1, 2000, 2000, 8, 2, 128, seed=i) for i in range(2)]
    refs = [hk.attn_fwd(*a, causal=True, window=300, sinks=4) for a in sets]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in sets]
    for a, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(hk.attn_fwd(*a, causal=True, window=300, sinks=4))
    got.append(hk.attn_fwd(*sets[0], causal=True, window=300, sinks=4, stream=streams[1]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = hk.attn_fwd(*sets[1], causal=True, window=300, sinks=4)
    inside[0].zero_()
    graph.replay()
    torch.cuda.synchronize()
    for r, g in ((refs[0], got[0]), (refs[1], got[1]), (refs[0], got[2]), (refs[1], inside)):
        assert torch.equal(r[0], g[0]) and torch.equal(r[1], g[1])
