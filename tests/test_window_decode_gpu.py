"""One new token over the paged cache with a window and sinks, against the definition in 64 bits.

Tolerances. P is rounded to bf16 for the product with V (2^-8 of each term) and O once more; exponentials and the products of
fp32 are good to 2^-18 of a term. L: a score is a sum of D products in fp32, good to D 2^-24 of the sum of their sizes; the logarithm
of a sum of n exponentials to 2^-20 and 2^-22 of itself."""
import math

import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need a B200"
    return torch.device("cuda:0")


def make(dev, lens, h, hkv, d, pool, seed=0, width=None):
    gen = torch.Generator().manual_seed(seed)
    s = len(lens)
    width = width or max(1, -(-max(lens) // 16))
    q = torch.randn(s, 1, h, d, generator=gen).to(torch.bfloat16)
    kp, vp = (torch.randn(pool, 16, hkv, d, generator=gen).to(torch.bfloat16) for _ in range(2))
    table = torch.stack([torch.randperm(pool, generator=gen)[torch.arange(width) % pool] for _ in range(s)]).to(torch.int32)
    return [t.to(dev) for t in (q, kp, vp, table, torch.tensor(lens, dtype=torch.int32))]


def seen(length, window, sinks):
    c = torch.arange(length)
    return c[(length - 1 - c < window) | (c < sinks)]


def reference(q, kp, vp, table, lens, window, sinks):
    """(o, bound, l, bound) in 64 bits on the CPU."""
    q, kp, vp, table, lens = (t.cpu() for t in (q, kp, vp, table, lens))
    s, _, h, d = q.shape
    g = h // kp.shape[2]
    o, bo = torch.zeros(s, 1, h, d).double(), torch.zeros(s, 1, h, d).double()
    l, bl = torch.full((s, h, 1, 1), -math.inf).double(), torch.zeros(s, h, 1, 1).double()
    for i in range(s):
        n = min(int(lens[i]), table.shape[1] * 16)
        if n <= 0:
            continue
        c = seen(n, window, sinks)
        page = table[i].long()[c // 16]
        k, v = kp[page, c % 16].double(), vp[page, c % 16].double()  # [n, hkv, d]
        for j in range(h):
            kj, vj, qj = k[:, j // g], v[:, j // g], q[i, 0, j].double()
            x = kj @ qj / math.sqrt(d)
            p = torch.softmax(x, 0)
            o[i, 0, j] = p @ vj
            bo[i, 0, j] = (p @ vj.abs()) * (2 ** -8 + 2 ** -17) + o[i, 0, j].abs() * 2 ** -8 + 1e-30
            l[i, j] = torch.logsumexp(x, 0)
            bl[i, j] = float((kj.abs() @ qj.abs()).max()) / math.sqrt(d) * d * 2 ** -24 + 2 ** -20 + float(l[i, j].abs()) * 2 ** -22
    return o, bo, l, bl


def check(got, ref):
    (o, l), (ro, bo, rl, bl) = [t.double().cpu() for t in got], ref
    assert bool(((o - ro).abs() <= bo).all()), float(((o - ro).abs() / bo.clamp(min=1e-300)).max())
    empty = rl == -math.inf
    assert torch.equal(l == -math.inf, empty)
    diff = torch.where(empty, 0.0, (l - rl).abs())
    assert bool((diff <= bl).all()), float((diff / bl.clamp(min=1e-300)).max())


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 100, 255, 256, 257, 700]
CASES = [
    # lens, h, hkv, window, sinks, pool
    (LENS, 8, 2, 1, 0, 60),
    (LENS, 4, 4, 1, 1, 60),
    (LENS, 6, 2, 16, 4, 60),
    (LENS, 8, 1, 17, 20, 60),
    (LENS, 5, 1, 100, 33, 60),
    (LENS, 14, 2, 250, 0, 60),
    (LENS, 2, 1, 5000, 7, 60),            # longer than every context
    (LENS, 2, 1, 64, 5000, 60),           # every key is a sink
    ([5000, 4999, 3], 32, 8, 4096, 4, 400),
    ([8192], 32, 8, 1000, 100, 600),
    ([9000, 20000], 4, 4, 16000, 5, 1300),   # more than 32 pages to a warp
    ([700 + 37 * i for i in range(64)], 16, 4, 600, 20, 400),
    ([30 * i for i in range(160)], 8, 2, 130, 2, 400),
    ([40000], 3, 1, 35000, 3, 2600),
]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,h,hkv,window,sinks,pool", CASES)
def test_against_the_definition(dev, lens, h, hkv, window, sinks, pool, d):
    args = make(dev, lens, h, hkv, d, pool, seed=len(lens) + window)
    out = torch.full((len(lens), 1, h, d), float("nan"), dtype=torch.bfloat16, device=dev)
    lse = torch.full((len(lens), h, 1, 1), float("nan"), device=dev)
    got = hk.paged_decode(*args, out=out, lse=lse, window=window, sinks=sinks)
    assert got[0].data_ptr() == out.data_ptr() and _native.device_status(0) == 0
    check(got, reference(*args, window, sinks))
    again = hk.paged_decode(*args, window=window, sinks=sinks)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("g", range(1, 9))
@pytest.mark.parametrize("d", [64, 128])
def test_every_group_size(dev, g, d):
    args = make(dev, [777, 40, 1500], 2 * g, 2, d, 120, seed=g)
    check(hk.paged_decode(*args, window=300, sinks=10), reference(*args, 300, 10))


def test_a_window_over_everything_is_the_call_without_one(dev):
    """A table whose pages all lie in the window is dealt as without one, so the sums are the same to the last bit."""
    for lens in ([2000, 17, 900], [1500] * 40, [8192, 5]):
        args = make(dev, lens, 16, 2, 128, 700, seed=3)
        plain = hk.paged_decode(*args)
        got = hk.paged_decode(*args, window=args[3].shape[1] * 16)
        assert torch.equal(plain[0], got[0]) and torch.equal(plain[1], got[1])


@pytest.mark.parametrize("d", [64, 128])
def test_what_is_not_seen_is_not_read(dev, d):
    """Pages between the sinks and the window have no ids that could be looked up, and every key that is not seen is NaN."""
    lens, window, sinks = [1000, 333, 64, 5], 100, 20
    q, kp, vp, table, cl = make(dev, lens, 8, 2, d, 300, seed=9)
    table = torch.randperm(300, generator=torch.Generator().manual_seed(1))[:4 * table.shape[1]].reshape(4, -1).to(torch.int32).to(dev)
    ref = reference(q, kp, vp, table, cl, window, sinks)
    for i, n in enumerate(lens):
        keep = torch.zeros(table.shape[1] * 16, dtype=torch.bool)
        keep[seen(n, window, sinks)] = True
        for page in range(table.shape[1]):
            rows = ~keep[page * 16:page * 16 + 16].to(dev)
            kp[table[i, page].long(), rows] = float("nan")
            vp[table[i, page].long(), rows] = float("inf")
        empty = ~keep.reshape(-1, 16).any(1)
        table[i, empty.to(dev)] = 2 ** 31 - 1
    got = hk.paged_decode(q, kp, vp, table, cl, window=window, sinks=sinks)
    assert _native.device_status(0) == 0
    check(got, ref)


def test_a_bad_page_in_the_window_is_reported(dev):
    args = make(dev, [1000, 500], 8, 2, 128, 100)
    args[3][0, 62] = 100
    hk.paged_decode(*args, window=64, sinks=4)
    assert _native.device_status(0) == _native.HK_EBADPAGE
    args[3][0, 62] = 5
    args[3][1, 0] = -1
    hk.paged_decode(*args, window=64, sinks=0)
    assert _native.device_status(0) == 0
    hk.paged_decode(*args, window=64, sinks=1)
    assert _native.device_status(0) == _native.HK_EBADPAGE


def test_a_context_longer_than_the_table_is_clamped_and_reported(dev):
    args = make(dev, [320, 100], 8, 2, 64, 100)
    args[4][0] = 321
    got = hk.paged_decode(*args, window=50, sinks=3)
    assert _native.device_status(0) == _native.HK_EBADLEN
    check(got, reference(*args, 50, 3))
    args[4][0] = -5
    got = hk.paged_decode(*args, window=50, sinks=3)
    assert _native.device_status(0) == 0
    check(got, reference(*args, 50, 3))


def test_a_table_wider_than_the_other_call_takes(dev):
    q, kp, vp, table, cl = make(dev, [150000, 149990, 20], 8, 2, 128, 500, width=9400)
    with pytest.raises(hk.HkError):
        hk.paged_decode(q, kp, vp, table, cl)
    check(hk.paged_decode(q, kp, vp, table, cl, window=1024, sinks=4), reference(q, kp, vp, table, cl, 1024, 4))


def test_large_scores_and_sinks_far_above_the_window(dev):
    """Sinks that take nearly all of the softmax, and scores of hundreds: no exponential overflows, and what is left of the
    others is left in the reference too."""
    for d in (64, 128):
        q, kp, vp, table, cl = make(dev, [2000], 4, 1, d, 200, seed=4)
        kp[table[0, 0].long(), 0] = 8 * q[0, 0, 0] / q[0, 0, 0].float().norm() * math.sqrt(d)
        check(hk.paged_decode(q, kp, vp, table, cl, window=500, sinks=2), reference(q, kp, vp, table, cl, 500, 2))


def test_streams_a_graph_and_a_workspace_of_the_caller(dev):
    sets = [make(dev, [3000 + 100 * i for i in range(6)], 16, 2, 128, 300, seed=i) for i in range(2)]
    refs = [hk.paged_decode(*a, window=2500, sinks=4) for a in sets]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in sets]
    for a, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(hk.paged_decode(*a, window=2500, sinks=4))
    torch.cuda.synchronize()
    need = hk.paged_decode_workspace_bytes(6, 16, 128, sets[0][3].shape[1], window=2500, sinks=4)
    assert 0 < need <= hk.paged_decode_workspace_bytes(6, 16, 128, sets[0][3].shape[1])
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    got.append(hk.paged_decode(*sets[0], window=2500, sinks=4, workspace=ws, stream=streams[0]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = hk.paged_decode(*sets[1], window=2500, sinks=4, workspace=ws)
    inside[0].zero_()
    graph.replay()
    torch.cuda.synchronize()
    for r, g in ((refs[0], got[0]), (refs[1], got[1]), (refs[0], got[2]), (refs[1], inside)):
        assert torch.equal(r[0], g[0]) and torch.equal(r[1], g[1])
