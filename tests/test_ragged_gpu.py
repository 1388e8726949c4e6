"""Attention over ragged batches, forward and backward, against the definition in 64 bits (the bounds are the reference's)."""
import math

import pytest
import torch

import hipkittens_b200 as hk
import ragged_reference as ref
from hipkittens_b200 import _native
from hipkittens_b200.attention import HipRaggedAttention, RaggedAttnFunction

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need a B200"
    return torch.device("cuda:0")


def rand(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()


def offsets(lens, first=0):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def make(lens_q, lens_k, h, hkv, d, seed=0, first=0, behind=0):
    """Views of packed projections, rows in front of the first sequence and behind the last."""
    gen = torch.Generator().manual_seed(seed)
    tq, tk = (first + sum(n) + behind for n in (lens_q, lens_k))
    q, kv = rand(gen, tq, h + 1, d)[:, :h], rand(gen, tk, 2, hkv, d)
    return q, kv, offsets(lens_q, first), offsets(lens_k, first), rand(gen, tq, h, d)


def status():
    return _native.device_status(0)


LENS = [
    ([1], [1]),
    ([128, 256], [128, 256]),
    ([1, 127, 129, 0, 300], [1, 127, 129, 0, 300]),
    ([5, 64, 200, 17], [50, 64, 700, 513]),
    ([300, 20, 129, 7], [10, 0, 128, 1]),
    ([0, 0, 3], [5, 130, 3]),
    ([1] * 40, list(range(1, 41))),
    ([777, 33], [777, 33]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hkv,d", [(4, 2, 128), (3, 1, 64), (8, 1, 64), (2, 2, 128), (5, 1, 128), (4, 4, 64)])
@pytest.mark.parametrize("lens_q,lens_k", LENS)
def test_forward_and_backward(dev, lens_q, lens_k, h, hkv, d, causal):
    q, kv, cu_q, cu_k, d_o = make(lens_q, lens_k, h, hkv, d, seed=h + len(lens_q), first=3, behind=9)
    k, v = kv.unbind(1)
    want = ref.attention(q, k, v, cu_q, cu_k, causal, d_o=d_o)
    o, l = hk.attn_fwd_ragged(q, k, v, cu_q, cu_k, causal=causal)
    ref.close(o, want[0], "O")
    ref.close(l, want[1], "L")
    grads = hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu_q, cu_k, causal=causal)
    for got, pair, what in zip(grads, want[2:], ("dQ", "dK", "dV")):
        ref.close(got, pair, what)
    assert status() == _native.HK_OK


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[2000, 1, 777, 1300, 90], [63] * 200, [4100], [129] * 31, [3000, 2999, 31]])
def test_longer_batches(dev, lens, d):
    h, hkv = 6, 3
    q, kv, cu, _, d_o = make(lens, lens, h, hkv, d, seed=len(lens))
    k, v = kv.unbind(1)
    want = ref.attention(q, k, v, cu, cu, True, d_o=d_o)
    o, l = hk.attn_fwd_ragged(q, k, v, cu)
    ref.close(o, want[0], "O")
    ref.close(l, want[1], "L")
    first = hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu)
    for got, pair, what in zip(first, want[2:], ("dQ", "dK", "dV")):
        ref.close(got, pair, what)
    # the same numbers again, whatever the order of the work
    for _ in range(3):
        again = (*hk.attn_fwd_ragged(q, k, v, cu), *hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu))
        assert all(torch.equal(x, y) for x, y in zip(again, (o, l, *first)))
    assert status() == _native.HK_OK


@pytest.mark.parametrize("n,most", [(257, 40), (1025, 20), (2100, 9)])
def test_more_sequences_than_a_plan_takes_at_a_time(dev, n, most):
    gen = torch.Generator().manual_seed(n)
    lens_q = torch.randint(0, most, (n,), generator=gen).tolist()
    lens_k = torch.randint(0, most, (n,), generator=gen).tolist()
    lens_q[n // 2], lens_k[n // 2] = 700, 900  # one that is not like the others
    q, kv, cu_q, cu_k, d_o = make(lens_q, lens_k, 2, 1, 64, seed=n, behind=3)
    k, v = kv.unbind(1)
    want = ref.attention(q, k, v, cu_q, cu_k, True, d_o=d_o)
    o, l = hk.attn_fwd_ragged(q, k, v, cu_q, cu_k)
    ref.close(o, want[0], "O")
    ref.close(l, want[1], "L")
    for got, pair, what in zip(hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu_q, cu_k), want[2:], ("dQ", "dK", "dV")):
        ref.close(got, pair, what)
    assert status() == _native.HK_OK


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_dq_of_rows_with_few_keys(dev, d, causal):
    """Where a row has few keys, delta is what P dP adds up to in fp32, and not a product with the rounded O: what is left in dS is its
    own rounding to bf16 (2^-8), the exponential's 2^-13 in it and in delta's terms, and the scores' and dP's sums in fp32."""
    lens_q = [1, 2, 3, 17, 31, 32, 33, 60, 5, 40, 16]
    lens_k = [1, 2, 3, 17, 31, 32, 33, 60, 29, 12, 0] if causal else [1, 2, 3, 4, 24, 23, 8, 9, 16, 5, 0]
    h, hkv = 3, 1
    q, kv, cu_q, cu_k, d_o = make(lens_q, lens_k, h, hkv, d, seed=d, first=2, behind=1)
    k, v = kv.unbind(1)
    o, l = hk.attn_fwd_ragged(q, k, v, cu_q, cu_k, causal=causal)
    dq = hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu_q, cu_k, causal=causal)[0].double()
    c = d ** -0.5
    for rq, rk in ref.sequences(cu_q, cu_k):
        n, m = rq.stop - rq.start, rk.stop - rk.start
        pos = torch.arange(n, device=dev)[:, None] + (m - n)
        see = torch.arange(m, device=dev)[None, :] <= pos if causal else torch.ones(n, m, dtype=torch.bool, device=dev)
        few = ((pos >= 0) & (pos < 32))[:, 0] if causal else torch.ones(n, dtype=torch.bool, device=dev)
        for j in range(h):
            if m == 0 or not few.any():
                continue
            qj, kj, vj, gj = q[rq, j].double()[few], k[rk, 0].double(), v[rk, 0].double(), d_o[rq, j].double()[few]
            p = torch.softmax((qj @ kj.T * c).masked_fill(~see[few], -math.inf), 1)
            dp, sizes = gj @ vj.T, qj.abs() @ kj.abs().T * c
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * c
            fp32 = d * 2 ** -23 * (gj.abs() @ vj.abs().T)
            terms = (p * (dp.abs() * (2 ** -13 + sizes * d * 2 ** -23) + fp32)).sum(1, keepdim=True)
            err = ds.abs() * (2 ** -8 + 2 ** -13 + sizes * d * 2 ** -23) + p * c * (terms + fp32)
            want = ds @ kj
            assert ((dq[rq, j][few] - want).abs() <= err @ kj.abs() + want.abs() * 2 ** -8 + 1e-30).all()
    assert status() == _native.HK_OK


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("fill", [math.nan, math.inf, 3e38])
def test_a_sequence_does_not_see_its_neighbours(dev, d, causal, fill):
    """Every other sequence, and the rows that belong to none, hold NaN, infinities or huge values: what the others compute stays the same to
    the last bit."""
    lens = [70, 200, 128, 5, 300, 129, 1, 77]
    h, hkv = 4, 2
    q, kv, cu, _, d_o = make(lens, lens, h, hkv, d, seed=3, first=11, behind=40)
    q = q.contiguous()
    k, v = kv.unbind(1)
    clean = [*hk.attn_fwd_ragged(q, k, v, cu, causal=causal)]
    clean += hk.attn_bwd_ragged(q, k, v, clean[0], d_o, clean[1], cu, causal=causal)
    keep = torch.zeros(q.shape[0], dtype=torch.bool, device=dev)
    for i, (a, b) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        if i % 2 == 0:
            keep[a:b] = True
    for t in (q, kv, d_o):
        t[~keep] = fill
    out = [*hk.attn_fwd_ragged(q, k, v, cu, causal=causal)]
    o, l = out
    o[~keep], l[:, ~keep] = fill, fill
    out += hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu, causal=causal)
    for i, (got, was) in enumerate(zip(out, clean)):
        rows = (lambda t: t[:, keep]) if i == 1 else (lambda t: t[keep])
        assert torch.equal(rows(got), rows(was)), i
    assert status() == _native.HK_OK


def test_rows_without_a_sequence(dev):
    q, kv, cu_q, cu_k, d_o = make([100, 20], [60, 130], 4, 2, 64, seed=5, first=7, behind=300)
    k, v = kv.unbind(1)
    o, l = hk.attn_fwd_ragged(q, k, v, cu_q, cu_k)
    none = torch.ones(q.shape[0], dtype=torch.bool, device=dev)
    none[7:127] = False
    assert not o[none].any() and (l[:, none] == -math.inf).all() and o[~none].any(-1).any(-1).sum() > 0
    dq, dk, dv = hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu_q, cu_k)
    no_key = torch.ones(k.shape[0], dtype=torch.bool, device=dev)
    no_key[7:197] = False
    assert not dq[none].any() and not dk[no_key].any() and not dv[no_key].any()
    # given outputs keep what they hold there
    dkv = torch.stack((dk, dv), 1)
    given = [torch.full_like(t, 5.0) for t in (o, l, dq, dkv)]
    back = hk.attn_fwd_ragged(q, k, v, cu_q, cu_k, out=given[0], lse=given[1])
    assert back[0] is given[0] and back[1] is given[1]
    hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu_q, cu_k, dq=given[2], dk=given[3][:, 0], dv=given[3][:, 1])
    for got, want, rows in ((given[0], o, ~none), (given[2], dq, ~none), (given[3], dkv, ~no_key)):
        assert torch.equal(got[rows], want[rows]) and (got[~rows] == 5).all()
    assert torch.equal(given[1][:, ~none], l[:, ~none]) and (given[1][:, none] == 5).all()
    assert status() == _native.HK_OK


@pytest.mark.parametrize("cu", [[0, 50, 20, 100], [-1, 20, 30, 100], [0, 20, 30, 101], [40, 30, 20, 10]])
def test_offsets_that_fall_or_lie_outside(dev, cu):
    gen = torch.Generator().manual_seed(1)
    q, kv = rand(gen, 100, 4, 64), rand(gen, 100, 2, 2, 64)
    k, v = kv.unbind(1)
    good, bad = offsets([20, 30, 50]), torch.tensor(cu, dtype=torch.int32, device=dev)
    assert status() == _native.HK_OK
    for a, b in ((bad, good), (good, bad), (bad, None)):
        o, l = torch.full_like(q, 5.0), torch.full((4, 100), 5.0, device=dev)
        hk.attn_fwd_ragged(q, k, v, a, b, out=o, lse=l)
        assert status() == _native.HK_EBADLEN
        grads = [torch.full_like(t, 5.0) for t in (q, k, v)]
        hk.attn_bwd_ragged(q, k, v, q, q, l, a, b, dq=grads[0], dk=grads[1], dv=grads[2])
        assert status() == _native.HK_EBADLEN
        assert all((t == 5).all() for t in (o, l, *grads))


def test_no_rows_at_all(dev):
    q, kv = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev), torch.randn(30, 2, 2, 64, device=dev).to(torch.bfloat16)
    cu_q, cu_k = torch.zeros(3, dtype=torch.int32, device=dev), offsets([10, 20])
    k, v = kv.unbind(1)
    o, l = hk.attn_fwd_ragged(q, k, v, cu_q, cu_k)
    assert o.shape == (0, 4, 64) and l.shape == (4, 0)
    dq, dk, dv = hk.attn_bwd_ragged(q, k, v, o, o, l, cu_q, cu_k)
    assert dq.shape == q.shape and not dk.any() and not dv.any()
    q = torch.randn(30, 4, 64, device=dev).to(torch.bfloat16)
    o, l = hk.attn_fwd_ragged(q, k[:0], v[:0], cu_k, cu_q)
    assert not o.any() and (l == -math.inf).all()
    dq, dk, dv = hk.attn_bwd_ragged(q, k[:0], v[:0], o, q, l, cu_k, cu_q)
    assert not dq.any() and dk.shape == (0, 2, 64)
    assert status() == _native.HK_OK


class _Nothing:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("d,causal", [(64, True), (128, False)])
def test_the_module(dev, monkeypatch, native, d, causal):
    """Gradients by the formula, and by differences of a loss along a direction."""
    if not native:
        monkeypatch.setattr(_native, "_front_module", _Nothing())
    lens = [60, 150, 1, 33]
    q, kv, cu, _, d_o = make(lens, lens, 4, 2, d, seed=7)
    q, kv = q.contiguous().requires_grad_(), kv.requires_grad_()
    m = HipRaggedAttention(causal=causal)
    o = m(q, kv, cu)
    dq, dkv = torch.autograd.grad(o, (q, kv), d_o)
    want = ref.attention(q.detach(), *kv.detach().unbind(1), cu, cu, causal, d_o=d_o)
    ref.close(o.detach(), want[0], "O")
    ref.close(dq, want[2], "dQ")
    ref.close(dkv[:, 0], want[3], "dK")
    ref.close(dkv[:, 1], want[4], "dV")
    gen = torch.Generator().manual_seed(9)
    step = [torch.randint(0, 2, t.shape, generator=gen).to(dev) * 2 - 1 for t in (q, kv)]
    eps = 2.0 ** -20

    def loss(sign):  # at points that bf16 does not hold: the definition stands in for the forward
        at = [t.detach().double() + sign * eps * s for t, s in zip((q, kv), step)]
        return float((ref.attention(at[0], *at[1].unbind(1), cu, cu, causal)[0][0] * d_o.double()).sum())

    slope = (loss(1) - loss(-1)) / (2 * eps)
    along = [float(sum((g.double() * s).sum() for g, s in zip(grads, step)))
             for grads in ((dq, dkv), (want[2][0], torch.stack((want[3][0], want[4][0]), 1)))]
    # a score moves by `rate` per unit of the step; the third derivative of a mean over softmax weights is 13 rate^3 of its values' size
    # at most (and of 3 more for the values' own movement), of which a central difference keeps eps^2 / 6. 2^-52 per value summed.
    q_sum, k_sum = (float(t.detach().double().abs().sum(-1).max()) for t in (q, kv))
    rate, size = (q_sum + k_sum + 1) / math.sqrt(d), float(d_o.double().abs().sum()) * (float(kv.detach().abs().max()) + 1)
    off = eps ** 2 / 6 * 16 * max(rate, 1) ** 3 * size + size * 2 ** -52 / eps
    assert abs(along[1] - slope) <= off
    assert abs(along[0] - slope) <= off + float(sum(b.sum() for _, b in want[2:]))
    with torch.no_grad():
        assert torch.equal(m(q, kv, cu, cu), o.detach())
    assert torch.equal(m(q.detach(), kv.detach(), cu, causal=not causal), hk.attn_fwd_ragged(q, *kv.unbind(1), cu, causal=not causal)[0])
    g = torch.autograd.grad(m(q, kv, cu).float().square().sum(), (q, kv), create_graph=True)
    for x in g:
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (m(q, kv, cu).float().sum() + x.float().square().sum()).backward()
    only_kv = torch.autograd.grad(m(q.detach(), kv, cu), kv, d_o)[0]
    assert torch.equal(only_kv, dkv)


@pytest.mark.parametrize("native", [True, False])
def test_a_captured_step(dev, monkeypatch, native):
    """Forward and backward in a graph, replayed with other lengths; and a capture beside a graph of the same leaves from before, on the
    default stream, which is refused."""
    if not native:
        class Front:
            def __getattr__(self, name):
                return real.captured_backward if name == "captured_backward" else lambda *args: None

        real = _native._front()
        monkeypatch.setattr(_native, "_front_module", Front())
    gen = torch.Generator().manual_seed(2)
    q, kv, d_o = rand(gen, 300, 4, 64).requires_grad_(), rand(gen, 300, 2, 2, 64).requires_grad_(), rand(gen, 300, 4, 64)
    cu = offsets([100, 150, 50])
    m = HipRaggedAttention(causal=True)
    m(q.detach(), kv.detach(), cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = m(q, kv, cu)
        got = torch.autograd.grad(o, (q, kv), d_o)
    for lens in ([100, 150, 50], [300, 0, 0], [1, 2, 297], [20, 30, 40]):
        cu.copy_(offsets(lens))
        graph.replay()
        with torch.no_grad():
            want = ref.attention(q, *kv.unbind(1), cu, cu, True, d_o=d_o)
        ref.close(o.detach(), want[0], "O")
        for x, pair in zip((got[0], got[1][:, 0], got[1][:, 1]), want[2:]):
            ref.close(x, pair, lens)
    del o, got, graph
    a, b = q.detach().clone().requires_grad_(), kv.detach().clone().requires_grad_()
    held = m(a, b, cu)
    torch.autograd.grad(held, (a, b), d_o, retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured backward"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(m(a, b, cu), (a, b), d_o)
    del held
    assert status() == _native.HK_OK


def test_streams_and_views(dev):
    """A packed projection of q, k and v with a gradient written into it, on a stream of its own; head strides that are not D."""
    gen = torch.Generator().manual_seed(4)
    lens = [90, 200]
    qkv, d_o, cu = rand(gen, 290, 8, 64), rand(gen, 290, 4, 64), offsets(lens)
    q, k, v = qkv.split((4, 2, 2), 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o, l = hk.attn_fwd_ragged(q, k, v, cu, stream=side)
    d_qkv = torch.full_like(qkv, 7.0)
    side.wait_stream(torch.cuda.current_stream())
    hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu, dq=d_qkv[:, :4], dk=d_qkv[:, 4:6], dv=d_qkv[:, 6:], stream=side)
    new = hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    want = ref.attention(q, k, v, cu, cu, True, d_o=d_o)
    for got, pair in zip((o, l, *d_qkv.split((4, 2, 2), 1)), want):
        ref.close(got, pair, "packed")
    assert torch.equal(torch.cat(new, 1), d_qkv)
    wide = rand(gen, 290, 4, 192)[:, :, 64:128]  # heads apart
    o2, l2 = hk.attn_fwd_ragged(wide, k, v, cu)
    o3, l3 = hk.attn_fwd_ragged(wide.contiguous(), k, v, cu)
    assert torch.equal(o2, o3) and torch.equal(l2, l3)
    # dQ in the place of q
    q2 = q.contiguous()
    hk.attn_bwd_ragged(q2, k, v, o, d_o, l, cu, dq=q2, dk=torch.empty_like(k), dv=torch.empty_like(v))
    assert torch.equal(q2, new[0])
    assert status() == _native.HK_OK


@pytest.mark.parametrize("d", [64, 128])
def test_strides_behind_32_bits(dev, d):
    """Rows 2^24 elements apart: the last lies 5 * 10^9 elements behind the first."""
    lens, h, hkv = [130, 1, 20, 149], 4, 2
    q, kv, cu, _, d_o = make(lens, lens, h, hkv, d, seed=9)
    k, v = kv.unbind(1)
    o, l = hk.attn_fwd_ragged(q, k, v, cu)
    want = hk.attn_bwd_ragged(q, k, v, o, d_o, l, cu)
    rows, step = q.shape[0], 1 << 24
    room = torch.empty(rows * step, dtype=torch.bfloat16, device=dev)
    far = [room.as_strided((rows, n, d), (step, d, 1), 4096 * i) for i, n in enumerate((h, hkv, hkv, h, hkv, hkv))]
    for x, y in zip(far, (q, k, v)):
        x.copy_(y)
    got = hk.attn_fwd_ragged(*far[:3], cu)
    assert torch.equal(got[0], o) and torch.equal(got[1], l)
    hk.attn_bwd_ragged(*far[:3], o, d_o, l, cu, dq=far[3], dk=far[4], dv=far[5])
    for x, y in zip(far[3:], want):
        assert torch.equal(x, y)
    assert status() == _native.HK_OK


def test_refusals(dev):
    gen = torch.Generator().manual_seed(6)
    q, kv, cu = rand(gen, 20, 4, 64), rand(gen, 20, 2, 2, 64), offsets([20])
    k, v = kv.unbind(1)
    for bad, text in (((q.half(), k, v, cu), "must be torch.bfloat16"), ((q[None], k, v, cu), "3-D"), ((q, k[:10], v[:10], cu), "q's rows"),
                      ((q, k, v[:, :1], cu), "k/v must be"), ((q, k, v, cu.long()), "int32"), ((q, k, v, cu.cpu()), "must be a tensor on"),
                      ((q, k, v, cu, offsets([10, 10])), "same shape"), ((q, k, v, cu[:1]), "S >= 1"),
                      ((q.transpose(1, 2).contiguous().transpose(1, 2), k, v, cu), "last dimension")):
        with pytest.raises(RuntimeError, match=text):
            hk.attn_fwd_ragged(*bad)
    o, l = hk.attn_fwd_ragged(q, k, v, cu)
    with pytest.raises(RuntimeError, match="belong together"):
        hk.attn_fwd_ragged(q, k, v, cu, out=o)
    with pytest.raises(RuntimeError, match="lse must be"):
        hk.attn_fwd_ragged(q, k, v, cu, out=o, lse=l[:2])
    with pytest.raises(RuntimeError, match="belong together"):
        hk.attn_bwd_ragged(q, k, v, o, q, l, cu, dq=q)
    with pytest.raises(RuntimeError, match="d_o must be"):
        hk.attn_bwd_ragged(q, k, v, o, q[:10], l, cu)
    with pytest.raises(RuntimeError, match="kv must be"):
        HipRaggedAttention()(q, k, cu)
    with pytest.raises(_native.HkError):
        hk.attn_fwd_ragged(q[:, :3], k, v, cu)  # 3 heads on 2
    with pytest.raises(RuntimeError):
        RaggedAttnFunction.apply(q[:, :, :32], kv[..., :32], cu)
    assert status() == _native.HK_OK
