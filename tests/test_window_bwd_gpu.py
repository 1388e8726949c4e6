"""Gradients of attention with a window and sinks against the definition in 64 bits (window_reference says how far off they may be),
against differences, and through the modules."""
import math

import pytest
import torch
import window_reference as ref

import hipkittens_b200 as hk
from hipkittens_b200 import _native
from hipkittens_b200.attention import HipAttnFunction, HipCrossAttention, HipSelfAttention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need a B200"
    return torch.device("cuda:0")


def make(dev, b, n, nk, h, hkv, d, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(b, x, y, d, generator=gen).to(torch.bfloat16).to(dev) for x, y in ((n, h), (nk, hkv), (nk, hkv), (n, h))]


def grads(q, k, v, d_o, window, sinks, kv_lens=None, **rest):
    o, lse = hk.attn_fwd(q, k, v, causal=True, kv_lens=kv_lens, window=window, sinks=sinks, **rest)
    out = [torch.full(t.shape, float("nan"), dtype=t.dtype, device=t.device) for t in (q, k, v)]
    _native.attn_bwd_strided(q, k, v, o, d_o, lse, *out, causal=True, kv_lens=kv_lens, window=window, sinks=sinks, **rest)
    return out


CASES = [
    # b, n, nk, h, hkv, window, sinks, key lengths
    (1, 1, 1, 1, 1, 1, 0, None),
    (1, 3, 3, 2, 1, 2, 1, None),
    (2, 77, 77, 4, 2, 1, 0, None),
    (1, 129, 129, 3, 1, 127, 0, None),
    (2, 300, 300, 4, 2, 128, 4, None),
    (1, 513, 513, 2, 2, 129, 0, None),
    (1, 1000, 1000, 8, 2, 100, 0, None),
    (1, 1000, 1000, 6, 2, 100, 1, None),
    (1, 1000, 1000, 4, 1, 300, 127, None),
    (1, 1000, 1000, 3, 3, 300, 128, None),
    (2, 1000, 1000, 2, 1, 64, 129, None),
    (1, 1000, 1000, 2, 1, 64, 500, None),
    (1, 1000, 1000, 2, 1, 999, 2, None),
    (1, 1000, 1000, 2, 1, 1000, 2, None),            # nothing hidden
    (1, 64, 1000, 4, 2, 100, 3, None),               # keys that no query sees
    (2, 130, 777, 3, 1, 200, 20, None),
    (1, 500, 200, 4, 2, 50, 4, None),                # rows without keys
    (3, 400, 400, 4, 2, 60, 5, [400, 1, 137]),
    (3, 400, 400, 3, 1, 130, 0, [129, 399, 256]),
    (2, 257, 900, 2, 1, 150, 33, [900, 100]),
    (1, 4000, 4000, 2, 1, 500, 4, None),             # sinks shared by many
    (2, 2100, 2100, 20, 10, 200, 7, None),           # ... with blocks for every SM
    (4, 1500, 1500, 16, 16, 128, 0, None),
    (1, 3000, 3000, 8, 8, 300, 300, [2500]),
]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,n,nk,h,hkv,window,sinks,lens", CASES)
def test_against_the_definition(dev, b, n, nk, h, hkv, window, sinks, lens, d):
    q, k, v, d_o = make(dev, b, n, nk, h, hkv, d, seed=n + window)
    kv_lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    got = grads(q, k, v, d_o, window, sinks, kv_lens)
    assert _native.device_status(0) == 0
    for name, g, (r, bound) in zip(("dQ", "dK", "dV"), got, ref.backward(q, k, v, d_o, window, sinks, lens)):
        ref.close(g, r, bound, name)
    again = grads(q, k, v, d_o, window, sinks, kv_lens)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


def test_gradients_are_those_of_differences(dev):
    """The slope of sum(O dO) along a direction, by central differences of the definition in 64 bits; the kernels' gradients are off by
    their bounds along it."""
    q, k, v, d_o = make(dev, 1, 150, 150, 2, 1, 64, seed=7)
    got = grads(q, k, v, d_o, 40, 3)
    bounds = ref.backward(q, k, v, d_o, 40, 3)
    gen = torch.Generator().manual_seed(1)
    x = [t.double() for t in (q, k, v)]
    for i in range(3):
        step = torch.randn(x[i].shape, generator=gen).double().to(dev)

        def loss(t):
            y = [x[j] + t * step if j == i else x[j] for j in range(3)]
            return float((ref.forward(*y, 40, 3)[0] * d_o.double()).sum())

        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        assert abs(float((got[i].double() * step).sum()) - slope) <= float((bounds[i][1] * step.abs()).sum()) + 1e-5


@pytest.mark.parametrize("h", [4, 3])
def test_modules_and_views_of_a_packed_projection(dev, h):
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(2, 333, 3, h, 64, generator=gen).to(torch.bfloat16).to(dev).requires_grad_()
    d_o = torch.randn(2, 333, h, 64, generator=gen).to(torch.bfloat16).to(dev)
    q, k, v = (t.contiguous() for t in qkv.detach().unbind(2))
    want = grads(q, k, v, d_o, 100, 5)
    o = HipSelfAttention(causal=True, window=100, sinks=5)(qkv)
    assert torch.equal(o, hk.attn_fwd(q, k, v, causal=True, window=100, sinks=5)[0])
    (got,) = torch.autograd.grad(o, qkv, d_o)
    assert all(torch.equal(got[:, :, i], want[i]) for i in range(3))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(HipAttnFunction.apply(*leaves, True, None, None, 100, 5), leaves, d_o)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_cross_module_with_a_padded_batch(dev):
    gen = torch.Generator().manual_seed(4)
    q = torch.randn(2, 200, 4, 128, generator=gen).to(torch.bfloat16).to(dev).requires_grad_()
    kv = torch.randn(2, 300, 2, 2, 128, generator=gen).to(torch.bfloat16).to(dev).requires_grad_()
    d_o = torch.randn(2, 200, 4, 128, generator=gen).to(torch.bfloat16).to(dev)
    lens = [300, 150]
    mask = torch.arange(300, device=dev)[None] < torch.tensor(lens, device=dev)[:, None]
    o = HipCrossAttention(causal=True, window=60, sinks=2)(q, kv, key_padding_mask=mask)
    got = torch.autograd.grad(o, (q, kv), d_o)
    k, v = kv.detach().unbind(2)
    want = ref.forward(q.detach(), k, v, 60, 2, lens)
    ref.close(o.detach(), want[0], want[1], "O")
    (rq, bq), (rk, bk), (rv, bv) = ref.backward(q.detach(), k, v, d_o, 60, 2, lens)
    ref.close(got[0], rq, bq, "dQ")
    ref.close(got[1][:, :, 0], rk, bk, "dK")
    ref.close(got[1][:, :, 1], rv, bv, "dV")
    with pytest.raises(RuntimeError, match="a window needs causal"):
        HipCrossAttention(causal=True, window=60)(q, kv, causal=False)


def test_a_window_over_all_keys_is_the_causal_backward(dev):
    """... but for the rows of few keys, whose delta is summed over their keys (dK is a sum over all rows)."""
    q, k, v, d_o = make(dev, 2, 500, 500, 8, 2, 128)
    o, lse = hk.attn_fwd(q, k, v, causal=True)
    plain = [torch.empty_like(t) for t in (q, k, v)]
    _native.attn_bwd_strided(q, k, v, o, d_o, lse, *plain, causal=True)
    got = grads(q, k, v, d_o, 500, 3)
    assert torch.equal(plain[0][:, 32:], got[0][:, 32:]) and torch.equal(plain[2], got[2])
    for name, g, (r, bound) in zip(("dQ", "dK", "dV"), got, ref.backward(q, k, v, d_o, 500, 3)):
        ref.close(g, r, bound, name)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,nk,lens", [(1, 1, None), (300, 300, None), (200, 333, None), (200, 455, None), (300, 300, [300, 128])])
def test_rows_that_see_one_key_have_no_gradient_of_their_scores(dev, n, nk, lens, d):
    """P is 1 whatever the score: dQ and dK are zero, not what rounding O leaves of dP - delta. (A chunk of 200 rows behind 255 keys
    starts on the last key of a block.)"""
    b = 1 if lens is None else len(lens)
    q, k, v, d_o = make(dev, b, n, nk, 4, 2, d, seed=n)
    dq, dk, dv = grads(q, k, v, d_o, 1, 0, None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev))
    assert not dq.any() and not dk.any()
    (_, _), (_, _), (rv, bv) = ref.backward(q, k, v, d_o, 1, 0, lens)
    ref.close(dv, rv, bv, "dV")
    dq, dk, _ = grads(q, k, v, d_o, 50, 3, None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev))
    if n == nk:
        assert not dq[0, 0].any()  # the first row of a sequence sees its own key alone


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,n,nk,window,sinks,h", [(1, 2000, 2000, 2, 0, 4), (1, 2000, 2000, 1, 1, 3), (1, 2000, 2000, 4, 0, 4), (1, 2000, 2000, 1, 3, 4),
                                                   (300, 2, 2, 9, 0, 4), (200, 4, 4, 9, 1, 4), (300, 3, 4, 2, 0, 3), (1, 2000, 2000, 5, 3, 4), (1, 2000, 2000, 24, 0, 8),
                                                   (1, 2000, 2000, 10, 14, 3), (1, 2000, 2000, 1, 23, 4), (100, 32, 32, 50, 0, 4), (50, 30, 41, 9, 7, 4),
                                                   (40, 45, 31, 50, 0, 6)])
def test_rows_of_few_keys_are_as_exact_as_others(dev, b, n, nk, window, sinks, h, d):
    """dQ and dK are off by two roundings to bf16, theirs and that of dS: each is uniform over a step, 2^-8 / sqrt(3) of the lower end of a
    binade and 0.74 of that over a binade, 1.67e-3, so 2.36e-3 for the two, and a tenth more for sums that are not random. With delta from
    the rounded O it was 3 to 4e-3."""
    q, k, v, d_o = make(dev, b, n, nk, h, 1, d, seed=b + window)
    for g, (r, _) in list(zip(grads(q, k, v, d_o, window, sinks), ref.backward(q, k, v, d_o, window, sinks)))[:2]:
        assert float((g.double() - r).norm() / r.norm()) <= 2.6e-3


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,nk,window", [(700, 700, 500), (700, 700, 699), (700, 700, 700), (300, 1000, 900), (9, 9, 40), (100, 3, 5)])
def test_windows_long_for_the_sequence(dev, n, nk, window, d):
    q, k, v, d_o = make(dev, 2, n, nk, 6, 2, d, seed=window)
    o, lse = hk.attn_fwd(q, k, v, causal=True, window=window, sinks=1)
    want = ref.forward(q, k, v, window, 1)
    ref.close(o, want[0], want[1], "O")
    ref.close(lse, want[2], want[3], "L")
    for name, g, (r, bound) in zip(("dQ", "dK", "dV"), grads(q, k, v, d_o, window, 1), ref.backward(q, k, v, d_o, window, 1)):
        ref.close(g, r, bound, name)


@pytest.mark.parametrize("sinks", [0, 4])
def test_dq_in_the_place_of_q_and_the_others_in_theirs(dev, sinks):
    q, k, v, d_o = make(dev, 1, 700, 700, 4, 2, 128, seed=9)
    want = grads(q, k, v, d_o, 200, sinks)
    o, lse = hk.attn_fwd(q, k, v, causal=True, window=200, sinks=sinks)
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    _native.attn_bwd_strided(q, k, v, o, d_o, lse, q, dk, dv, causal=True, window=200, sinks=sinks)
    assert torch.equal(q, want[0]) and torch.equal(dk, want[1]) and torch.equal(dv, want[2])


def test_scores_far_apart(dev):
    for d in (64, 128):
        q, k, v, d_o = make(dev, 1, 500, 500, 2, 1, d, seed=5)
        k[:, 0] *= 10
        k[:, 300:310] *= 6
        for name, g, (r, bound) in zip(("dQ", "dK", "dV"), grads(q, k, v, d_o, 100, 2), ref.backward(q, k, v, d_o, 100, 2)):
            ref.close(g, r, bound, name)


def test_streams_and_a_graph(dev):
    sets = [make(dev, 1, 1500, 1500, 4, 2, 64, seed=i) for i in range(2)]
    want = [grads(*s, 200, 4) for s in sets]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in sets]
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(grads(*s, 200, 4))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = grads(*sets[1], 200, 4)
    for t in inside:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for w, g in ((want[0], got[0]), (want[1], got[1]), (want[1], inside)):
        assert all(torch.equal(x, y) for x, y in zip(w, g))


def test_one_in_a_chain_after_another(dev):
    """Backward after backward without a wait: what the second writes is not what the first still reads."""
    q, k, v, d_o = make(dev, 1, 900, 900, 4, 2, 128, seed=2)
    want = grads(q, k, v, d_o, 150, 3)
    many = [grads(q, k, v, d_o, 150, 3) for _ in range(20)]
    assert all(torch.equal(x, y) for m in many for x, y in zip(m, want))
    assert math.isfinite(float(want[0].float().sum()))
