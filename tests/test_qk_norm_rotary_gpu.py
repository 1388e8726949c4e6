"""The norm and rotation of q and k, and its gradients, against the formulas in 64 bits.

Tolerances. Outputs are rounded once to bf16, off by at most 2^-8 of the value. Before that everything is fp32: a sum of D
squares is D / 16 + 7 roundings deep (16 in a lane, at most 4 across lanes), the square root's reciprocal is good to 2 ulp and
the products behind it are four roundings, so a value of the normalised pair (a, b) is good to (D / 16 + 24) 2^-24 of itself and
a turned one to that of |a| + |b|. The gradients have one more sum of the same depth. dw is a sum of rows; adding n terms in any order
is good to n 2^-24 of the sum of their sizes."""
import itertools

import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native
from hipkittens_b200.attention import QkNormRotary, QkNormRotaryFunction

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need a B200"
    return torch.device("cuda:0")


def make(dev, b, n, h, hkv, d, rot, rows=None, table=torch.float32, weight=torch.bfloat16, scattered=False, packed=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rows = rows or n
    if packed:
        qkv = (torch.randn(b, n, h + 2 * hkv, d, generator=gen) * 1.7).to(torch.bfloat16).to(dev)
        q, k = qkv[:, :, :h], qkv[:, :, h:h + hkv]
    else:
        q, k = ((torch.randn(b, n, x, d, generator=gen) * 1.7).to(torch.bfloat16).to(dev) for x in (h, hkv))
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=gen)).to(weight).to(dev) for _ in range(2))
    angle = torch.arange(rows, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    cos, sin = angle.cos().to(table).to(dev), angle.sin().to(table).to(dev)
    pos = torch.randint(0, rows, (b, n), generator=gen, dtype=torch.int32).to(dev) if scattered else None
    dq, dk = (torch.randn(b, n, x, d, generator=gen).to(torch.bfloat16).to(dev) for x in (h, hkv))
    return q, k, wq, wk, cos, sin, pos, dq, dk


def pairs(rot, interleaved):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def reference(x, w, cos, sin, pos, pos0, eps, interleaved, dy=None):
    """(o, bound of its error) or (dx, bound, dw, bound), in 64 bits on the CPU."""
    x, cos, sin = (t.detach().double().cpu() for t in (x, cos, sin))
    b, n, h, d = x.shape
    w = torch.ones(d, dtype=torch.float64) if w is None else w.detach().double().cpu()
    rot = 2 * cos.shape[1]
    at = torch.arange(n)[None].expand(b, n) + pos0 if pos is None else pos.long().cpu()
    good = (at >= 0) & (at < cos.shape[0])
    row = at.clamp(0, cos.shape[0] - 1)
    c, s = cos[row][:, :, None], sin[row][:, :, None]
    good = good[:, :, None, None]
    a, e = pairs(rot, interleaved)
    depth = (d / 16 + 24) * U
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if dy is None:
        y = x * r * w
        o, size = y.clone(), y.abs()
        o[..., a] = y[..., a] * c - y[..., e] * s
        o[..., e] = y[..., e] * c + y[..., a] * s
        size[..., a] = size[..., e] = y[..., a].abs() + y[..., e].abs()
        return o * good, (o.abs() * 2 ** -8 + depth * size + 1e-38) * good
    dy = dy.double().cpu()
    g, size = dy.clone(), dy.abs()
    g[..., a] = dy[..., a] * c + dy[..., e] * s
    g[..., e] = dy[..., e] * c - dy[..., a] * s
    size[..., a] = size[..., e] = dy[..., a].abs() + dy[..., e].abs()
    hat = x * r
    dx = r * (g * w - hat * (g * w * hat).mean(-1, keepdim=True))
    err = r * (size * w.abs() + hat.abs() * (size * w.abs() * hat.abs()).mean(-1, keepdim=True))
    terms = (g * hat * good).sum((0, 1, 2)), (size * hat.abs() * good).sum((0, 1, 2))
    return dx * good, (dx.abs() * 2 ** -8 + 2 * depth * err + 1e-38) * good, terms[0], (b * n * h + 2 * (d / 16 + 24)) * U * terms[1] + 1e-38


def close(got, ref, bound, what):
    diff = (got.double().cpu() - ref).abs()
    assert bool((diff <= bound).all()), (what, float((diff - bound).max()), float((diff / bound.clamp(min=1e-300)).max()))


CASES = [
    # b, n, h, hkv, d, rotated, interleaved, tables, weights, scattered positions, packed
    (1, 1, 1, 1, 64, 64, False, torch.float32, torch.bfloat16, False, False),
    (2, 77, 12, 4, 64, 32, True, torch.float32, torch.bfloat16, True, True),
    (3, 130, 8, 2, 128, 128, False, torch.bfloat16, torch.float32, False, True),
    (1, 515, 5, 1, 128, 48, False, torch.float32, torch.float32, True, False),
    (2, 33, 7, 7, 128, 128, True, torch.bfloat16, torch.bfloat16, True, True),
    (2, 19, 3, 1, 96, 96, False, torch.float32, torch.bfloat16, False, True),
    (1, 41, 6, 2, 80, 16, True, torch.bfloat16, torch.float32, True, True),
    (2, 29, 4, 2, 256, 128, False, torch.float32, torch.bfloat16, False, True),
    (1, 23, 4, 4, 192, 192, True, torch.float32, torch.bfloat16, True, True),
    (1, 9, 2, 1, 16, 16, False, torch.float32, torch.bfloat16, False, False),
    (4, 700, 24, 8, 128, 128, False, torch.float32, torch.bfloat16, False, True),   # rows for four a thread
    (2, 4096, 6, 2, 64, 64, True, torch.bfloat16, torch.bfloat16, True, True),
]


@pytest.mark.parametrize("b,n,h,hkv,d,rot,inter,table,weight,scattered,packed", CASES)
def test_forward_and_gradients(dev, b, n, h, hkv, d, rot, inter, table, weight, scattered, packed):
    q, k, wq, wk, cos, sin, pos, dq, dk = make(dev, b, n, h, hkv, d, rot, n + 5, table, weight, scattered, packed)
    args = (q, k, wq, wk, cos, sin)
    offset = 0 if scattered else 3
    out = hk.qk_norm_rotary(*args, positions=pos, pos_offset=offset, eps=1e-5, interleaved=inter)
    grads = hk.qk_norm_rotary_bwd(*args, dq, dk, positions=pos, pos_offset=offset, eps=1e-5, interleaved=inter)
    again = hk.qk_norm_rotary_bwd(*args, dq, dk, positions=pos, pos_offset=offset, eps=1e-5, interleaved=inter)
    assert _native.device_status(0) == 0
    assert all(torch.equal(x, y) for x, y in zip(grads, again))
    for name, x, w, o, dy, dx, dw in (("q", q, wq, out[0], dq, grads[0], grads[2]), ("k", k, wk, out[1], dk, grads[1], grads[3])):
        close(o, *reference(x, w, cos, sin, pos, offset, 1e-5, inter), name)
        rdx, bdx, rdw, bdw = reference(x, w, cos, sin, pos, offset, 1e-5, inter, dy)
        close(dx, rdx, bdx, "d" + name)
        assert dw.dtype == weight
        close(dw, rdw, bdw + rdw.abs() * (2 ** -8 if weight == torch.bfloat16 else U), "dw" + name)


def test_without_weights(dev):
    q, k, _, _, cos, sin, _, dq, dk = make(dev, 2, 65, 4, 2, 128, 64)
    out = hk.qk_norm_rotary(q, k, None, None, cos, sin)
    grads = hk.qk_norm_rotary_bwd(q, k, None, None, cos, sin, dq, dk)
    assert grads[2] is None and grads[3] is None
    for x, o, dy, dx in ((q, out[0], dq, grads[0]), (k, out[1], dk, grads[1])):
        close(o, *reference(x, None, cos, sin, None, 0, 1e-6, False), "o")
        close(dx, *reference(x, None, cos, sin, None, 0, 1e-6, False, dy)[:2], "dx")


def test_one_weight_only(dev):
    q, k, wq, _, cos, sin, _, dq, dk = make(dev, 2, 65, 4, 2, 64, 64)
    out = hk.qk_norm_rotary(q, k, wq, None, cos, sin)
    grads = hk.qk_norm_rotary_bwd(q, k, wq, None, cos, sin, dq, dk)
    assert grads[3] is None
    close(out[1], *reference(k, None, cos, sin, None, 0, 1e-6, False), "k")
    _, _, rdw, bdw = reference(q, wq, cos, sin, None, 0, 1e-6, False, dq)
    close(grads[2], rdw, bdw + rdw.abs() * 2 ** -8, "dwq")


def test_in_place_and_rows_of_others_stay(dev):
    q, k, wq, wk, cos, sin, _, _, _ = make(dev, 2, 100, 8, 2, 128, 128, packed=False)
    ref = hk.qk_norm_rotary(q, k, wq, wk, cos, sin)
    qkv = torch.full((2, 100, 12, 128), 7.0, dtype=torch.bfloat16, device=dev)
    qkv[:, :, :8], qkv[:, :, 8:10] = q, k
    packed = hk.qk_norm_rotary(qkv[:, :, :8], qkv[:, :, 8:10], wq, wk, cos, sin)
    out = hk.qk_norm_rotary(q, k, wq, wk, cos, sin, q_out=q, k_out=k)
    assert out[0].data_ptr() == q.data_ptr() and out[1].data_ptr() == k.data_ptr()
    assert all(torch.equal(x, y) for x, y in itertools.chain(zip(ref, out), zip(ref, packed)))
    assert bool((qkv[:, :, 10:] == 7).all())


def test_the_rotation_is_rotary_s_where_the_norm_is_the_identity(dev):
    """Rows of +-1 have a mean square of one: with eps = 0 and bf16 tables what is left is the rotation, whose two products and
    one sum are exact enough in fp32 to differ from rotary_bnhd's three bf16 roundings by three half steps at most."""
    gen = torch.Generator().manual_seed(1)
    x = torch.where(torch.rand(2, 64, 4, 128, generator=gen) < 0.5, -1.0, 1.0).to(torch.bfloat16).to(dev)
    *_, cos, sin, _, _, _ = make(dev, 2, 64, 4, 2, 128, 128, table=torch.bfloat16)
    o, _ = hk.qk_norm_rotary(x, x, None, None, cos, sin, eps=0.0)
    assert float((o.float() - hk.rotary_bnhd(x, cos, sin).float()).abs().max()) <= 3 * 2 * 2 ** -8


def test_positions_outside_the_tables_are_zeros_and_reported(dev):
    q, k, wq, wk, cos, sin, pos, dq, dk = make(dev, 2, 50, 4, 2, 64, 64, 50, scattered=True)
    pos[0, 3], pos[1, 49], pos[1, 0] = -1, 50, 2 ** 31 - 1
    out = hk.qk_norm_rotary(q, k, wq, wk, cos, sin, positions=pos)
    assert _native.device_status(0) == _native.HK_EBADPOS
    grads = hk.qk_norm_rotary_bwd(q, k, wq, wk, cos, sin, dq, dk, positions=pos)
    assert _native.device_status(0) == _native.HK_EBADPOS and _native.device_status(0) == 0
    for x, w, o, dy, dx, dw in ((q, wq, out[0], dq, grads[0], grads[2]), (k, wk, out[1], dk, grads[1], grads[3])):
        close(o, *reference(x, w, cos, sin, pos, 0, 1e-6, False), "o")
        rdx, bdx, rdw, bdw = reference(x, w, cos, sin, pos, 0, 1e-6, False, dy)
        close(dx, rdx, bdx, "dx")
        close(dw, rdw, bdw + rdw.abs() * 2 ** -8, "dw")


def test_rows_of_zeros_large_and_small_values(dev):
    q, k, wq, wk, cos, sin, _, dq, dk = make(dev, 1, 8, 4, 2, 128, 128, packed=False)
    q[0, 0] = 0
    q[0, 1] *= 2.0 ** 40
    q[0, 2] *= 2.0 ** -40
    out = hk.qk_norm_rotary(q, k, wq, wk, cos, sin)
    grads = hk.qk_norm_rotary_bwd(q, k, wq, wk, cos, sin, dq, dk)
    close(out[0], *reference(q, wq, cos, sin, None, 0, 1e-6, False), "q")
    close(grads[0], *reference(q, wq, cos, sin, None, 0, 1e-6, False, dq)[:2], "dq")


@pytest.mark.parametrize("inter", [False, True])
def test_gradients_are_those_of_differences(dev, inter):
    """d/dt of sum(o dy) along a direction, by central differences of the definition in 64 bits, against the kernel's gradients:
    what is left is their own rounding to bf16 (2^-8 of each term) and the differences' (1e-6)."""
    q, k, wq, wk, cos, sin, _, dq, dk = make(dev, 1, 17, 3, 1, 64, 32, weight=torch.float32)
    grads = hk.qk_norm_rotary_bwd(q, k, wq, wk, cos, sin, dq, dk, interleaved=inter)
    gen = torch.Generator().manual_seed(5)
    c, s = cos.double().cpu()[:, None], sin.double().cpu()[:, None]
    a, e = pairs(32, inter)

    def loss(x, w, dy):
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        o = y.clone()
        o[..., a], o[..., e] = y[..., a] * c - y[..., e] * s, y[..., e] * c + y[..., a] * s
        return float((o * dy).sum())

    for x, w, dy, dx, dw in ((q, wq, dq, grads[0], grads[2]), (k, wk, dk, grads[1], grads[3])):
        x, w, dy, dx, dw = (t.double().cpu() for t in (x, w, dy, dx, dw))
        vx, vw = torch.randn(x.shape, generator=gen).double(), torch.randn(w.shape, generator=gen).double()
        for got, terms, f in ((float((dx * vx).sum()), (dx * vx).abs().sum(), lambda t: loss(x + t * vx, w, dy)),
                              (float((dw * vw).sum()), (dw * vw).abs().sum(), lambda t: loss(x, w + t * vw, dy))):
            slope = (f(1e-5) - f(-1e-5)) / 2e-5
            assert abs(got - slope) <= float(terms) * (2 ** -8 + 1e-6)


def test_module_and_function_give_the_call_s_results(dev):
    q, k, wq, wk, cos, sin, _, dq, dk = make(dev, 2, 40, 4, 2, 64, 64, weight=torch.bfloat16)
    mod = QkNormRotary(64, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        mod.q_weight.copy_(wq)
        mod.k_weight.copy_(wk)
    q1, k1 = q.detach().requires_grad_(), k.detach().requires_grad_()
    out = mod(q1, k1, cos, sin)
    got = torch.autograd.grad(out, (q1, k1, mod.q_weight, mod.k_weight), (dq, dk))
    ref = hk.qk_norm_rotary_bwd(q, k, wq, wk, cos, sin, dq, dk)
    assert all(torch.equal(x, y) for x, y in zip(out, hk.qk_norm_rotary(q, k, wq, wk, cos, sin)))
    assert all(torch.equal(x, y) for x, y in zip(got, ref))
    # one output unused, its gradient zero; gradients in another layout
    dq_t = dq.transpose(1, 2).contiguous().transpose(1, 2)
    got = torch.autograd.grad(mod(q1, k1, cos, sin)[0], (q1, k1, mod.q_weight), dq_t)
    assert torch.equal(got[0], ref[0]) and not bool(got[1].any()) and torch.equal(got[2], ref[2])
    with pytest.raises(RuntimeError, match="cos and sin have no gradients"):
        QkNormRotaryFunction.apply(q1, k1, wq, wk, cos.requires_grad_(), sin)


def test_two_calls_at_once_on_other_streams_and_in_a_graph(dev):
    sets = [make(dev, 2, 300, 8, 2, 128, 128, seed=i) for i in range(2)]
    refs = [(hk.qk_norm_rotary(*s[:6]), hk.qk_norm_rotary_bwd(*s[:6], *s[7:])) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append((hk.qk_norm_rotary(*s[:6]), hk.qk_norm_rotary_bwd(*s[:6], *s[7:])))
    torch.cuda.synchronize()
    given = hk.qk_norm_rotary(*sets[0][:6], stream=streams[1]), hk.qk_norm_rotary_bwd(*sets[0][:6], *sets[0][7:], stream=streams[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = hk.qk_norm_rotary(*sets[1][:6]), hk.qk_norm_rotary_bwd(*sets[1][:6], *sets[1][7:])
    for t in (*inside[0], *inside[1]):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for r, g in ((refs[0], got[0]), (refs[1], got[1]), (refs[0], given), (refs[1], inside)):
        assert all(torch.equal(x, y) for x, y in zip((*r[0], *r[1]), (*g[0], *g[1])))
