"""The modules' native autograd functions and the Python ones behind them: the same outputs and gradients, and what a graph can
ask of a function (hooks on what it saves, a second derivative, a second backward, parts of the gradients, no graph at all)."""
import pytest
import torch

from hipkittens_b200 import _native
from hipkittens_b200.attention import HipCrossAttention, HipSelfAttention, QkNormRotary, QkNormRotaryFunction

pytestmark = pytest.mark.gpu


class _Nothing:
    """A front end that leaves every call to the Python code."""

    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture
def dev():
    assert torch.cuda.is_available(), "these tests need a B200"
    return torch.device("cuda:0")


def rand(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()


def both(monkeypatch, call):
    got = call()
    with monkeypatch.context() as m:
        m.setattr(_native, "_front_module", _Nothing())
        want = call()
    for x, y in zip(got, want):
        assert (x is None and y is None) or (x.dtype == y.dtype and torch.equal(x, y))
    return got


WINDOWS = [dict(), dict(window=50), dict(window=50, sinks=3)]


@pytest.mark.parametrize("window", WINDOWS)
@pytest.mark.parametrize("padded", [False, True])
def test_cross_attention(dev, monkeypatch, window, padded):
    gen = torch.Generator().manual_seed(1)
    q, kv, d_o = rand(gen, 2, 130, 6, 64).requires_grad_(), rand(gen, 2, 200, 2, 2, 64).requires_grad_(), rand(gen, 2, 130, 6, 64)
    mask = torch.arange(200, device=dev)[None] < torch.tensor([200, 140], device=dev)[:, None] if padded else None
    m = HipCrossAttention(causal=True, softmax_scale=0.2, **window)

    def call():
        o = m(q, kv, key_padding_mask=mask)
        return (o.detach(), *torch.autograd.grad(o, (q, kv), d_o))

    both(monkeypatch, call)
    both(monkeypatch, lambda: torch.autograd.grad(m(q, kv, key_padding_mask=mask), kv, d_o))
    both(monkeypatch, lambda: torch.autograd.grad(m(q.detach(), kv, key_padding_mask=mask), kv, d_o))
    both(monkeypatch, lambda: torch.autograd.grad(m(q, kv, key_padding_mask=mask), q, d_o.transpose(1, 2).contiguous().transpose(1, 2)))


@pytest.mark.parametrize("window", WINDOWS)
@pytest.mark.parametrize("layout", ["dense", "slice", "odd"])
def test_self_attention(dev, monkeypatch, window, layout):
    gen = torch.Generator().manual_seed(2)
    qkv, d_o = rand(gen, 2, 150, 3, 4, 128), rand(gen, 2, 150, 4, 128)
    if layout == "slice":
        qkv = rand(gen, 2, 300, 3, 4, 128)[:, ::2]
    if layout == "odd":  # strides that the kernels do not read: copied by the code behind
        qkv = rand(gen, 2, 150, 3, 4, 132)[..., :128]
    qkv.requires_grad_()
    m = HipSelfAttention(causal=True, **window)

    def call():
        o = m(qkv)
        return (o.detach(), *torch.autograd.grad(o, qkv, d_o))

    both(monkeypatch, call)
    with torch.no_grad():
        assert not m(qkv).requires_grad


@pytest.mark.parametrize("window", WINDOWS)
def test_saved_tensors_come_back_in_other_layouts(dev, window):
    gen = torch.Generator().manual_seed(3)
    q, kv, d_o = rand(gen, 2, 130, 4, 64).requires_grad_(), rand(gen, 2, 130, 2, 2, 64).requires_grad_(), rand(gen, 2, 130, 4, 64)
    m = HipCrossAttention(causal=True, **window)
    want = torch.autograd.grad(m(q, kv), (q, kv), d_o)

    def odd(t):  # the same values with strides that the kernels do not read
        if t.dim() < 4:
            return t
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 4, dtype=t.dtype, device=t.device)
        wide[..., :t.shape[-1]] = t
        return wide[..., :t.shape[-1]]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, odd):
        o = m(q, kv)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(o, (q, kv), d_o), want))
    with torch.autograd.graph.save_on_cpu():
        o = m(q, kv)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(o, (q, kv), d_o), want))


def test_graphs_of_a_module(dev):
    gen = torch.Generator().manual_seed(4)
    qkv, d_o = rand(gen, 1, 100, 3, 2, 64).requires_grad_(), rand(gen, 1, 100, 2, 64)
    m = HipSelfAttention(causal=True, window=30)
    o = m(qkv)
    first = torch.autograd.grad(o, qkv, d_o, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(o, qkv, d_o)[0], first)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(o, qkv, d_o)
    o = m(qkv)
    with torch.no_grad():
        qkv[0, 0] = 0
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(o, qkv, d_o)
    # accumulated into a leaf, and through a checkpoint
    qkv.grad = None
    m(qkv).backward(d_o)
    want = qkv.grad.clone()
    qkv.grad = None
    torch.utils.checkpoint.checkpoint(m, qkv, use_reentrant=False).backward(d_o)
    assert torch.equal(qkv.grad, want)


@pytest.mark.parametrize("weights", ["both", "one", "none", "frozen"])
@pytest.mark.parametrize("positions", [False, True])
def test_norm_and_rotation(dev, monkeypatch, weights, positions):
    gen = torch.Generator().manual_seed(5)
    qkv = rand(gen, 2, 70, 8, 64)
    q, k = qkv[:, :, :4].requires_grad_(), qkv[:, :, 4:6].requires_grad_()
    wq, wk = (1 + rand(gen, 64).float() / 4 for _ in range(2))
    wq = None if weights == "none" else wq
    wk = None if weights in ("one", "none") else wk
    leaves = [q, k] + [w.requires_grad_() for w in (wq, wk) if w is not None and weights != "frozen"]
    angle = torch.arange(80, device=dev)[:, None] / 100.0 ** (torch.arange(0, 64, 2, device=dev) / 64)
    pos = torch.randint(0, 80, (2, 70), generator=gen, dtype=torch.int32).to(dev) if positions else None
    dy = rand(gen, 2, 70, 4, 64), rand(gen, 2, 70, 2, 64)

    def call():
        y = QkNormRotaryFunction.apply(q, k, wq, wk, angle.cos(), angle.sin(), pos, 0 if positions else 4, 1e-5, positions)
        return (*(t.detach() for t in y), *torch.autograd.grad(y, leaves, dy))

    both(monkeypatch, call)
    both(monkeypatch, lambda: torch.autograd.grad(QkNormRotaryFunction.apply(q, k, wq, wk, angle.cos(), angle.sin(), pos)[1], leaves,
                                                  dy[1], allow_unused=True, materialize_grads=True))


def test_graphs_of_the_norm_and_rotation(dev, monkeypatch):
    gen = torch.Generator().manual_seed(6)
    q, k = rand(gen, 2, 70, 4, 64).requires_grad_(), rand(gen, 2, 70, 2, 64).requires_grad_()
    m = QkNormRotary(64, device=dev, dtype=torch.bfloat16)
    angle = torch.arange(70, device=dev)[:, None] / 100.0 ** (torch.arange(0, 64, 2, device=dev) / 64)
    cos, sin = angle.cos(), angle.sin()
    dy = rand(gen, 2, 70, 4, 64), rand(gen, 2, 70, 2, 64)
    y = m(q, k, cos, sin)
    want = torch.autograd.grad(y, (q, k, m.q_weight), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (q, k, m.q_weight), dy), want))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, q, dy)
    y = m(q, k, cos, sin)
    grads = torch.autograd.grad(y, (q, k), dy, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grads[0].float().sum().backward()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() == 4 else t):
        y = m(q, k, cos, sin)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (q, k, m.q_weight), dy), want))
    with torch.no_grad():
        assert not m(q, k, cos, sin)[0].requires_grad


def test_norm_and_rotation_in_a_graph(dev):
    """Captured forward and backward, on leaves that no other graph holds: torch joins the streams of two graphs of one leaf, which a
    capture does not survive."""
    gen = torch.Generator().manual_seed(6)
    x = [rand(gen, 2, 70, 4, 64).requires_grad_(), rand(gen, 2, 70, 2, 64).requires_grad_()]
    angle = torch.arange(70, device=dev)[:, None] / 100.0 ** (torch.arange(0, 64, 2, device=dev) / 64)
    cos, sin = angle.cos(), angle.sin()
    dy = rand(gen, 2, 70, 4, 64), rand(gen, 2, 70, 2, 64)
    m = QkNormRotary(64, device=dev, dtype=torch.bfloat16)
    want = torch.autograd.grad(m(*x, cos, sin), (*x, m.q_weight), dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = torch.autograd.grad(m(*x, cos, sin), (*x, m.q_weight), dy)
    for t in inside:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(inside, want))


def test_a_captured_backward_of_leaves_that_an_eager_graph_holds_is_refused(dev):
    """... before torch joins the two graphs' streams."""
    gen = torch.Generator().manual_seed(6)
    x = [rand(gen, 2, 70, 4, 64).requires_grad_(), rand(gen, 2, 70, 2, 64).requires_grad_()]
    cos = torch.ones(70, 32, device=dev)
    dy = rand(gen, 2, 70, 4, 64), rand(gen, 2, 70, 2, 64)
    m = QkNormRotary(64, device=dev, dtype=torch.bfloat16)
    eager = m(*x, cos, cos)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="no graph from before the capture holds"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(m(*x, cos, cos), (*x, m.q_weight), dy)
    want = torch.autograd.grad(eager, (*x, m.q_weight), dy)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = torch.autograd.grad(m(*x, cos, cos), (*x, m.q_weight), dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(inside, want))


def test_a_failure_of_the_backward_is_an_error(dev, monkeypatch):
    """A status that the device reports ends the call in either direction."""
    gen = torch.Generator().manual_seed(7)
    q, k = rand(gen, 1, 8, 2, 64).requires_grad_(), rand(gen, 1, 8, 2, 64).requires_grad_()
    qkv, d_o = rand(gen, 1, 100, 3, 2, 64).requires_grad_(), rand(gen, 1, 100, 2, 64)
    cos = torch.ones(8, 32, device=dev)
    bad = torch.full((1, 8), 9, dtype=torch.int32, device=dev)
    m = HipSelfAttention(causal=True, window=30)
    o = m(qkv)
    QkNormRotaryFunction.apply(q, k, None, None, cos, cos, bad)  # leaves a status behind, which the next wait reports
    with pytest.raises(RuntimeError, match="attention backward failed on the device"):
        torch.autograd.grad(o, qkv, d_o)
    QkNormRotaryFunction.apply(q, k, None, None, cos, cos, bad)
    with pytest.raises(RuntimeError, match="attention forward failed on the device"):
        m(qkv)
    assert _native.device_status(0) == 0
