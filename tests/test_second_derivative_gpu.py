"""Gradients that were asked for with a graph of their own (create_graph) have none through these functions: differentiating them
again is an error, and not a term that is missing."""
import pytest
import torch

from hipkittens_b200 import _native
from hipkittens_b200.attention import HipAttnFunction, HipCrossAttention, HipSelfAttention

pytestmark = pytest.mark.gpu


class _Nothing:
    def __getattr__(self, name):
        return lambda *args: None


def rand(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(len(shape))).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("window", [dict(), dict(window=20, sinks=2)])
@pytest.mark.parametrize("kind", ["self", "cross", "cross_kv_only", "apart"])
def test_a_second_derivative_is_refused(monkeypatch, kind, window, native):
    if not native:
        monkeypatch.setattr(_native, "_front_module", _Nothing())
    q, kv, qkv = rand(2, 50, 4, 64), rand(2, 50, 2, 2, 64), rand(2, 50, 3, 4, 64)
    if kind == "self":
        leaves, call = [qkv], lambda x: HipSelfAttention(causal=True, **window)(x)
    elif kind == "cross":
        leaves, call = [q, kv], lambda *x: HipCrossAttention(causal=True, **window)(*x)
    elif kind == "cross_kv_only":
        leaves, call = [kv], lambda x: HipCrossAttention(causal=True, **window)(q, x)
    else:
        leaves = [q, *(t.contiguous() for t in kv.unbind(2))]
        call = lambda *x: HipAttnFunction.apply(*x, True, None, None, window.get("window"), window.get("sinks", 0))  # noqa: E731
    for t in leaves:
        t.requires_grad_()
    want = torch.autograd.grad(call(*leaves).float().square().sum(), leaves)
    got = torch.autograd.grad(call(*leaves).float().square().sum(), leaves, create_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    for g in got:
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (call(*leaves).float().sum() + g.float().square().sum()).backward()
