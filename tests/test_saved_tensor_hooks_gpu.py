"""The functions behind the modules under hooks on what they save: whatever layout the tensors come back in, the gradients are the same."""
import pytest
import torch

from hipkittens_b200 import _native
from hipkittens_b200.attention import HipAttnFunction, HipCrossAttention

pytestmark = pytest.mark.gpu


class _Nothing:
    """A front end whose modules leave every call to the Python code."""

    def __init__(self, front):
        self.front = front

    def __getattr__(self, name):
        return (lambda *args: None) if name == "packed_attention" else getattr(self.front, name)


def rand(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()


def wider(t, dims):
    """The same values with strides that the kernels do not read, for tensors of so many dimensions."""
    if t.dim() not in dims:
        return t
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 4, dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


@pytest.mark.parametrize("window", [(None, 0), (50, 3)])
@pytest.mark.parametrize("apart", [True, False])
def test_what_is_saved_comes_back_in_another_layout(monkeypatch, apart, window):
    gen = torch.Generator().manual_seed(3)
    d_o = rand(gen, 2, 130, 4, 64)
    if apart:
        leaves = [rand(gen, 2, 130, h, 64).requires_grad_() for h in (4, 2, 2)]
        call = lambda: HipAttnFunction.apply(*leaves, True, None, None, *window)  # noqa: E731
    else:
        leaves = [rand(gen, 2, 130, 4, 64).requires_grad_(), rand(gen, 2, 130, 2, 2, 64).requires_grad_()]
        monkeypatch.setattr(_native, "_front_module", _Nothing(_native._front()))
        call = lambda: HipCrossAttention(causal=True, window=window[0], sinks=window[1])(*leaves)  # noqa: E731
    want = torch.autograd.grad(call(), leaves, d_o)
    only_l = lambda t: wider(t, (4,)) if t.dtype == torch.float32 else t  # noqa: E731
    only_o = lambda t: wider(t, (4,)) if t.shape == d_o.shape else t  # noqa: E731
    hooks = [torch.autograd.graph.saved_tensors_hooks(lambda t: t, back) for back in
             (lambda t: wider(t, (4, 5)), only_l, only_o, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1))]
    for hook in (*hooks, torch.autograd.graph.save_on_cpu()):
        with hook:
            o = call()
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(o, leaves, d_o), want))
