"""Self-attention with a window over a right-padded batch: every sequence gives what it gives alone, at its rows' own positions; rows of
padding are zeros and pass nothing on. Against the definition in 64 bits, sequence by sequence."""
import pytest
import torch
import window_reference as ref

from hipkittens_b200 import _native
from hipkittens_b200.attention import HipSelfAttention

pytestmark = pytest.mark.gpu


def rand(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen).to(dtype).cuda()


def keep(lens, n):
    return torch.arange(n, device="cuda")[None] < torch.tensor(lens, device="cuda")[:, None]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,lens,window,sinks", [(300, (300, 150, 1), 60, 2), (257, (20, 256, 129), 9, 0), (40, (39, 2, 40), 64, 0),
                                                 (200, (7, 100, 200), 1, 3)])
def test_each_sequence_is_as_it_is_alone(d, n, lens, window, sinks):
    gen = torch.Generator().manual_seed(n + d)
    qkv, d_o = rand(gen, 3, n, 3, 2, d).requires_grad_(), rand(gen, 3, n, 2, d)
    o = HipSelfAttention(causal=True, window=window, sinks=sinks)(qkv, key_padding_mask=keep(lens, n))
    (got,) = torch.autograd.grad(o, qkv, d_o)
    for i, length in enumerate(lens):
        assert not bool(o[i, length:].any()) and not bool(got[i, length:].any())
        q, k, v = (t[None] for t in qkv[i, :length].detach().unbind(1))
        want = ref.forward(q, k, v, window, sinks)
        ref.close(o[i:i + 1, :length].detach(), want[0], want[1], "O")
        for j, (g, bound) in enumerate(ref.backward(q, k, v, d_o[i:i + 1, :length], window, sinks)):
            ref.close(got[i:i + 1, :length, j], g, bound, "dQ dK dV".split()[j])
    assert _native.device_status(0) == 0


def test_masks_that_are_refused_and_one_that_keeps_all():
    gen = torch.Generator().manual_seed(1)
    qkv = rand(gen, 2, 90, 3, 2, 64)
    m = HipSelfAttention(causal=True, window=20, sinks=1)
    assert torch.equal(m(qkv, key_padding_mask=keep((90, 90), 90)), m(qkv))
    holes = keep((90, 50), 90)
    holes[1, 3] = False
    for bad in (holes, ~keep((5, 5), 90), keep((90, 0), 90)):
        with pytest.raises(ValueError, match="right-padded"):
            m(qkv, key_padding_mask=bad)
    for bad in (keep((89, 89), 89), keep((50,), 90), keep((90, 50, 50), 90), keep((90, 50), 90).int()):
        with pytest.raises(ValueError, match="bool tensor"):
            m(qkv, key_padding_mask=bad)
    half = qkv.to(torch.float16)
    padded = m(half, key_padding_mask=keep((90, 33), 90))
    assert padded.dtype == torch.float16 and torch.equal(padded[1, :33], m(half)[1, :33]) and not bool(padded[1, 33:].any())
