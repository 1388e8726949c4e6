"""A sliding-window layer as it is trained and served: norm and rotation of q and k, the cache, attention with a window over a
sequence, over pages and for single tokens, one after the other, against the formulas in fp64."""
import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native
from hipkittens_b200.attention import HipCrossAttention, QkNormRotary

pytestmark = pytest.mark.gpu

EPS = 1e-6
HALF_STEP = torch.finfo(torch.bfloat16).eps / 2


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("a GPU test was selected without a GPU")
    return torch.device("cuda", 0)


def tables(rows, r, dev):
    angle = torch.arange(rows, device=dev)[:, None] / 1e4 ** (torch.arange(0, r, 2, device=dev) / r)
    return angle.cos(), angle.sin()


def plain_norm_rotary(x, w, cos, sin):
    """x [B, N, H, D] fp64, the halves of the first 2 cos.shape[1] values rotated."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    half = cos.shape[1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    c, s = cos[None, :, None], sin[None, :, None]
    return torch.cat((a * c - b * s, a * s + b * c, rest), -1)


def plain_attention(q, k, v, window, sinks):
    g = q.shape[2] // k.shape[2]
    k, v = (t.repeat_interleave(g, 2) for t in (k, v))
    s = torch.einsum("bnhd,bmhd->bhnm", q, k) * q.shape[3] ** -0.5
    n, c = torch.arange(q.shape[1], device=q.device)[:, None], torch.arange(k.shape[1], device=q.device)[None]
    seen = (c <= n) & ((n - c < window) | (c < sinks))
    return torch.einsum("bhnm,bmhd->bnhd", s.masked_fill(~seen, float("-inf")).softmax(-1), v)


def make(dev, b, n, h, hkv, d, seed):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, n, h + 2 * hkv, d, generator=gen).to(torch.bfloat16).to(dev)
    m = QkNormRotary(d, eps=EPS, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        for w in (m.q_weight, m.k_weight):
            w.copy_(1 + 0.1 * torch.randn(d, generator=gen))
    return qkv, m, gen


def off(got, want):
    got, want = got.detach().double(), want.detach()
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("b,n,h,hkv,d,window,sinks", [(2, 300, 4, 2, 128, 70, 4), (3, 333, 6, 2, 64, 100, 0), (1, 5, 2, 1, 64, 3, 1)])
def test_trained(dev, b, n, h, hkv, d, window, sinks):
    """Each rounding to bf16 moves what it rounds by at most half a step of it, in norm, and scores of size 1 pass theirs on as they are.
    On the way to O four: q and k behind the rotation, P, O. To the gradients eight: q, k, P, O (by delta), P once more in the backward,
    dS, the gradients behind the rotation and those in front of it."""
    qkv, m, gen = make(dev, b, n, h, hkv, d, n)
    qkv.requires_grad_()
    d_o = torch.randn(b, n, h, d, generator=gen).to(torch.bfloat16).to(dev)
    cos, sin = tables(n, d, dev)
    attention = HipCrossAttention(causal=True, window=window, sinks=sinks)
    q, k, v = qkv.split((h, hkv, hkv), 2)
    q, k = m(q, k, cos, sin)
    o = attention(q, torch.stack((k, v), 2))
    got = torch.autograd.grad(o, (qkv, m.q_weight, m.k_weight), d_o)

    x, wq, wk = (t.detach().double().requires_grad_() for t in (qkv, m.q_weight, m.k_weight))
    q, k, v = x.split((h, hkv, hkv), 2)
    c, s = cos.double(), sin.double()
    exact = plain_attention(plain_norm_rotary(q, wq, c, s), plain_norm_rotary(k, wk, c, s), v, window, sinks)
    want = torch.autograd.grad(exact, (x, wq, wk), d_o.double())
    assert off(o, exact.detach()) <= 4 * HALF_STEP
    for name, g, r in zip(("qkv", "q_weight", "k_weight"), got, want):
        assert off(g, r) <= 8 * HALF_STEP, name


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(40, 4), (17, 0), (500, 0)])
def test_served(dev, d, window, sinks):
    """Two users' prompts in chunks, then token by token, each token's q and k normalised and rotated at its position; the cache's other
    pages are never looked up."""
    b, n, h, hkv, pages = 2, 150, 4, 2, 10
    qkv, m, gen = make(dev, b, n, h, hkv, d, d)
    cos, sin = tables(n, d, dev)
    kp, vp = (torch.zeros(40, 16, hkv, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    table = torch.randperm(40, generator=gen)[:b * pages].view(b, pages).to(torch.int32).to(dev)
    done, outs = 0, []
    with torch.no_grad():
        for t in (64, 61, 19, *[1] * 6):
            q, k, v = qkv[:, done:done + t].split((h, hkv, hkv), 2)
            if t == 1:
                pos = torch.full((b, 1), done, dtype=torch.int32, device=dev)
                q, k = m(q, k, cos, sin, positions=pos)
            else:
                q, k = m(q, k, cos, sin, pos_offset=done)
            hk.paged_kv_append(k, v.contiguous(), kp, vp, table, torch.full((b,), done, dtype=torch.int32, device=dev))
            done += t
            lens = torch.full((b,), done, dtype=torch.int32, device=dev)
            attend = hk.paged_decode if t == 1 else lambda *a, **kw: hk.attn_fwd_paged(*a, causal=True, **kw)
            outs.append(attend(q, kp, vp, table, lens, window=window, sinks=sinks)[0])
            gone = max(0, (done + 1 - window) // 16)  # pages of keys that no later query sees
            table[:, -(-sinks // 16):gone] = -1
    assert _native.device_status(0) == 0 and done == n
    q, k, v = qkv.double().split((h, hkv, hkv), 2)
    c, s = cos.double(), sin.double()
    want = plain_attention(plain_norm_rotary(q, m.q_weight.double(), c, s), plain_norm_rotary(k, m.k_weight.double(), c, s), v, window, sinks)
    assert off(torch.cat(outs, 1), want.detach()) <= 4 * HALF_STEP
    for i in range(n - 6, n):
        assert off(torch.cat(outs, 1)[:, i], want[:, i].detach()) <= 4 * HALF_STEP
