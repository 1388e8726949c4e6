"""The first row of a sequence sees one key. Its P is 1 whatever the score, so that it has no gradient of it: zeros where a window hides
something, and no more than rounding where it hides nothing and the causal kernels run."""
import math

import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native

pytestmark = pytest.mark.gpu


def backward(q, k, v, d_o, window, sinks):
    o, lse = hk.attn_fwd(q, k, v, causal=True, window=window, sinks=sinks)
    out = [torch.empty_like(t) for t in (q, k, v)]
    _native.attn_bwd_strided(q, k, v, o, d_o, lse, *out, causal=True, window=window, sinks=sinks)
    return lse, *out


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,window,sinks", [(129, 128, 1), (300, 299, 1), (300, 5, 299), (700, 64, 0), (129, 129, 0), (300, 300, 0), (300, 2, 300),
                                            (300, 301, 4), (128, 128, 0), (40, 50, 60), (1000, 1 << 20, 0)])
def test_the_first_row(d, n, window, sinks):
    """Only the first row has a gradient of O here, so that dK and dV are of it alone.
    dS = P (dP - delta), delta = P' dP': dP and dP' are good to D 2^-23 of the sum of their products' sizes. P' is e^(s - L) with s good to
    D 2^-23 of the sum of its products' sizes, as is the s in L, L to 2^-19 + 2^-22 |L| beside that, and the exponential to 2^-20."""
    gen = torch.Generator().manual_seed(n + window)
    q, d_o = (torch.randn(2, n, 4, d, generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    k, v = (torch.randn(2, n, 2, d, generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    d_o[:, 1:] = 0
    lse, dq, dk, dv = backward(q, k, v, d_o, window, sinks)
    assert not bool(dq[:, 1:].any()) and not bool(dk[:, 1:].any()) and not bool(dv[:, 1:].any())
    kept = (dq[:, 0], dk[:, 0])
    if min(window, n) + sinks < n or max(window, sinks) < n or n <= 128:  # something is hidden, or there is one tile of keys
        assert not any(bool(t.any()) for t in kept)
    q0, g0 = q[:, 0].double(), d_o[:, 0].double()
    k0, v0 = (t[:, 0].double().repeat_interleave(2, 1) for t in (k, v))
    c, unit = 1 / math.sqrt(d), d * 2.0 ** -23
    p_err = 2 * unit * c * (q0 * k0).abs().sum(-1) + 2.0 ** -19 + 2.0 ** -22 * lse[:, :, 0, 0].abs().double() + 2.0 ** -20
    ds = (2 * unit * (g0 * v0).abs().sum(-1) + p_err * (g0 * v0).sum(-1).abs()) * c * (1 + 2.0 ** -6)
    assert bool((dq[:, 0].double().abs() <= ds[..., None] * k0.abs()).all())
    assert bool((dk[:, 0].double().abs() <= (ds[..., None] * q0.abs()).unflatten(1, (2, 2)).sum(2)).all())
    want = g0.unflatten(1, (2, 2)).sum(2)
    # P is rounded to bf16, and dV; at D = 64 an exponential of the causal kernel may be a polynomial's, good to 2^-13
    assert bool(((dv[:, 0].double() - want).abs() <= want.abs() * 2.0 ** -8 + g0.abs().unflatten(1, (2, 2)).sum(2) * (2.0 ** -8 + 2.0 ** -12)).all())
    assert _native.device_status(0) == 0


@pytest.mark.parametrize("window,sinks", [(300, 0), (7, 300), (1 << 20, 5)])
def test_where_nothing_is_hidden_the_forward_is_the_causal_one(window, sinks):
    for d in (64, 128):
        gen = torch.Generator().manual_seed(d)
        q = torch.randn(2, 200, 4, d, generator=gen).to(torch.bfloat16).cuda()
        k, v = (torch.randn(2, 300, 2, d, generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
        o, lse = hk.attn_fwd(q, k, v, causal=True, window=window, sinks=sinks)
        want, want_lse = hk.attn_fwd(q, k, v, causal=True)
        if d == 128:
            assert torch.equal(o, want) and torch.equal(lse, want_lse)
        else:
            # L: there a share of the exponentials are a polynomial's, good to 1.02e-4 (ex2_poly), by which a sum of them is off at most, and
            # its logarithm; the other terms of both L are 2^-19 each. O: two roundings each
            assert float((lse - want_lse).abs().max()) <= 1.02e-4 + 2 * 2.0 ** -19
            assert float((o.double() - want.double()).norm() / want.double().norm()) <= 2 * 2.0 ** -8
