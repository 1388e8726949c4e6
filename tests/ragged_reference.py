"""Attention over a ragged batch and its gradients, sequence by sequence from the definition in 64 bits, with bounds of what kernels that
compute in bf16 and fp32 may be off by. Runs where its inputs are.

Forward. P is rounded to bf16 for the product with V (2^-8 of each term) and O once more; exponentials and fp32 sums are good to 2^-16 of a
term. L: a score is a sum of D products in fp32, good to D 2^-23 of the sum of their sizes, the sum of exponentials to 2^-20, its
logarithm to 2^-20 and L to 2^-22 of itself.

Backward. With P and dS rounded to bf16 once each and the products' sums in fp32: dV is good to 2^-8 of the sum of its terms' sizes, and the
rounding of dV. dS = P (dP - delta): P carries the exponential's 2^-13 (a polynomial's 10^-4 for some), delta is a sum over the rounded O,
good to 2^-8 of the sum of |dO O|, and dS is rounded to bf16; an error of a score is one of P. dQ and dK are sums over dS, and rounded."""
import math

import torch


def sequences(cu_q, cu_k):
    q, k = cu_q.tolist(), cu_k.tolist()
    return [(slice(a, b), slice(c, d)) for a, b, c, d in zip(q, q[1:], k, k[1:])]


def attention(q, k, v, cu_q, cu_k, causal=True, scale=None, d_o=None):
    """[(value, bound)] of O, L and, with d_o, dQ, dK, dV. Rows without a sequence: 0 and -inf."""
    h, d, hkv = q.shape[1], q.shape[2], k.shape[1]
    c = 1 / math.sqrt(d) if scale is None else scale
    zero = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=q.device)  # noqa: E731
    o, bo, dq, bq, dk, bk, dv, bv = (zero(t) for t in (q, q, q, q, k, k, v, v))
    l, bl = torch.full((h, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device), torch.zeros(h, q.shape[0], dtype=torch.float64, device=q.device)
    for rq, rk in sequences(cu_q, cu_k):
        n, m = rq.stop - rq.start, rk.stop - rk.start
        if n == 0 or m == 0:
            continue
        pos = torch.arange(n, device=q.device)[:, None] + (m - n)
        see = torch.arange(m, device=q.device)[None, :] <= pos if causal else torch.ones(n, m, dtype=torch.bool, device=q.device)
        for j in range(h):
            qj, kj, vj = q[rq, j].double(), k[rk, j * hkv // h].double(), v[rk, j * hkv // h].double()
            x = (qj @ kj.T * c).masked_fill(~see, -math.inf)
            lj = torch.logsumexp(x, 1)
            p = torch.exp(x - lj[:, None]).masked_fill(~see, 0.0)
            oj, sizes = p @ vj, qj.abs() @ kj.abs().T * c
            o[rq, j], bo[rq, j] = oj, (p @ vj.abs()) * (2 ** -8 + 2 ** -16) + oj.abs() * 2 ** -8 + 1e-30
            l[j, rq] = lj
            bl[j, rq] = sizes.max() * d * 2 ** -23 + 2 ** -20 + lj.abs() * 2 ** -22
            if d_o is None:
                continue
            gj = d_o[rq, j].double()
            dp, delta = gj @ vj.T, (gj * oj).sum(1, keepdim=True)
            ds = p * (dp - delta) * c
            err = ds.abs() * (2 ** -8 + 2 ** -13 + sizes * d * 2 ** -23) + p * c * (
                2 ** -8 * (gj * oj).abs().sum(1, keepdim=True) + d * 2 ** -23 * (gj.abs() @ vj.abs().T))
            dq[rq, j], bq[rq, j] = ds @ kj, err @ kj.abs()
            dk[rk, j * hkv // h] += ds.T @ qj
            bk[rk, j * hkv // h] += err.T @ qj.abs()
            dv[rk, j * hkv // h] += p.T @ gj
            bv[rk, j * hkv // h] += (p * (2 ** -8 + 2 ** -13)).T @ gj.abs()
    grads = [(x, e + x.abs() * 2 ** -8 + 1e-30) for x, e in ((dq, bq), (dk, bk), (dv, bv))] if d_o is not None else []
    return [(o, bo), (l, bl), *grads]


def close(got, pair, what):
    ref, bound = pair
    got = got.double()
    same = (got == ref) | ((got - ref).abs() <= bound)
    assert bool(same.all()), (what, int((~same).sum()), float(((got - ref).abs() / bound.clamp(min=1e-300))[~same].max()),
                              (~same).nonzero()[:3].tolist())
