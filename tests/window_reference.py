"""Attention with a window and sinks, and its gradients, from the definition in 64 bits, with bounds of what kernels that compute in
bf16 and fp32 may be off by. Runs where its inputs are.

Forward. P is rounded to bf16 for the product with V (2^-8 of each term) and O once more; exponentials and fp32 sums are good to
2^-16 of a term. L: a score is a sum of D products in fp32, good to D 2^-23 of the sum of their sizes, the sum of exponentials to
2^-20, its logarithm to 2^-20 and L to 2^-22 of itself.

Backward. With P and dS rounded to bf16 once each and the products' sums in fp32: dV is good to 2^-8 of the sum of its terms' sizes,
and the rounding of dV. dS = P (dP - delta): P carries the exponential's 2^-13 (a polynomial's 10^-4 for some), delta is a sum over the
rounded O, good to 2^-8 of the sum of |dO O|, and dS is rounded to bf16. dQ and dK are sums over dS, and rounded."""
import math

import torch


def visible(n, length, window, sinks, device):
    pos = torch.arange(n, device=device)[:, None] + (length - n)
    key = torch.arange(length, device=device)[None, :]
    return (key <= pos) & ((pos - key < window) | (key < sinks))


def forward(q, k, v, window, sinks, lens=None):
    """O, its bound, L, its bound."""
    b, n, h, d = q.shape
    nk, hkv = k.shape[1], k.shape[2]
    g = h // hkv
    o, bo = (torch.zeros(b, n, h, d, dtype=torch.float64, device=q.device) for _ in range(2))
    l = torch.full((b, h, 1, n), -math.inf, dtype=torch.float64, device=q.device)
    bl = torch.zeros_like(l)
    for i in range(b):
        length = nk if lens is None else int(lens[i])
        see = visible(n, length, window, sinks, q.device)
        for j in range(h):
            qj, kj, vj = q[i, :, j].double(), k[i, :length, j // g].double(), v[i, :length, j // g].double()
            x = (qj @ kj.T / math.sqrt(d)).masked_fill(~see, -math.inf)
            lj = torch.logsumexp(x, 1)
            p = torch.exp(x - lj[:, None]).masked_fill(~see, 0.0)
            o[i, :, j] = p @ vj
            bo[i, :, j] = (p @ vj.abs()) * (2 ** -8 + 2 ** -16) + o[i, :, j].abs() * 2 ** -8 + 1e-30
            l[i, j, 0] = lj
            size = (qj.abs() @ kj.abs().T).masked_fill(~see, 0.0).amax(1) / math.sqrt(d)
            bl[i, j, 0] = size * d * 2 ** -23 + 2 ** -19 + lj.abs().nan_to_num(posinf=0, neginf=0) * 2 ** -22
    return o, bo, l, bl


def backward(q, k, v, d_o, window, sinks, lens=None):
    """(dQ, bound), (dK, bound), (dV, bound)."""
    b, n, h, d = q.shape
    nk, hkv = k.shape[1], k.shape[2]
    g, c = h // hkv, 1 / math.sqrt(d)
    dq, bq = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    dk, bk, dv, bv = (torch.zeros(k.shape, dtype=torch.float64, device=q.device) for _ in range(4))
    for i in range(b):
        length = nk if lens is None else int(lens[i])
        see = visible(n, length, window, sinks, q.device)
        for j in range(h):
            qj, gj = q[i, :, j].double(), d_o[i, :, j].double()
            kj, vj = k[i, :length, j // g].double(), v[i, :length, j // g].double()
            x = (qj @ kj.T * c).masked_fill(~see, -math.inf)
            p = torch.exp(x - torch.logsumexp(x, 1)[:, None]).masked_fill(~see, 0.0)
            o = p @ vj
            dp, delta = gj @ vj.T, (gj * o).sum(1, keepdim=True)
            ds = p * (dp - delta) * c
            err = ds.abs() * (2 ** -8 + 2 ** -13) + p * c * (2 ** -8 * (gj * o).abs().sum(1, keepdim=True) +
                                                              d * 2 ** -23 * (gj.abs() @ vj.abs().T))
            # the score's own error moves P
            err = err + ds.abs() * (qj.abs() @ kj.abs().T) * c * d * 2 ** -23
            dq[i, :, j], bq[i, :, j] = ds @ kj, err @ kj.abs()
            dk[i, :length, j // g] += ds.T @ qj
            bk[i, :length, j // g] += err.T @ qj.abs()
            dv[i, :length, j // g] += p.T @ gj
            bv[i, :length, j // g] += (p * (2 ** -8 + 2 ** -13)).T @ gj.abs()
    return [(x, e + x.abs() * 2 ** -8 + 1e-30) for x, e in ((dq, bq), (dk, bk), (dv, bv))]


def close(got, ref, bound, what):
    got = got.double()
    same = (got == ref) | ((got - ref).abs() <= bound)
    assert bool(same.all()), (what, int((~same).sum()), float(((got - ref).abs() / bound.clamp(min=1e-300))[~same].max()),
                              (~same).nonzero()[:3].tolist())
