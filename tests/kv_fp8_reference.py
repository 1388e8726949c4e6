"""The paged cache in 8 bits from its definition in 64 bits: what an append leaves in the blocks, and attention over them with bounds of what
a kernel that computes in fp32, fp16 and bf16 may be off by. Runs on the CPU.

A block is what a page holds of one head: 16 tokens of codes, and a scale. Rounding to e4m3 keeps 4 significant bits (half a step is 2^-4
of the value at most), or steps of 2^-9 below 2^-6.

Decode. The scores are sums of D products of exact factors in fp32, after a power of two of q's row (a value of q below 2^-14 of the row's
largest loses what lies below 2^-25 of that): D 2^-23 of the sum of the products' sizes, and 2^-24 of the row's largest q times the sum of |k|;
scaling them rounds twice more (2^-23 each). P, after the page's scale, is rounded to bf16 (2^-8 of each term), O once more; exponentials and
fp32 sums are good to 2^-16 of a term, and an error of a score is one of its exponential. L as the scores, the logarithm of a sum of
exponentials to 2^-20 and 2^-22 of itself."""
import math

import torch

PAGE, TOP = 16, 448.0


def e4m3(x):
    """The nearest e4m3 value, the even one of two, 448 at most; NaN stays."""
    x = x.double().clamp(-1e6, 1e6)
    size = x.abs().clamp(min=2.0 ** -40)
    power = torch.floor(torch.log2(size))
    power = torch.where(size < torch.exp2(power), power - 1, torch.where(size >= torch.exp2(power + 1), power + 1, power)).clamp(min=-6)
    step = torch.exp2(power - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def scale_for(amax):
    if math.isnan(amax):
        return math.nan
    if math.isinf(amax):
        return 2.0 ** 119
    e = -120
    while e < 119 and amax > TOP * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(codes, scales, pages, start, x):
    """Writes x [n, heads, D] at positions start ... of the sequence whose pages these are; codes [P,16,heads,D] and scales [P,heads], both
    64 bits, are changed in place."""
    n = x.shape[0]
    for slot in range(start // PAGE, (start + n - 1) // PAGE + 1):
        r0, r1 = max(0, start - slot * PAGE), min(PAGE, start + n - slot * PAGE)
        page = int(pages[slot])
        for h in range(x.shape[1]):
            new = x[slot * PAGE + r0 - start:slot * PAGE + r1 - start, h].double()
            s = scale_for(float(new.abs().max()) if not new.isnan().any() else math.nan)
            if r0 > 0:
                old = float(scales[page, h])
                s = math.nan if math.isnan(old) or math.isnan(s) else max(s, old)
                if s != old:
                    codes[page, :, h] = e4m3(codes[page, :, h] * old / s)
            codes[page, r0:r1, h] = e4m3(new / s)
            scales[page, h] = s


def rotate(x, start, cos, sin):
    """x [n, heads, D] at positions start ..., in 64 bits, and the size of what the two products add up to."""
    half = cos.shape[1]
    c, s = (t[start:start + x.shape[0]].double()[:, None] for t in (cos, sin))
    x = x.double()
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    y = torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()], -1)
    return y, size


def tokens(codes, scales, pages, n):
    pages = pages[:-(-n // PAGE)].long()
    return (codes[pages].double() * scales[pages].double()[:, None, :, None]).flatten(0, 1)[:n]


def decode(q, kc, vc, ks, vs, table, lens, window=None, sinks=0, scale=None):
    """(o, bound, l, bound)."""
    q, kc, vc, ks, vs, table, lens = (t.cpu() for t in (q, kc, vc, ks, vs, table, lens))
    s, _, h, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    g = h // kc.shape[2]
    o, bo = torch.zeros(s, 1, h, d).double(), torch.zeros(s, 1, h, d).double()
    l, bl = torch.full((s, h, 1, 1), -math.inf).double(), torch.zeros(s, h, 1, 1).double()
    for i in range(s):
        n = min(int(lens[i]), table.shape[1] * PAGE)
        if n <= 0:
            continue
        at = torch.arange(n)
        if window is not None:
            at = at[(n - 1 - at < window) | (at < sinks)]
        page = table[i].long()[at // PAGE]  # of the keys that are seen, and no others
        k, v = (c[page, at % PAGE].double() * t[page].double()[..., None] for c, t in ((kc, ks), (vc, vs)))
        for j in range(h):
            kj, vj, qj = k[:, j // g], v[:, j // g], q[i, 0, j].double()
            x = kj @ qj * scale
            p = torch.softmax(x, 0)
            off = scale * float((kj.abs() @ qj.abs()).max() * (d + 4) * 2 ** -23 + kj.abs().sum(1).max() * qj.abs().max() * 2 ** -24)
            o[i, 0, j] = p @ vj
            bo[i, 0, j] = (p @ vj.abs()) * (2 ** -8 + 2 ** -16 + 2 * off) + o[i, 0, j].abs() * 2 ** -8 + 1e-36
            l[i, j] = torch.logsumexp(x, 0)
            bl[i, j] = off + 2 ** -20 + float(l[i, j].abs()) * 2 ** -22
    return o, bo, l, bl
