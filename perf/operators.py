"""Operators of a sliding-window layer, as cases that can be timed: plain torch, or the package's own kernels.

    train    HipCrossAttention(causal=True, window=, sinks=) on q and a packed kv, forward and gradients
    prefill  attn_fwd(causal=True, window=, sinks=) on strided views of a packed projection
    chunk    attn_fwd_paged(causal=True, window=, sinks=): a chunk of each sequence against its paged cache
    decode   paged_decode(window=, sinks=): one new token of each sequence against its paged cache
    qkn      qk_norm_rotary: RMS norm of every head of q and k and the rotation of its position, in one pass
    qkn_train  QkNormRotaryFunction: the same with its gradients

A query at position p (the last query of a sequence is at its last key) sees the keys c <= p with p - c < window or
c < sinks. Lengths come from the case alone, values, page ids and scattered positions from the seed.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
EPS = 1e-6


def listed():
    return [
        # one pre-training step of a window layer with grouped heads at the long-context benchmark's length
        dict(name="train_gqa_d128", kind="train", b=2, n=8192, nk=8192, h=32, hkv=8, d=128, window=1024, sinks=4, padded=False, lens=0),
        # an odd length, three heads to a group, no sinks
        dict(name="train_odd_d64", kind="train", b=3, n=1777, nk=1777, h=12, hkv=4, d=64, window=300, sinks=0, padded=False, lens=0),
        # gradients of a small model, where launches and host work count
        dict(name="train_small_d64", kind="train", b=1, n=384, nk=384, h=8, hkv=2, d=64, window=128, sinks=2, padded=False, lens=0),
        # fine-tuning on right-padded sequences: rows in front of the padding see no key at all
        dict(name="train_padded_mha_d64", kind="train", b=8, n=1024, nk=1024, h=16, hkv=16, d=64, window=256, sinks=16, padded=True, lens=3),
        # a long prompt in one forward
        dict(name="prefill_long_d128", kind="prefill", b=1, n=16384, nk=16384, h=32, hkv=8, d=128, window=2048, sinks=64, padded=False, lens=0),
        # chunked prefill of a few sequences against what they have cached
        dict(name="chunk_d128", kind="chunk", b=4, t=512, lo=2048, hi=8192, h=64, hkv=8, d=128, window=2048, sinks=4, pool=4096, lens=1),
        # one interactive user behind a long conversation
        dict(name="decode_single_d128", kind="decode", b=1, lo=12000, hi=12500, h=32, hkv=8, d=128, window=4096, sinks=4, pool=4096, lens=2),
        # a full serving batch
        dict(name="decode_batch64_d128", kind="decode", b=64, lo=512, hi=8192, h=64, hkv=8, d=128, window=2048, sinks=4, pool=40000, lens=1),
        # small heads, six to a group, contexts from one token on, a window that is no multiple of a page
        dict(name="decode_odd_d64", kind="decode", b=33, lo=1, hi=4096, h=48, hkv=8, d=64, window=500, sinks=20, pool=10000, lens=5),
        # the pass in front of attention in a training step, on views of the packed projection
        dict(name="qkn_train_d128", kind="qkn_train", b=4, n=4096, h=32, hkv=8, d=128, rot=128, interleaved=False, table="float32", scattered=False, rows=4096),
        # part of the head rotated, neighbours as pairs, positions of packed documents
        dict(name="qkn_train_odd_d64", kind="qkn_train", b=3, n=1777, h=12, hkv=4, d=64, rot=32, interleaved=True, table="float32", scattered=True, rows=1777),
        # one new token of each sequence of a serving batch, far into its context
        dict(name="qkn_token_d128", kind="qkn", b=64, n=1, h=64, hkv=8, d=128, rot=128, interleaved=False, table="bfloat16", scattered=True, rows=131072),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    flops, nbytes, scores = max(w["flops"] for w in most), max(w["bytes"] for w in most), max(_scores(c) for c in listed())
    while True:
        kind = rng.choice(["train", "train", "prefill", "chunk", "decode", "decode", "qkn", "qkn_train"])
        hkv, g = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 5, 6, 7, 8])
        c = dict(kind=kind, h=hkv * g, hkv=hkv, d=rng.choice([64, 128]))
        if kind in ("qkn", "qkn_train"):
            c["d"] = rng.choice([64, 64, 96, 128, 128, 128, 192, 256])
            c |= dict(b=_log_int(rng, 1, 64), n=_log_int(rng, 1, 8192) if kind == "qkn_train" or rng.random() < 0.5 else 1)
            c |= dict(rot=16 * rng.randint(1, c["d"] // 16) if rng.random() < 0.4 else c["d"], interleaved=rng.random() < 0.5)
            c |= dict(table=rng.choice(["float32", "bfloat16"]), scattered=rng.random() < 0.5)
            c["rows"] = c["n"] + _log_int(rng, 1, 100000) if c["scattered"] else c["n"]
        else:
            c |= dict(window=_log_int(rng, 1, 4096), sinks=rng.choice([0, rng.randint(1, 8), rng.randint(1, 200)]), lens=rng.randint(0, 999))
            if kind in ("train", "prefill"):
                c |= dict(b=_log_int(rng, 1, 16), n=_log_int(rng, 1, 8192 if kind == "train" else 16384), padded=rng.random() < 0.3)
                c["nk"] = c["n"] if rng.random() < 0.6 else _log_int(rng, 1, 8192)
            else:
                c |= dict(b=_log_int(rng, 1, 64 if kind == "decode" else 8), lo=_log_int(rng, 1, 4096))
                c["hi"] = c["lo"] + _log_int(rng, 1, 8192)
                if kind == "chunk":
                    c["t"] = _log_int(rng, 1, 1024)
                c["pool"] = c["b"] * -(-c["hi"] // PAGE) + rng.randint(1, 100)
        w = work(c)
        if w["flops"] <= flops and w["bytes"] <= nbytes and _scores(c) <= scores:
            return c


def _lens(c):
    """Keys of each sequence: kept ones of a padded batch, or what the cache holds."""
    r = np.random.RandomState(c["lens"])
    if c["kind"] in ("chunk", "decode"):
        return r.randint(c["lo"], c["hi"] + 1, c["b"])
    if c["padded"]:
        return r.randint(max(1, c["nk"] // 4), c["nk"] + 1, c["b"])
    return np.full(c["b"], c["nk"])


def _queries(c):
    return c.get("t", 1) if c["kind"] in ("chunk", "decode") else c["n"]


def _block(c):
    """Query rows that the plain form takes together."""
    return min(_queries(c), 512)


def _scores(c):
    if c["kind"].startswith("qkn"):
        return 0
    n, rows = _queries(c), _block(c)
    return c["b"] * c["h"] * -(-n // rows) * rows * (rows - 1 + c["window"] + c["sinks"])


def work(c):
    if c["kind"].startswith("qkn"):
        values = c["b"] * c["n"] * (c["h"] + c["hkv"]) * c["d"]
        table = min(c["rows"], c["b"] * c["n"]) * c["rot"] * (4 if c["table"] == "float32" else 2)
        passes = 5 if c["kind"] == "qkn_train" else 2  # x in, y out; x and dy in, dx out
        return {"bytes": values * 2 * passes + table * (2 if passes == 5 else 1) + 4 * c["d"], "flops": values * (24 if passes == 5 else 8)}
    n, lens, d = _queries(c), _lens(c), c["d"]
    pairs = touched = 0
    for length in lens:
        p = np.arange(n, dtype=np.int64) + (int(length) - n)
        p = p[p >= 0]
        if p.size:
            pairs += int(np.sum(np.minimum(p + 1, c["window"]) + np.clip(p - c["window"] + 1, 0, c["sinks"])))
            lo = max(0, int(p[0]) - c["window"] + 1)
            touched += int(p[-1]) + 1 - lo + min(lo, c["sinks"])
    q_bytes, kv_bytes = 2 * c["b"] * n * c["h"] * d, 4 * touched * c["hkv"] * d
    if c["kind"] == "train":  # O, dQ and dO beside Q; dK and dV beside K and V, with a row for every key
        return {"bytes": 4 * q_bytes + kv_bytes + 4 * c["b"] * c["nk"] * c["hkv"] * d, "flops": 14 * d * c["h"] * pairs}
    return {"bytes": 2 * q_bytes + kv_bytes + 4 * c["b"] * n * c["h"], "flops": 4 * d * c["h"] * pairs}


# ---------------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)


def prepare(case, seed):
    c = case
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    b, h, hkv, d = c["b"], c["h"], c["hkv"], c["d"]
    s = {"case": c}
    if c["kind"].startswith("qkn"):
        n, rot, dtype = c["n"], c["rot"], getattr(torch, c["table"])
        qkv = _randn(gen, b, n, h + 2 * hkv, d, scale=1.7)  # a packed projection, of which v is not looked at
        s["q"], s["k"] = qkv[:, :, :h], qkv[:, :, h:h + hkv]
        s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(torch.bfloat16) for _ in range(2))
        angle = torch.arange(c["rows"], device="cuda", dtype=torch.float64)[:, None] / 500000.0 ** (
            torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        s["cos"], s["sin"] = angle.cos().to(dtype), angle.sin().to(dtype)
        s["positions"] = torch.randint(0, c["rows"], (b, n), generator=gen, device="cuda", dtype=torch.int32) if c["scattered"] else None
        if c["kind"] == "qkn_train":
            s["dq"], s["dk"] = _randn(gen, b, n, h, d), _randn(gen, b, n, hkv, d)
            for name in ("q", "k", "wq", "wk"):
                s[name] = s[name].requires_grad_()
        return s
    lens = _lens(c)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if c["kind"] in ("chunk", "decode"):
        n, width = _queries(c), -(-c["hi"] // PAGE)
        s["q"] = _randn(gen, b, n, h, d)
        s["k_pages"], s["v_pages"] = (_randn(gen, c["pool"], PAGE, hkv, d) for _ in range(2))
        order = torch.randperm(c["pool"], generator=gen, device="cuda").to(torch.int32)
        s["table"] = order[torch.arange(b * width, device="cuda") % c["pool"]].reshape(b, width).contiguous()
        return s
    n, nk = c["n"], c["nk"]
    if c["kind"] == "prefill" and n == nk:  # views of one packed projection
        qkv = _randn(gen, b, n, h + 2 * hkv, d)
        s["q"], s["k"], s["v"] = qkv[:, :, :h], qkv[:, :, h:h + hkv], qkv[:, :, h + hkv:]
    else:
        s["q"], s["kv"] = _randn(gen, b, n, h, d), _randn(gen, b, nk, 2, hkv, d)
        s["k"], s["v"] = s["kv"].unbind(2)
    if c["kind"] == "train":
        s["d_o"] = _randn(gen, b, n, h, d)
        s["q"], s["kv"] = s["q"].requires_grad_(), s["kv"].requires_grad_()
        if c["padded"]:
            s["mask"] = torch.arange(nk, device="cuda")[None, :] < s["lens"][:, None]
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state)
    if kind.startswith("qkn"):
        return _plain_qkn(state)
    return _plain_attention(state)


def _run_own(s):
    import hipkittens_b200 as hk
    from hipkittens_b200.attention import HipCrossAttention, QkNormRotaryFunction

    c = s["case"]
    if c["kind"] == "qkn":
        return hk.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], positions=s["positions"], eps=EPS,
                                 interleaved=c["interleaved"])
    if c["kind"] == "qkn_train":
        y = QkNormRotaryFunction.apply(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"], 0, EPS, c["interleaved"])
        return (*(t.detach() for t in y), *torch.autograd.grad(y, (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"])))
    window = dict(window=c["window"], sinks=c["sinks"])
    if c["kind"] == "train":
        if "module" not in s:  # which a program makes once
            s["module"] = HipCrossAttention(causal=True, **window)
        o = s["module"](s["q"], s["kv"], key_padding_mask=s.get("mask"))
        return (o.detach(), *torch.autograd.grad(o, (s["q"], s["kv"]), s["d_o"]))
    if c["kind"] == "prefill":
        return hk.attn_fwd(s["q"], s["k"], s["v"], causal=True, kv_lens=s["lens"] if c["padded"] else None, **window)
    if c["kind"] == "chunk":
        return hk.attn_fwd_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], causal=True, **window)
    return hk.paged_decode(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], **window)


def _plain_attention(s):
    """Blocks of query rows, each against the keys that one of its rows may see, gathered by index."""
    c = s["case"]
    q, lens, window, sinks, d = s["q"].detach(), s["lens"].long(), c["window"], c["sinks"], c["d"]
    b, n, h, _ = q.shape
    hkv, rows, scale = c["hkv"], _block(c), 1 / math.sqrt(d)
    blocks = -(-n // rows)
    at = torch.arange(blocks * rows, device="cuda").reshape(blocks, rows)[None] + (lens - n)[:, None, None]  # position of a row
    lo = (at[:, :, :1] - window + 1).clamp(min=0)
    keys = torch.cat([torch.arange(sinks, device="cuda").expand(b, blocks, sinks), lo + torch.arange(window + rows - 1, device="cuda")], 2)
    first = torch.cat([torch.zeros_like(lo).expand(b, blocks, sinks), lo.expand(b, blocks, window + rows - 1)], 2)
    own_span = (keys >= first) & ((torch.arange(keys.shape[2], device="cuda") >= sinks) | (keys < lo))  # each key once
    key, pos = keys[:, :, None, :], at[:, :, :, None]
    seen = own_span[:, :, None, :] & (key <= pos) & ((key > pos - window) | (key < sinks)) & (key < lens[:, None, None, None])
    pad = (0, 0, 0, 0, 0, blocks * rows - n)
    qb = torch.nn.functional.pad(q.float(), pad).reshape(b, blocks, rows, hkv, h // hkv, d)
    which = torch.arange(b, device="cuda")[:, None, None]
    if "k_pages" in s:
        place = keys.clamp(max=s["table"].shape[1] * PAGE - 1)
        page, row = s["table"][which, place // PAGE].long(), place % PAGE
        k, v = s["k_pages"][page, row].float(), s["v_pages"][page, row].float()
    else:
        place = keys.clamp(max=c["nk"] - 1)
        k, v = s["k"].detach()[which, place].float(), s["v"].detach()[which, place].float()
    score = torch.einsum("bnrhgd,bnkhd->bnhgrk", qb, k) * scale
    score = torch.where(seen[:, :, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total == 0, -math.inf, top + torch.log(total))
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.einsum("bnhgrk,bnkhd->bnrhgd", p, v)
    out = o.reshape(b, blocks * rows, h, d)[:, :n].to(torch.bfloat16)
    if c["kind"] != "train":
        return out, lse[..., 0].permute(0, 2, 3, 1, 4).reshape(b, h, 1, blocks * rows)[..., :n].contiguous()
    g = torch.nn.functional.pad(s["d_o"].float(), pad).reshape(qb.shape)
    delta = (g * o).sum(-1).permute(0, 1, 3, 4, 2)[..., None]
    ds = p * (torch.einsum("bnrhgd,bnkhd->bnhgrk", g, v) - delta) * scale
    dq = torch.einsum("bnhgrk,bnkhd->bnrhgd", ds, k).reshape(b, blocks * rows, h, d)[:, :n]
    dkv = torch.stack([torch.einsum("bnhgrk,bnrhgd->bnkhd", ds, qb), torch.einsum("bnhgrk,bnrhgd->bnkhd", p, g)], 3)
    to = (which * c["nk"] + place).reshape(-1)
    grad = torch.zeros(b * c["nk"], 2, hkv, d, device="cuda").index_add_(0, to, dkv.reshape(-1, 2, hkv, d))
    return out, dq.to(torch.bfloat16), grad.reshape(s["kv"].shape).to(torch.bfloat16)


def _halves(x, rot, interleaved):
    """The two values of each rotated pair."""
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])


def _joined(a, b, x, rot, interleaved):
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_qkn(s):
    c = s["case"]
    rot, inter = c["rot"], c["interleaved"]
    n = torch.arange(c["n"], device="cuda") if s["positions"] is None else s["positions"].long()
    cos, sin = s["cos"].float()[n][..., None, :], s["sin"].float()[n][..., None, :]

    def forward(x, w):
        x, w = x.detach().float(), w.detach().float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        y = x * r * w
        a, b = _halves(y, rot, inter)
        return x, w, r, _joined(a * cos - b * sin, b * cos + a * sin, y, rot, inter).to(torch.bfloat16)

    def backward(x, w, r, dy):
        dy = dy.float()
        a, b = _halves(dy, rot, inter)
        g = _joined(a * cos + b * sin, b * cos - a * sin, dy, rot, inter)
        hat = x * r
        dhat = g * w
        dx = r * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))
        return dx.to(torch.bfloat16), (g * hat).sum((0, 1, 2)).to(torch.bfloat16)

    xq, wq, rq, q = forward(s["q"], s["wq"])
    xk, wk, rk, k = forward(s["k"], s["wk"])
    if c["kind"] == "qkn":
        return q, k
    dq, dwq = backward(xq, wq, rq, s["dq"])
    dk, dwk = backward(xk, wk, rk, s["dk"])
    return q, k, dq, dk, dwq, dwk


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_qkn(s) if case["kind"].startswith("qkn") else _exact_attention(s)


def _exact_qkn(s):
    """The rotation as a product of complex numbers, the gradients by automatic differentiation."""
    c = s["case"]
    leaves = [s[name].detach().double().requires_grad_() for name in ("q", "k", "wq", "wk")]
    at = torch.arange(c["n"], device="cuda") if s["positions"] is None else s["positions"].long()
    turn = torch.complex(s["cos"].double()[at], s["sin"].double()[at]).unsqueeze(-2)

    def one(x, w):
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["d"] + EPS) * w
        head, tail = y.split([c["rot"], c["d"] - c["rot"]], -1)
        pairs = head.unflatten(-1, (-1, 2)) if c["interleaved"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return torch.cat([z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2), tail], -1)

    y = one(leaves[0], leaves[2]), one(leaves[1], leaves[3])
    if c["kind"] == "qkn":
        return tuple(t.detach() for t in y)
    grads = torch.autograd.grad(y, leaves, (s["dq"].double(), s["dk"].double()))
    return (*(t.detach() for t in y), *grads)


def _exact_attention(s):
    """Sequence by sequence and K/V head by K/V head, every row against every key, the mask from its definition."""
    c = s["case"]
    q = s["q"].detach()
    b, n, h, d = q.shape
    g, scale, lens = h // c["hkv"], 1 / math.sqrt(d), _lens(c)
    train = c["kind"] == "train"
    o = torch.zeros(b, n, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h, 1, n), -math.inf, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(o) if train else None
    dkv = torch.zeros(b, c["nk"], 2, c["hkv"], d, dtype=torch.float64, device="cuda") if train else None
    for i in range(b):
        length = int(lens[i])
        if "k_pages" in s:
            pages = s["table"][i].long()
            k, v = (s[name][pages].flatten(0, 1)[:length] for name in ("k_pages", "v_pages"))
        else:
            k, v = s["k"].detach()[i, :length], s["v"].detach()[i, :length]
        key = torch.arange(length, device="cuda")
        step = max(1, (1 << 27) // (g * length))
        for j in range(c["hkv"]):
            kj, vj, heads = k[:, j].double(), v[:, j].double(), slice(j * g, j * g + g)
            for r in range(0, n, step):
                pos = torch.arange(r, min(n, r + step), device="cuda")[:, None] + length - n
                hidden = (key > pos) | ((pos - key >= c["window"]) & (key >= c["sinks"]))
                rows = slice(r, min(n, r + step))
                qj = q[i, rows, heads].double().transpose(0, 1)
                x = (qj @ kj.T * scale).masked_fill(hidden, -math.inf)
                logs = torch.logsumexp(x, -1)
                p = torch.exp(x - logs[..., None]).masked_fill(hidden, 0.0)
                o[i, rows, heads] = (p @ vj).transpose(0, 1)
                lse[i, heads, 0, rows] = logs
                if train:
                    go = s["d_o"][i, rows, heads].double().transpose(0, 1)
                    dp = go @ vj.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                    dq[i, rows, heads] = (ds @ kj).transpose(0, 1)
                    dkv[i, :length, 0, j] += (ds.transpose(1, 2) @ qj).sum(0)
                    dkv[i, :length, 1, j] += (p.transpose(1, 2) @ go).sum(0)
    return (o, dq, dkv) if train else (o, lse)
