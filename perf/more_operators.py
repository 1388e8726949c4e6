"""Operators of an 8-bit paged cache and of ragged batches, as cases that can be timed: plain torch, or the package's own kernels.

    append   paged_kv_append_fp8: new tokens into e4m3 pages with a scale for each block of 16 tokens and head, K rotated on the way
    read     paged_kv_read_fp8: what such pages hold, as bf16 rows for the attention of a chunk
    decode   paged_decode_fp8: one new token of each sequence against them
    prompts  attn_fwd_ragged: sequences of different lengths one after the other, without padding
    train    HipRaggedAttention: the same, forward and gradients

A block's scale is the smallest power of two that brings its largest value to 448 at most, and never shrinks while the block fills up: where
a new token needs a larger one, the block's other tokens are rounded anew. Lengths come from the case alone, values, page ids and
amplitudes from the seed.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
TOP = 448.0  # the largest e4m3 value
LEAST, MOST = -120, 119  # exponents of a scale


def listed():
    return [
        # the prompts of a batch, packed, as they enter the cache behind the projection; K is rotated on the way
        dict(name="append_prompts_d128", kind="append", s=16, lo=1000, hi=4000, ragged=True, start=0, hkv=8, d=128, rot=128, table="float32", lens=1),
        # one new token of each sequence of a serving batch: a page's scale may grow, and its other tokens with it
        dict(name="append_token_d128", kind="append", s=64, lo=1, hi=1, ragged=False, start=8000, hkv=8, d=128, rot=128, table="bfloat16", lens=2),
        # chunks of an odd length behind odd positions, small heads, half of a head rotated
        dict(name="append_chunk_d64", kind="append", s=9, lo=333, hi=333, ragged=False, start=2000, hkv=4, d=64, rot=32, table="float32", lens=3),
        # what a few long conversations have cached, for the attention of a chunk
        dict(name="read_context_d128", kind="read", s=4, lo=4096, hi=8192, ragged=True, hkv=8, d=128, pow2=True, lens=4),
        # a batch with room behind each sequence, from one token on, scales of another quantiser
        dict(name="read_padded_d64", kind="read", s=33, lo=1, hi=700, ragged=False, hkv=3, d=64, pow2=False, lens=5),
        # one interactive user behind a long conversation
        dict(name="decode_single_d128", kind="decode", s=1, lo=12000, hi=12500, h=32, hkv=8, d=128, window=0, sinks=0, pow2=True, lens=2),
        # a full serving batch
        dict(name="decode_batch64_d128", kind="decode", s=64, lo=512, hi=8192, h=64, hkv=8, d=128, window=0, sinks=0, pow2=True, lens=1),
        # a window layer: small heads, six to a group, contexts from one token on, scales of another quantiser
        dict(name="decode_window_d64", kind="decode", s=33, lo=1, hi=4096, h=48, hkv=8, d=64, window=500, sinks=20, pow2=False, lens=5),
        # two long prompts, eight heads to a group
        dict(name="prompts_long_d128", kind="prompts", s=2, lo=7000, hi=10000, more=0, h=16, hkv=2, d=128, causal=True, lens=1),
        # short chunks of many sequences, each behind its own cached keys
        dict(name="prompts_cached_d64", kind="prompts", s=17, lo=20, hi=600, more=1500, h=12, hkv=4, d=64, causal=True, lens=2),
        # one pre-training step of a layer on packed documents
        dict(name="train_documents_d128", kind="train", s=10, lo=400, hi=3000, more=0, h=32, hkv=8, d=128, causal=True, lens=3),
        # fine-tuning on short samples, where launches and host work count
        dict(name="train_samples_d64", kind="train", s=23, lo=1, hi=400, more=0, h=8, hkv=2, d=64, causal=True, lens=4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    flops, nbytes, cells = max(w["flops"] for w in most), max(w["bytes"] for w in most), max(_cells(c) for c in listed())
    while True:
        kind = rng.choice(["append", "append", "read", "decode", "decode", "prompts", "train"])
        hkv, g = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 5, 6, 7, 8])
        c = dict(kind=kind, s=_log_int(rng, 1, 64), hkv=hkv, d=rng.choice([64, 128]), lens=rng.randint(0, 999), lo=_log_int(rng, 1, 4096))
        c["hi"] = c["lo"] + _log_int(rng, 1, 8192)
        if kind in ("append", "read"):
            c["ragged"] = rng.random() < 0.5
        if kind == "append":
            if not c["ragged"]:
                c["lo"] = c["hi"] = 1 if rng.random() < 0.3 else c["lo"]
            c |= dict(start=rng.choice([0, _log_int(rng, 1, 9000)]), table=rng.choice(["float32", "bfloat16"]))
            c["rot"] = rng.choice([0, 16 * rng.randint(1, c["d"] // 16), c["d"]])
        elif kind in ("read", "decode"):
            c["pow2"] = rng.random() < 0.5
        if kind == "decode":
            c |= dict(h=hkv * g, window=rng.choice([0, _log_int(rng, 1, 4096)]))
            c["sinks"] = rng.choice([0, rng.randint(1, 200)]) if c["window"] else 0
        if kind in ("prompts", "train"):
            c |= dict(h=hkv * g, more=rng.choice([0, 0, _log_int(rng, 1, 4096)]), causal=rng.random() < 0.8)
        w = work(c)
        if w["flops"] <= flops and w["bytes"] <= nbytes and _cells(c) <= cells:
            return c


def _lens(c):
    """New tokens, cached tokens or queries of each sequence."""
    r = np.random.RandomState(c["lens"])
    lens = np.exp(r.uniform(math.log(c["lo"]), math.log(c["hi"] + 1), c["s"])).astype(np.int64).clip(c["lo"], c["hi"])
    return np.full(c["s"], lens[0]) if c["kind"] == "append" and not c["ragged"] else lens


def _before(c):
    """Tokens in front of an append, or of a ragged batch's queries."""
    most = c["start"] if c["kind"] == "append" else c["more"]
    return np.random.RandomState(c["lens"] + 1000).randint(0, most + 1, c["s"]) if most else np.zeros(c["s"], np.int64)


def _cells(c):
    """Values that the plain form holds at a time."""
    if c["kind"] in ("prompts", "train"):
        n = _lens(c)
        return c["s"] * c["h"] * int(n.max()) * int((n + _before(c)).max())
    return c["s"] * (int(_lens(c).max()) + PAGE) * c["hkv"] * c["d"]


def _seen(c, n, nk):
    """(query, key) pairs that a sequence of n queries at the end of nk keys has."""
    return n * nk - n * (n - 1) // 2 if c["causal"] else n * nk


def work(c):
    lens, d = _lens(c), c["d"]
    tokens = int(lens.sum())
    token, scale = c["hkv"] * d, 8 * c["hkv"]  # values of one token's K, bytes of a block's two scales
    if c["kind"] == "append":
        blocks = int(((_before(c) + lens + PAGE - 1) // PAGE - _before(c) // PAGE).sum())
        table = c["rot"] * min(tokens, int((_before(c) + lens).max())) * (4 if c["table"] == "float32" else 2)
        return {"bytes": tokens * token * 6 + blocks * scale + table, "flops": tokens * token * 10}
    if c["kind"] == "read":
        rows = tokens if c["ragged"] else c["s"] * int(lens.max())
        return {"bytes": tokens * token * 2 + rows * token * 4 + -(-tokens // PAGE) * scale, "flops": tokens * token * 4}
    if c["kind"] == "decode":
        seen = lens if not c["window"] else np.minimum(lens, c["window"]) + np.clip(lens - c["window"], 0, c["sinks"])
        keys = int(seen.sum())
        return {"bytes": keys * token * 2 + -(-keys // PAGE) * scale + 4 * c["s"] * c["h"] * d, "flops": 4 * d * c["h"] * keys}
    more = _before(c)
    keys = int((lens + more).sum())
    pairs = sum(_seen(c, int(n), int(n + m)) for n, m in zip(lens, more))
    q, kv = 2 * tokens * c["h"] * d, 4 * keys * token
    if c["kind"] == "train":  # O, dQ and dO beside Q, dK and dV beside K and V
        return {"bytes": 4 * q + 2 * kv, "flops": 14 * d * c["h"] * pairs}
    return {"bytes": 2 * q + kv + 4 * tokens * c["h"], "flops": 4 * d * c["h"] * pairs}


# ---------------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)


def _scale_for(amax):
    """The smallest power of two that brings amax to 448 at most, NaN for NaN."""
    m, e = torch.frexp(amax / TOP)
    e = torch.where(m == 0.5, e - 1, e).clamp(LEAST, MOST)
    e = torch.where(amax == math.inf, MOST, torch.where(amax == 0, LEAST, e))
    return torch.where(amax.isnan(), math.nan, torch.ldexp(torch.ones_like(amax), e))


def _cache(gen, pool, c):
    """Pages as a cache holds them: another amplitude for each page and head."""
    pages, scales = [], []
    for _ in range(2):
        x = torch.randn(pool, PAGE, c["hkv"], c["d"], generator=gen, device="cuda")
        x *= torch.exp2(torch.randn(pool, 1, c["hkv"], 1, generator=gen, device="cuda"))
        amax = x.abs().amax((1, 3))
        scales.append(_scale_for(amax) if c.get("pow2", True) else amax / TOP)
        pages.append((x / scales[-1][:, None, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn))
    return pages, scales


def _cu(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    s, hkv, d, lens = c["s"], c["hkv"], c["d"], _lens(c)
    st = {"case": c}
    if c["kind"] in ("append", "read", "decode"):
        ends = lens + _before(c) if c["kind"] == "append" else lens
        width = -(-int(ends.max()) // PAGE)
        pool = s * width + 5
        (st["k_pages"], st["v_pages"]), (st["k_scales"], st["v_scales"]) = _cache(gen, pool, c)
        order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
        st["table"] = order[:s * width].reshape(s, width).contiguous()
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if c["kind"] == "read":
            st["cu"] = _cu(lens) if c["ragged"] else None
            st["rows"] = int(lens.sum()) if c["ragged"] else int(lens.max())
        if c["kind"] == "decode":
            st["q"] = _randn(gen, s, 1, c["h"], d)
        if c["kind"] == "append":
            shape = (int(lens.sum()),) if c["ragged"] else (s, int(lens[0]))
            kv = _randn(gen, *shape, 2 * hkv, d)  # K and V of a packed projection
            kv *= torch.exp2(torch.randn(*shape, 1, 1, generator=gen, device="cuda"))
            st["k"], st["v"] = kv[..., :hkv, :], kv[..., hkv:, :]
            st["start"] = torch.tensor(_before(c), dtype=torch.int32, device="cuda")
            st["cu"] = _cu(lens) if c["ragged"] else None
            st["cos"] = st["sin"] = None
            if c["rot"]:
                at = torch.arange(int(ends.max()), device="cuda", dtype=torch.float64)[:, None]
                angle = at / 500000.0 ** (torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
                st["cos"], st["sin"] = (f(angle).to(getattr(torch, c["table"])) for f in (torch.cos, torch.sin))
        return st
    nk = lens + _before(c)
    st["cu_q"], st["cu_k"] = _cu(lens), _cu(nk) if c["more"] else None
    q_rows, k_rows = int(lens.sum()), int(nk.sum())
    if c["kind"] == "prompts" and not c["more"]:  # views of one packed projection
        qkv = _randn(gen, q_rows, c["h"] + 2 * hkv, d)
        st["q"], st["k"], st["v"] = qkv[:, :c["h"]], qkv[:, c["h"]:c["h"] + hkv], qkv[:, c["h"] + hkv:]
    else:
        st["q"], st["kv"] = _randn(gen, q_rows, c["h"], d), _randn(gen, k_rows, 2, hkv, d)
        st["k"], st["v"] = st["kv"].unbind(1)
    if c["kind"] == "train":
        st["d_o"] = _randn(gen, q_rows, c["h"], d)
        st["q"], st["kv"] = st["q"].requires_grad_(), st["kv"].requires_grad_()
    return st


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode}.get(state["case"]["kind"], _plain_ragged)(state)


def _run_own(s):
    import hipkittens_b200 as hk

    c = s["case"]
    if c["kind"] in ("append", "read", "decode"):
        cache = (s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"])
    if c["kind"] == "append":
        hk.paged_kv_append_fp8(s["k"], s["v"], *cache, s["start"], cos=s["cos"], sin=s["sin"], cu_seqlens=s["cu"])
        return cache[:4]
    if c["kind"] == "read":
        return hk.paged_kv_read_fp8(*cache, s["rows"], ctx_lens=None if c["ragged"] else s["lens"], cu_seqlens=s["cu"])
    if c["kind"] == "decode":
        return hk.paged_decode_fp8(s["q"], *cache, s["lens"], window=c["window"] or None, sinks=c["sinks"])
    if c["kind"] == "prompts":
        return hk.attn_fwd_ragged(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=c["causal"])
    if "module" not in s:  # which a program makes once
        from hipkittens_b200.attention import HipRaggedAttention

        s["module"] = HipRaggedAttention(causal=c["causal"])
    o = s["module"](s["q"], s["kv"], s["cu_q"], s["cu_k"])
    return (o.detach(), *torch.autograd.grad(o, (s["q"], s["kv"]), s["d_o"]))


def _plain_append(s):
    """Block by block: the rows of every block that gets a token, new ones from the input and the others as they stand."""
    c = s["case"]
    start, lens, table = s["start"].long(), s["lens"].long(), s["table"].long()
    blocks = -(-int(_lens(c).max()) // PAGE) + 1
    slot = start[:, None] // PAGE + torch.arange(blocks, device="cuda")
    at = slot[:, :, None] * PAGE + torch.arange(PAGE, device="cuda") - start[:, None, None]  # the new token that a row gets
    new = (at >= 0) & (at < lens[:, None, None])
    which, block = new.any(2).nonzero(as_tuple=True)
    new, at = new[which, block], at[which, block].clamp(min=0)
    at = torch.minimum(at, lens[which, None] - 1)
    page = table[which, slot[which, block]]
    row = at + (s["cu"].long()[which, None] if c["ragged"] else which[:, None] * int(_lens(c)[0]))
    again = ~new[:, 0]  # a block that has tokens already

    def one(x, pages, scales, rotated):
        x = x.reshape(-1, c["hkv"], c["d"])[row].float()
        if rotated and c["rot"]:
            half = c["rot"] // 2
            cos, sin = (t.float()[at + start[which, None]][:, :, None] for t in (s["cos"], s["sin"]))
            a, b = x[..., :half], x[..., half:c["rot"]]
            x = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., c["rot"]:]], -1)
        codes, before = pages[page].float(), scales[page]
        need = _scale_for(torch.where(new[:, :, None, None], x.abs(), 0.0).amax((1, 3)))
        scale = torch.where(again[:, None], torch.maximum(before, need), need)
        kept = torch.where(again[:, None, None, None], codes * before[:, None, :, None] / scale[:, None, :, None], codes)
        x = torch.where(new[:, :, None, None], x / scale[:, None, :, None], kept)
        pages[page] = x.clamp(-TOP, TOP).to(torch.float8_e4m3fn)
        scales[page] = scale
        return pages, scales

    (k, ks), (v, vs) = one(s["k"], s["k_pages"], s["k_scales"], True), one(s["v"], s["v_pages"], s["v_scales"], False)
    return k, v, ks, vs


def _plain_read(s):
    c, lens = s["case"], s["lens"].long()
    rows = torch.arange(s["rows"], device="cuda")
    if c["ragged"]:
        which = torch.searchsorted(s["cu"].long()[1:], rows, right=True)
        at, there = rows - s["cu"].long()[which], None
    else:
        which, at = torch.arange(c["s"], device="cuda")[:, None], rows[None, :]
        there = (at < lens[:, None])[:, :, None, None]
        at = torch.minimum(at, lens[:, None] - 1)
    page = s["table"].long()[which, at // PAGE]

    def one(pages, scales):
        x = pages[page, at % PAGE].float() * scales[page][..., None]
        return (x if there is None else torch.where(there, x, 0.0)).to(torch.bfloat16)

    return one(s["k_pages"], s["k_scales"]), one(s["v_pages"], s["v_scales"])


def _plain_decode(s):
    c, lens, page = s["case"], s["lens"].long(), s["table"].long()
    b, h, d, hkv = c["s"], c["h"], c["d"], c["hkv"]
    k, v = ((s[n + "_pages"][page].float() * s[n + "_scales"][page][:, :, None, :, None]).flatten(1, 2) for n in "kv")
    key = torch.arange(k.shape[1], device="cuda")
    seen = key < lens[:, None]
    if c["window"]:
        seen &= (key >= lens[:, None] - c["window"]) | (key < c["sinks"])
    score = torch.einsum("bhgd,bkhd->bhgk", s["q"].float().reshape(b, hkv, h // hkv, d), k) / math.sqrt(d)
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgk,bkhd->bhgd", p / total, v)
    return o.reshape(b, 1, h, d).to(torch.bfloat16), (top + torch.log(total)).reshape(b, h, 1, 1)


def _plain_ragged(s):
    """The sequences side by side, padded to the longest, and their rows taken back out."""
    c = s["case"]
    b, h, hkv, d = c["s"], c["h"], c["hkv"], c["d"]
    cu_q, cu_k = s["cu_q"].long(), (s["cu_q"] if s["cu_k"] is None else s["cu_k"]).long()
    nq, nk = cu_q.diff(), cu_k.diff()
    i, j = torch.arange(int(_lens(c).max()), device="cuda"), torch.arange(int((_lens(c) + _before(c)).max()), device="cuda")
    q_there, k_there = i < nq[:, None], j < nk[:, None]
    q_row, k_row = (cu_q[:-1, None] + i)[q_there], (cu_k[:-1, None] + j)[k_there]

    def padded(x, there):
        out = torch.zeros(*there.shape, *x.shape[1:], device="cuda")
        out[there] = x.detach().float()
        return out

    q = padded(s["q"][q_row], q_there).reshape(b, -1, hkv, h // hkv, d)
    k, v = padded(s["k"][k_row], k_there), padded(s["v"][k_row], k_there)
    seen = q_there[:, :, None] & k_there[:, None, :]
    if c["causal"]:
        seen &= j <= i[:, None] + (nk - nq)[:, None, None]
    scale = 1 / math.sqrt(d)
    p = torch.einsum("bqhgd,bkhd->bhgqk", q, k) * scale
    p = torch.where(seen[:, None, None], p, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(p - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total))[..., 0].permute(1, 2, 0, 3).reshape(h, b, -1)[:, q_there]
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.einsum("bhgqk,bkhd->bqhgd", p, v)
    out = o.reshape(b, -1, h, d)[q_there].to(torch.bfloat16)
    if c["kind"] == "prompts":
        return out, lse.contiguous()
    g = padded(s["d_o"], q_there).reshape(q.shape)
    dv = torch.einsum("bhgqk,bqhgd->bkhd", p, g)
    ds = torch.einsum("bqhgd,bkhd->bhgqk", g, v)
    ds = p * (ds - (g * o).sum(-1).permute(0, 2, 3, 1)[..., None]) * scale
    dq = torch.einsum("bhgqk,bkhd->bqhgd", ds, k).reshape(b, -1, h, d)[q_there]
    dk = torch.einsum("bhgqk,bqhgd->bkhd", ds, q)
    return out, dq.to(torch.bfloat16), torch.stack([dk, dv], 2)[k_there].to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "decode": _exact_decode}.get(case["kind"], _exact_ragged)(s)


def _e4m3(x):
    """The nearest e4m3 value, the even one of two: steps of an eighth of a value's own power of two, of 2^-9 below 2^-6."""
    power = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30)))
    power = torch.where(x.abs() < torch.exp2(power), power - 1, power).clamp(min=-6)
    step = torch.exp2(power - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def _exact_append(s):
    """Sequence by sequence: its tokens in front of the blocks' new rows, every block's maximum over powers of two in turn."""
    c, lens, before = s["case"], _lens(s["case"]), _before(s["case"])
    out = [s["k_pages"].double(), s["v_pages"].double(), s["k_scales"].double(), s["v_scales"].double()]
    powers = torch.exp2(torch.arange(LEAST, MOST + 1, device="cuda", dtype=torch.float64))
    offset = np.concatenate([[0], np.cumsum(lens)])
    for i in range(c["s"]):
        n, start = int(lens[i]), int(before[i])
        front, blocks = start % PAGE, -(-(start % PAGE + n) // PAGE)
        pages = s["table"][i, start // PAGE:start // PAGE + blocks].long()
        for x, pool, scales, rotated in ((s["k"], out[0], out[2], True), (s["v"], out[1], out[3], False)):
            x = (x[offset[i]:offset[i + 1]] if c["ragged"] else x[i]).double()
            if rotated and c["rot"]:
                half = c["rot"] // 2
                turn = torch.complex(s["cos"][start:start + n].double(), s["sin"][start:start + n].double())[:, None]
                z = torch.complex(x[..., :half].contiguous(), x[..., half:c["rot"]].contiguous()) * turn
                x = torch.cat([z.real, z.imag, x[..., c["rot"]:]], -1)
            rows = torch.zeros(blocks * PAGE, *x.shape[1:], dtype=torch.float64, device="cuda")
            rows[front:front + n] = x
            rows = rows.unflatten(0, (blocks, PAGE))
            need = powers[torch.searchsorted(powers * TOP, rows.abs().amax((1, 3))).clamp(max=powers.numel() - 1)]
            kept = pool[pages]
            if front:
                need[0] = torch.maximum(need[0], scales[pages[0]])
                kept[0] = _e4m3(kept[0] * (scales[pages[0]] / need[0])[None, :, None])
            rows = _e4m3(rows / need[:, None, :, None])
            fresh = torch.zeros(blocks * PAGE, dtype=torch.bool, device="cuda")
            fresh[front:front + n] = True
            pool[pages] = torch.where(fresh.reshape(blocks, PAGE, 1, 1), rows, kept)
            scales[pages] = need
    return tuple(out)


def _rows_of(s, i, n):
    """The first n cached tokens of sequence i, K and V."""
    pages = s["table"][i, :-(-n // PAGE)].long()
    return tuple((s[x + "_pages"][pages].double() * s[x + "_scales"][pages].double()[:, None, :, None]).flatten(0, 1)[:n] for x in "kv")


def _exact_read(s):
    c, lens = s["case"], _lens(s["case"])
    found = [_rows_of(s, i, int(lens[i])) for i in range(c["s"])]
    if c["ragged"]:
        return tuple(torch.cat([f[k] for f in found]) for k in (0, 1))
    return tuple(torch.nn.utils.rnn.pad_sequence([f[k] for f in found], batch_first=True) for k in (0, 1))


def _attend(q, k, v, hidden):
    """One sequence: q [n,h,d], k and v [m,hkv,d], hidden [n,m] -> O, L [h,n] and the probabilities, in 64 bits."""
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    x = (q.transpose(0, 1) @ k.permute(1, 2, 0) / math.sqrt(q.shape[2])).masked_fill(hidden, -math.inf)
    logs = torch.logsumexp(x, -1)
    p = torch.exp(x - logs[..., None]).masked_fill(hidden, 0.0)
    return (p @ v.transpose(0, 1)).transpose(0, 1), logs, p, k, v


def _exact_decode(s):
    c, lens = s["case"], _lens(s["case"])
    o, l = [], []
    for i in range(c["s"]):
        n = int(lens[i])
        key = torch.arange(n, device="cuda")
        hidden = ((n - 1 - key >= c["window"]) & (key >= c["sinks"]) if c["window"] else key < 0)[None]
        one = _attend(s["q"][i].double(), *_rows_of(s, i, n), hidden)
        o.append(one[0])
        l.append(one[1][..., None])
    return torch.stack(o), torch.stack(l)


def _exact_ragged(s):
    c, lens, more = s["case"], _lens(s["case"]), _before(s["case"])
    h, hkv, d = c["h"], c["hkv"], c["d"]
    outs = []
    q0 = k0 = 0
    for n, m in zip(map(int, lens), map(int, lens + more)):
        q, k, v = s["q"].detach()[q0:q0 + n].double(), s["k"].detach()[k0:k0 + m].double(), s["v"].detach()[k0:k0 + m].double()
        d_o = s["d_o"][q0:q0 + n].double() if c["kind"] == "train" else None
        o, logs, dq = torch.zeros_like(q), torch.zeros(h, n, dtype=torch.float64, device="cuda"), torch.zeros_like(q)
        dk, dv = torch.zeros_like(k), torch.zeros_like(v)
        g, step = h // hkv, max(1, (1 << 28) // (h * m))
        for r in range(0, n, step):
            rows = slice(r, min(n, r + step))
            pos = torch.arange(n, device="cuda")[rows, None] + m - n
            hidden = torch.arange(m, device="cuda") > (pos if c["causal"] else m)
            o[rows], logs[:, rows], p, kr, vr = _attend(q[rows], k, v, hidden)
            if d_o is not None:
                go = d_o[rows].transpose(0, 1)
                dp = go @ vr.permute(1, 2, 0)
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[rows] = (ds @ kr.transpose(0, 1)).transpose(0, 1)
                dk += (ds.transpose(1, 2) @ q[rows].transpose(0, 1)).transpose(0, 1).unflatten(1, (hkv, g)).sum(2)
                dv += (p.transpose(1, 2) @ go).transpose(0, 1).unflatten(1, (hkv, g)).sum(2)
        outs.append((o, dq, torch.stack([dk, dv], 1)) if d_o is not None else (o, logs))
        q0, k0 = q0 + n, k0 + m
    if c["kind"] == "train":
        return tuple(torch.cat([x[i] for x in outs]) for i in range(3))
    return torch.cat([x[0] for x in outs]), torch.cat([x[1] for x in outs], 1)
