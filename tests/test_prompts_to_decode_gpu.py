"""Prompts, a second message and new tokens of a few conversations, as a server runs them over a cache in 8 bits: attention over the ragged
prompts, their K and V into pages, the next messages' behind them, what is cached back as bf16 for the messages' attention, and then a
token at a time: append and decode, in a graph that is replayed. Each step is checked against the definition in 64 bits of what it was given."""
import pytest
import torch

import hipkittens_b200 as hk
import kv_fp8_reference as kv_ref
import ragged_reference as ref
from hipkittens_b200 import _native

pytestmark = pytest.mark.gpu


def int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def offsets(lens):
    return int32([sum(lens[:i]) for i in range(len(lens) + 1)])


@pytest.mark.parametrize("h,hkv,d,dtype", [(8, 2, 128, torch.float32), (6, 1, 64, torch.bfloat16)])
def test_conversations(h, hkv, d, dtype):
    assert torch.cuda.is_available(), "this test needs a B200"
    gen = torch.Generator().manual_seed(h)
    prompts, messages, new = [37, 300, 1, 129], [20, 1, 150, 16], 5
    s, width = len(prompts), 32
    pool = s * width + 1
    table = torch.randperm(pool, generator=gen)[:s * width].reshape(s, width).to(torch.int32).cuda()
    pages = [torch.zeros(pool, 16, hkv, d, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pool, hkv, device="cuda") for _ in range(2)]
    angle = torch.arange(512)[:, None] / 1000.0 ** (torch.arange(0, d, 2) / d)
    turn = dict(cos=angle.cos().to(dtype).cuda(), sin=angle.sin().to(dtype).cuda())

    def tokens(*shape):
        x = torch.randn(*shape, h + 2 * hkv, d, generator=gen).to(torch.bfloat16).cuda()
        return x[..., :h, :], x[..., h:h + hkv, :], x[..., h + hkv:, :]

    def cached(i, n):
        """Two definitions of the first n tokens of a conversation: [n, H_KV, D] in 64 bits, from the pages."""
        return [kv_ref.tokens(c.cpu().double(), t.cpu().double(), table[i].cpu(), n) for c, t in zip(pages, scales)]

    # the prompts: attention, and their tokens into the cache
    q, k, v = tokens(sum(prompts))
    cu = offsets(prompts)
    o, l = hk.attn_fwd_ragged(q, k, v, cu)
    for got, pair, what in zip((o, l), ref.attention(q, k, v, cu, cu), ("O", "L")):
        ref.close(got, pair, what)
    hk.paged_kv_append_fp8(k, v, *pages, *scales, table, int32([0] * s), cu_seqlens=cu, **turn)
    lens = list(prompts)
    given = [(k[a:a + n], v[a:a + n]) for a, n in zip(cu.tolist(), prompts)]

    # the next messages, over all that is cached
    q, k, v = tokens(sum(messages))
    cu = offsets(messages)
    hk.paged_kv_append_fp8(k, v, *pages, *scales, table, int32(lens), cu_seqlens=cu, **turn)
    lens = [a + b for a, b in zip(lens, messages)]
    given = [(torch.cat([gk, k[a:a + n]]), torch.cat([gv, v[a:a + n]])) for (gk, gv), a, n in zip(given, cu.tolist(), messages)]
    cu_k = offsets(lens)
    k_all, v_all = hk.paged_kv_read_fp8(*pages, *scales, table, cu_seqlens=cu_k, rows=sum(lens))
    for i, (gk, gv) in enumerate(given):
        rows = slice(int(cu_k[i]), int(cu_k[i + 1]))
        want_k, want_v = cached(i, lens[i])
        # products with powers of two: bf16 holds them
        assert torch.equal(k_all[rows].cpu().double(), want_k) and torch.equal(v_all[rows].cpu().double(), want_v)
        # two roundings to e4m3 of what was given, where a block's scale has grown, and steps of 2^-10 of its largest below 2^-14 of that
        turned, _ = kv_ref.rotate(gk.cpu(), 0, turn["cos"].cpu(), turn["sin"].cpu())
        for got, want in ((want_k, turned), (want_v, gv.cpu().double())):
            assert ((got - want).abs() <= want.abs() * (2 * 2 ** -4 + 2 ** -8 + 2 ** -20) + 2 ** -13).all()
    o, l = hk.attn_fwd_ragged(q, k_all, v_all, cu, cu_k)
    for got, pair, what in zip((o, l), ref.attention(q, k_all, v_all, cu, cu_k), ("O", "L")):
        ref.close(got, pair, what)

    # a token at a time: set up outside the capture, then the same two calls in a graph
    q1, k1, v1 = (x.contiguous() for x in tokens(s, 1))
    start, length = int32(lens), int32([n + 1 for n in lens])
    out = torch.empty(s, 1, h, d, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(s, h, 1, 1, device="cuda")

    def step():
        hk.paged_kv_append_fp8(k1, v1, *pages, *scales, table, start, **turn)
        hk.paged_decode_fp8(q1, *pages, *scales, table, length, out=out, lse=lse)

    def check():
        want = kv_ref.decode(q1, *pages, *scales, table, length)
        assert ((out.cpu().double() - want[0]).abs() <= want[1]).all() and ((lse.cpu().double() - want[2]).abs() <= want[3]).all()

    step()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(new):
        for x, y in zip((q1, k1, v1), tokens(s, 1)):
            x.copy_(y)
        start += 1
        length += 1
        graph.replay()
        check()
    assert _native.device_status(0) == _native.HK_OK
