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


def test_two_streams_at_once_and_shared_pages():
    """Two servers on one GPU, each with a stream, a cache and a graph of its own, replayed side by side; inside a cache two sequences that
    share the pages of a prefix. What they leave is what each leaves alone."""
    h, hkv, d, s, width = 8, 2, 128, 6, 40

    class Server:
        def __init__(self, seed):
            gen = torch.Generator().manual_seed(seed)
            self.stream = torch.cuda.Stream()
            pool = s * width
            self.pages = [torch.randint(0, 126, (pool, 16, hkv, d), generator=gen, dtype=torch.uint8).cuda().view(torch.float8_e4m3fn) for _ in range(2)]
            self.scales = [torch.exp2(torch.randint(-12, -8, (pool, hkv), generator=gen).float()).cuda() for _ in range(2)]
            self.table = torch.randperm(pool, generator=gen).reshape(s, width).to(torch.int32).cuda()
            self.table[1, :20] = self.table[0, :20]
            self.start = torch.tensor([330, 400, 15, 600, 0, 77], dtype=torch.int32, device="cuda")
            self.x = torch.randn(s, 1, h + 2 * hkv, d, generator=gen).to(torch.bfloat16).cuda()
            self.cu = offsets([200, 1, 130, 64])
            self.q, self.kv = (torch.randn(395, n, d, generator=gen).to(torch.bfloat16).cuda() for n in (h, 2 * hkv))
            self.out = []

        def step(self):
            q, k, v = self.x.split([h, hkv, hkv], 2)
            hk.paged_kv_append_fp8(k, v, *self.pages, *self.scales, self.table, self.start)
            self.out = [*hk.paged_decode_fp8(q.contiguous(), *self.pages, *self.scales, self.table, self.start + 1),
                        *hk.attn_fwd_ragged(self.q, self.kv[:, :hkv], self.kv[:, hkv:], self.cu)]
            self.out += hk.attn_bwd_ragged(self.q, self.kv[:, :hkv], self.kv[:, hkv:], self.out[2], self.q, self.out[3], self.cu)
            self.start += 1
            self.x.neg_()

        def capture(self):
            with torch.cuda.stream(self.stream):
                self.step()
                self.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self.graph, stream=self.stream):
                    self.step()

        def state(self):
            return [t.clone() for t in (*(c.view(torch.uint8) for c in self.pages), *self.scales, *self.out)]

    def run(servers, together):
        torch.cuda.synchronize()
        for server in servers:
            server.capture()
            torch.cuda.synchronize()
        for _ in range(20):
            for server in servers:
                with torch.cuda.stream(server.stream):
                    server.graph.replay()
                if not together:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        return [server.state() for server in servers]

    alone, beside = run([Server(1), Server(2)], False), run([Server(1), Server(2)], True)
    for a, b in zip(alone, beside):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    server = Server(3)
    q = server.x[:, :, :h].contiguous()
    lens = int32([320, 400, 16, 600, 0, 77])
    got = hk.paged_decode_fp8(q, *server.pages, *server.scales, server.table, lens)
    want = kv_ref.decode(q, *server.pages, *server.scales, server.table, lens)
    assert ((got[0].cpu().double() - want[0]).abs() <= want[1]).all()
    assert _native.device_status(0) == _native.HK_OK
