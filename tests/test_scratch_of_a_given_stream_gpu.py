"""What a call with `stream=` allocates for itself goes back to that stream at once: the caller's never reads it, so the memory does not wait
until that one has passed the call."""
import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native

pytestmark = pytest.mark.gpu


def rand(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(len(shape))).to(torch.bfloat16).cuda()


def calls():
    s, h, hkv, d = 3, 8, 2, 128
    cu = torch.tensor([0, 100, 100, 333], dtype=torch.int32, device="cuda")
    q, k, v, d_o = rand(333, h, d), rand(333, hkv, d), rand(333, hkv, d), rand(333, h, d)
    o, lse = hk.attn_fwd_ragged(q, k, v, cu)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    codes = [torch.zeros(12, 16, hkv, d, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones(12, hkv, device="cuda") for _ in range(2)]
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(s, 4)
    lens = torch.tensor([40, 64, 1], dtype=torch.int32, device="cuda")
    pages = [rand(12, 16, hkv, d) for _ in range(2)]
    q1, l1 = rand(s, 1, h, d), torch.empty(s, h, 1, 1, device="cuda")
    o1 = torch.empty_like(q1)
    return {
        "attn_fwd_ragged": lambda st: hk.attn_fwd_ragged(q, k, v, cu, out=o, lse=lse, stream=st),
        "attn_bwd_ragged": lambda st: hk.attn_bwd_ragged(q, k, v, o, d_o, lse, cu, dq=grads[0], dk=grads[1], dv=grads[2], stream=st),
        "paged_decode_fp8": lambda st: hk.paged_decode_fp8(q1, *codes, *scales, table, lens, out=o1, lse=l1, stream=st),
        "paged_decode": lambda st: hk.paged_decode(q1, *pages, table, lens, out=o1, lse=l1, stream=st),
        "paged_decode_window": lambda st: hk.paged_decode(q1, *pages, table, lens, out=o1, lse=l1, stream=st, window=9, sinks=2),
    }


@pytest.mark.parametrize("name", ["attn_fwd_ragged", "attn_bwd_ragged", "paged_decode_fp8", "paged_decode", "paged_decode_window"])
def test_scratch_is_free_when_the_call_returns(name):
    call = calls()[name]
    here, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(here)
    call(side)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()  # what waits for a stream is free now
    before = torch.cuda.memory_stats()["active_bytes.all.current"]
    torch.cuda._sleep(200_000_000)  # a tenth of a second
    call(side)
    assert torch.cuda.memory_stats()["active_bytes.all.current"] == before and not here.query()
    torch.cuda.synchronize()
    assert _native.device_status(0) == _native.HK_OK


def test_scratch_of_the_weights_gradients():
    """Of a call that returns all that it makes: what stays is that."""
    q, k, d_o, d_k = rand(2, 40, 4, 128), rand(2, 40, 2, 128), rand(2, 40, 4, 128), rand(2, 40, 2, 128)
    w, angle = torch.ones(128, device="cuda"), torch.ones(40, 64, device="cuda")
    here, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(here)
    kept = hk.qk_norm_rotary_bwd(q, k, w, w, angle, angle, d_o, d_k, stream=side)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_stats()["active_bytes.all.current"]
    torch.cuda._sleep(200_000_000)
    got = hk.qk_norm_rotary_bwd(q, k, w, w, angle, angle, d_o, d_k, stream=side)
    grown = torch.cuda.memory_stats()["active_bytes.all.current"] - before
    assert not here.query() and grown == sum(-(-t.numel() * t.element_size() // 512) * 512 for t in got)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, kept))
