"""What a call with `stream=` allocates is memory of that stream: a block that another stream gave back may still be read by work
that waits there, and the kernel would write over it."""
import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native

pytestmark = pytest.mark.gpu


def stream_of_memory(t):
    for segment in torch.cuda.memory_snapshot():
        if segment["address"] <= t.data_ptr() < segment["address"] + segment["total_size"]:
            return segment["stream"]
    raise AssertionError("not memory of torch's allocator")


def rand(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(len(shape))).to(torch.bfloat16).cuda()


def calls():
    q, k, v, d_o = rand(2, 40, 4, 128), rand(2, 40, 2, 128), rand(2, 40, 2, 128), rand(2, 40, 4, 128)
    lse, delta = (torch.zeros(2, 4, 1, 40, device="cuda") for _ in range(2))
    kp, vp = rand(8, 16, 2, 128), rand(8, 16, 2, 128)
    paged = (kp, vp, torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), torch.tensor([40, 50], dtype=torch.int32, device="cuda"))
    angle = torch.ones(40, 64, device="cuda")
    table = angle.to(torch.bfloat16)
    w = torch.ones(128, device="cuda")
    window = dict(causal=True, window=9, sinks=2)
    return {
        "attn_fwd": lambda s: hk.attn_fwd(q, k, v, stream=s),
        "attn_fwd_window": lambda s: hk.attn_fwd(q, k, v, stream=s, **window),
        "attn_fwd_paged": lambda s: hk.attn_fwd_paged(q, *paged, stream=s),
        "attn_fwd_paged_window": lambda s: hk.attn_fwd_paged(q, *paged, stream=s, **window),
        "paged_decode": lambda s: hk.paged_decode(q[:, :1].contiguous(), *paged, stream=s),
        "paged_decode_window": lambda s: hk.paged_decode(q[:, :1].contiguous(), *paged, stream=s, window=9, sinks=2),
        "attn_bwd_prep": lambda s: [hk.attn_bwd_prep(q, d_o, stream=s)],
        "attn_bwd": lambda s: hk.attn_bwd(q, k, v, d_o, lse, delta, stream=s),
        "dq_shuffle": lambda s: [_native.dq_shuffle(q, stream=s)],
        "rotary": lambda s: [hk.rotary(q, table[:4], table[:4], stream=s)],
        "rotary_bnhd": lambda s: [hk.rotary_bnhd(q, table, table, stream=s)],
        "qk_norm_rotary": lambda s: hk.qk_norm_rotary(q, k, w, w, angle, angle, stream=s),
        "qk_norm_rotary_bwd": lambda s: hk.qk_norm_rotary_bwd(q, k, w, w, angle, angle, d_o, k, stream=s),
    }


@pytest.mark.parametrize("name", ["attn_fwd", "attn_fwd_window", "attn_fwd_paged", "attn_fwd_paged_window", "paged_decode",
                                  "paged_decode_window", "attn_bwd_prep", "attn_bwd", "dq_shuffle", "rotary", "rotary_bnhd",
                                  "qk_norm_rotary", "qk_norm_rotary_bwd"])
def test_outputs_lie_in_memory_of_the_stream(name):
    call = calls()[name]
    want = call(None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = call(side)
    torch.cuda.synchronize()
    assert all(stream_of_memory(t) == side.cuda_stream for t in got)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert _native.device_status(0) == 0


@pytest.mark.parametrize("name", ["attn_fwd_window", "paged_decode", "qk_norm_rotary_bwd"])
def test_what_the_caller_s_stream_still_reads_is_not_given_away(name):
    call = calls()[name]
    want = call(None)
    here, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(here)
    got = call(side)
    here.wait_stream(side)
    torch.cuda._sleep(200_000_000)  # a tenth of a second
    read = [t.clone() for t in got]
    places, shapes = [t.data_ptr() for t in got], [(t.shape, t.dtype) for t in got]
    del got
    with torch.cuda.stream(side):
        others = [torch.empty(shape, dtype=dtype, device="cuda").zero_() for shape, dtype in shapes]
    assert not here.query() and not set(places) & {t.data_ptr() for t in others}
    assert all(torch.equal(x, y) for x, y in zip(read, want))
