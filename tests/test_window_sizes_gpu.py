"""Window attention where offsets pass 32 bits: strides, whole tensors, pools of pages."""
import pytest
import torch
import window_reference as ref

import hipkittens_b200 as hk
from hipkittens_b200 import _native

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    yield
    torch.cuda.empty_cache()


def rand(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("window,sinks", [(5, 1), (50, 3)])  # delta of all rows from their keys, of the first ones only
@pytest.mark.parametrize("d,strides", [(64, ((1 << 31) + 8, 512, 64)), (128, (512, (1 << 24) + 256, 128)),
                                       (64, (25600, 128, (1 << 30) + 8))])
def test_strides(d, strides, window, sinks):
    """Batch, sequence and head strides of q, k, v and of the gradients. Bit by bit what dense tensors give."""
    b, n, h = 2, 200, 3
    gen = torch.Generator().manual_seed(d)
    dense, d_o = [rand(gen, b, n, h, d) for _ in range(3)], rand(gen, b, n, h, d)
    size = sum((x - 1) * s for x, s in zip((b, n, h), strides)) + d
    shared = torch.empty(size, dtype=torch.bfloat16, device="cuda")  # one after the other: 3 of them at a time would be 40 GB
    want_o = hk.attn_fwd(*dense, causal=True, window=window, sinks=sinks)
    want = [torch.empty_like(t) for t in dense]
    _native.attn_bwd_strided(*dense, want_o[0], d_o, want_o[1], *want, causal=True, window=window, sinks=sinks)
    far = shared.as_strided((b, n, h, d), (*strides, 1))
    for i in range(3):
        far.copy_(dense[i])
        args = [far if j == i else t for j, t in enumerate(dense)]
        got_o = hk.attn_fwd(*args, causal=True, window=window, sinks=sinks)
        got = [torch.empty_like(t) for t in dense]
        _native.attn_bwd_strided(*args, got_o[0], d_o, got_o[1], *got, causal=True, window=window, sinks=sinks)
        assert all(torch.equal(x, y) for x, y in zip((*want_o, *want), (*got_o, *got)))
        got = [far if j == i else torch.empty_like(t) for j, t in enumerate(dense)]
        far.zero_()
        _native.attn_bwd_strided(*dense, got_o[0], d_o, got_o[1], *got, causal=True, window=window, sinks=sinks)
        assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert _native.device_status(0) == 0


@pytest.mark.parametrize("n,h,hkv,d,window", [(270080, 64, 8, 128, 70), (270080, 128, 8, 64, 20)])
def test_elements(n, h, hkv, d, window):
    """More than 2^31 values in q. The ends of the sequence are compared: keys behind the window of a row change nothing in it."""
    torch.manual_seed(1)
    q, d_o = (torch.empty(1, n, h, d, dtype=torch.bfloat16, device="cuda").normal_() for _ in range(2))
    k, v = (torch.empty(1, n, hkv, d, dtype=torch.bfloat16, device="cuda").normal_() for _ in range(2))
    o, lse = hk.attn_fwd(q, k, v, causal=True, window=window)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    _native.attn_bwd_strided(q, k, v, o, d_o, lse, *grads, causal=True, window=window)
    assert _native.device_status(0) == 0
    g, rows = h // hkv, 150
    heads, kv = slice(h - g, h), slice(hkv - 1, hkv)
    for first in (0, n - rows):
        keys = max(first - window, 0)  # the first that a row sees, or one before it
        behind = min(first + rows, n)
        part = q[:, first:behind, heads], k[:, keys:behind, kv], v[:, keys:behind, kv]
        want = ref.forward(*part, window, 0)
        ref.close(o[:, first:behind, heads], want[0], want[1], "O")
        ref.close(lse[:, heads, :, first:behind], want[2], want[3], "L")
        at = slice(first, behind - window + 1) if first == 0 else slice(first, behind)  # keys that no row outside sees
        for name, got, (r, bound) in zip(("dQ", "dK", "dV"), grads, ref.backward(*part, d_o[:, first:behind, heads], window, 0)):
            if name == "dQ":
                ref.close(got[:, first:behind, heads], r, bound, name)
            else:
                inside = slice(at.start - keys, at.stop - keys)
                ref.close(got[:, at, kv], r[:, inside], bound[:, inside], name)


@pytest.mark.parametrize("d", [64, 128])
def test_pools_of_pages(d):
    hkv, h, pool = 8, 16, 1 + (1 << 31) // (16 * 8 * d) + 40
    gen = torch.Generator().manual_seed(d)
    kp, vp = (torch.zeros(pool, 16, hkv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = (pool - 1 - torch.arange(24).view(2, 12)).to(torch.int32)
    table[:, 0] = torch.tensor([0, 1])
    table = table.cuda()
    k, v, q = rand(gen, 2, 190, hkv, d), rand(gen, 2, 190, hkv, d), rand(gen, 2, 190, h, d)
    hk.paged_kv_append(k, v, kp, vp, table, torch.zeros(2, dtype=torch.int32, device="cuda"))
    lens = torch.tensor([190, 190], dtype=torch.int32, device="cuda")
    for window, sinks in ((60, 4), (9, 0)):
        want = ref.forward(q, k, v, window, sinks)
        o, lse = hk.paged_decode(q[:, -1:].contiguous(), kp, vp, table, lens, window=window, sinks=sinks)
        ref.close(o, want[0][:, -1:], want[1][:, -1:], "O")
        ref.close(lse, want[2][..., -1:], want[3][..., -1:], "L")
        o, lse = hk.attn_fwd_paged(q[:, -70:].contiguous(), kp, vp, table, lens, window=window, sinks=sinks)
        ref.close(o, want[0][:, -70:], want[1][:, -70:], "O")
        ref.close(lse, want[2][..., -70:], want[3][..., -70:], "L")
    assert _native.device_status(0) == 0
