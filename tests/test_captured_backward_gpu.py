"""A captured backward of leaves that a graph from before the capture holds. Their gradients go to the stream on which that graph was
made: another stream is taken into the capture, and the call is refused where it cannot be."""
import pytest
import torch

import hipkittens_b200 as hk
from hipkittens_b200 import _native
from hipkittens_b200.attention import QkNormRotary

pytestmark = pytest.mark.gpu


def rand(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()


def setup(native, seed):
    gen = torch.Generator().manual_seed(seed)
    x = [rand(gen, 2, 70, 4, 64).requires_grad_(), rand(gen, 2, 70, 2, 64).requires_grad_()]
    dy = rand(gen, 2, 70, 4, 64), rand(gen, 2, 70, 2, 64)
    angle = torch.arange(70, device="cuda")[:, None] / 100.0 ** (torch.arange(0, 64, 2, device="cuda") / 64)
    # the code behind the native function takes what that leaves to it: here an eps that is not a float
    m = QkNormRotary(64, eps=1e-6 if native else 1, device="cuda", dtype=torch.bfloat16)
    return x, dy, m, angle.cos(), angle.sin()


@pytest.mark.parametrize("into_grad", [True, False])
@pytest.mark.parametrize("native", [True, False])
def test_leaves_of_a_graph_on_a_side_stream_are_captured(native, into_grad):
    """What a warm-up on a side stream leaves behind, as wrappers for data-parallel training do."""
    x, dy, m, cos, sin = setup(native, 1)
    leaves = (*x, m.q_weight, m.k_weight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = m(*x, cos, sin)
        torch.autograd.backward(held, dy, retain_graph=True)
    torch.cuda.synchronize()
    want = [t.grad.clone() for t in leaves]
    for t in leaves:
        t.grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if into_grad:
            torch.autograd.backward(m(*x, cos, sin), dy)
            inside = [t.grad for t in leaves]
        else:
            inside = torch.autograd.grad(m(*x, cos, sin), leaves, dy)
    for t in inside:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(inside, want))
    for t in leaves:
        t.grad = None
    with torch.cuda.stream(side):  # the graph from before is as it was
        torch.autograd.backward(held, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(t.grad, b) for t, b in zip(leaves, want))


@pytest.mark.parametrize("native", [True, False])
def test_leaves_of_a_graph_on_the_default_stream_are_refused(native):
    """... before the engine makes that stream wait, which ends the capture and may end the process."""
    x, dy, m, cos, sin = setup(native, 2)
    leaves = (*x, m.q_weight)
    held = m(*x, cos, sin)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="no graph from before the capture holds"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(m(*x, cos, sin), leaves, dy)
    want = torch.autograd.grad(held, leaves, dy)
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = torch.autograd.grad(m(*x, cos, sin), leaves, dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(inside, want))
    assert _native.device_status(0) == 0 and hk.kernel_launch_count() > 0
