"""Captures beside living eager graphs, where the leaves stand behind other operations."""
import pytest
import torch

from immunostruct_amd import functional as HF, nn as HN
from immunostruct_amd.models.layers import DifferentialAttention

pytestmark = pytest.mark.gpu


def test_leaves_behind_a_projection(cuda_device):
    """a module whose eager outputs are alive: its capture is refused, and works once they are gone (a backward pass in it would make the eager
    stream wait for the captured one)"""
    torch.manual_seed(4)
    m = DifferentialAttention(64, 4, kv_heads=2, rotary=HN.RotaryEmbedding(8)).cuda()
    x = torch.randn(2, 9, 64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(x)
    torch.cuda.current_stream().wait_stream(side)
    eager = m(x)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            m(x)
    want = eager.detach().clone()
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = m(x)
    for scale in (1.0, 0.5):
        with torch.no_grad():
            x.mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        if scale == 1.0:
            assert torch.equal(held, want)
        else:
            with torch.no_grad():
                assert torch.equal(held, m(x))


@pytest.mark.parametrize("wrap", [lambda t: t * 1.0, lambda t: t.view(t.shape) + 0.0, lambda t: t.transpose(1, 2).transpose(1, 2)], ids=["product", "sum", "views"])
def test_leaves_behind_elementary_operations(cuda_device, wrap):
    q, k = (torch.randn(1, 12, 2, 16, device="cuda", requires_grad=True) for _ in range(2))
    v, lam = torch.randn(1, 12, 1, 32, device="cuda", requires_grad=True), torch.ones(1, device="cuda")
    freq = HN.RotaryEmbedding(16).freq
    calls = [lambda: HF.differential_attention(wrap(q), wrap(k), wrap(v), lam), lambda: HF.rotary(wrap(q), None, freq)[0], lambda: HF.group_norm(wrap(v), 2)]
    for call in calls:
        eager = call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        want = eager.detach().clone()
        del eager
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
        del held      # (it would keep the leaves' nodes on the captures' stream, where nothing has to wait)


def test_an_eager_input_is_no_leaf_of_the_capture(cuda_device):
    """a forward pass over something computed before the capture records nothing of what lies behind it"""
    leaf = torch.randn(2, 12, 32, device="cuda", requires_grad=True)
    x = leaf * 2.0
    want = HF.group_norm(x, 2).detach().clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = HF.group_norm(x, 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, want)
