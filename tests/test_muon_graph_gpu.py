"""The whole optimiser step in a graph, matrices and biases, replayed beside the eager one; and a graph from before a step."""
import pytest
import torch

from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy
from detectron_pytorch_amd.muon import Muon

pytestmark = pytest.mark.gpu
DEV = "cuda"


def parameters():
    torch.manual_seed(3)
    shapes = [(40, 60), (130, 200), (16, 8, 3, 3), (60,)]
    ps = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in shapes]
    ps[2].data = ps[2].data.contiguous(memory_format=torch.channels_last)
    for p in ps:
        p.grad = torch.randn_like(p)
    return ps


def test_captured_after_a_first_step():
    held, eager = parameters(), parameters()
    a, b = (Muon(ps, lr=0.02, sgd_lr=0.1, weight_decay=0.01) for ps in (held, eager))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a.step()
    torch.cuda.current_stream().wait_stream(stream)
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for turn in range(4):
        for p, q in zip(held, eager):
            p.grad.mul_(-0.7)
            q.grad.mul_(-0.7)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for p, q in zip(held, eager):
            assert torch.equal(p, q), turn
            assert torch.equal(a.state[p]["momentum_buffer"], b.state[q]["momentum_buffer"]), turn


def test_a_graph_from_before_the_step_is_refused():
    w = torch.nn.Parameter(torch.randn(90, 64, device=DEV, dtype=torch.bfloat16))
    x = torch.randn(20, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = torch.randint(0, 90, (20,), device=DEV)
    opt = Muon([w], lr=0.02)
    linear_cross_entropy(x, w, None, y).backward()
    late = linear_cross_entropy(x, w, None, y)      # multiplies the weight where it lies, again in its backward
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late.backward()
