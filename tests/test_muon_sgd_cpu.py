"""The parameters of an optimiser with orthogonalised updates that take the momentum SGD step."""
import pytest
import torch

from detectron_pytorch_amd import muon
from detectron_pytorch_amd.muon import Muon


def test_a_float64_bias_keeps_its_bits():
    start = torch.tensor([1.0 + 2.0 ** -40, -3.0 + 2.0 ** -45], dtype=torch.float64)
    p = torch.nn.Parameter(start.clone())
    opt = Muon([p], lr=0.5, sgd_lr=0.25, sgd_momentum=0.5)
    p.grad = torch.zeros_like(p)
    opt.step()
    assert torch.equal(p.detach(), start)
    p.grad = torch.tensor([0.5, -0.25], dtype=torch.float64)
    opt.step()
    opt.step()   # momentum 0.5 g + g
    assert torch.equal(p.detach(), start - 0.25 * torch.tensor([0.5 + 0.75, -0.25 - 0.375], dtype=torch.float64))
    assert opt.state[p]["momentum_buffer"].dtype == torch.float32


def test_16_bit_biases_are_rounded_once():
    torch.manual_seed(0)
    for dtype in (torch.float16, torch.bfloat16):
        p = torch.nn.Parameter(torch.randn(50).to(dtype))
        opt = Muon([p], lr=0.5, sgd_lr=0.1, weight_decay=0.01)
        m, w = torch.zeros(50), p.detach().clone()
        for _ in range(3):
            p.grad = torch.randn(50).to(dtype)
            m = 0.9 * m + p.grad.float() + 0.01 * w.float()
            opt.step()
            assert float((p.detach().double() - (w.double() - 0.1 * m.double())).abs().max()) <= \
                torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8) * float(p.detach().abs().max().double() + 1)
            w = p.detach().clone()


def test_momenta_are_not_made_inside_a_graph(monkeypatch):
    """They would be cleared, or taken from a tensor that is gone, at every replay."""
    w = torch.nn.Parameter(torch.randn(4, 3, 2, 2))
    opt = Muon([w], orthogonalize=False)
    w.grad = torch.randn(4, 3, 2, 2)
    monkeypatch.setattr(muon, "_is_captured", lambda p: True)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    assert len(opt.state) == 0 or "momentum_buffer" not in opt.state[w]
    monkeypatch.setattr(muon, "_is_captured", lambda p: False)
    opt.step()
    monkeypatch.setattr(muon, "_is_captured", lambda p: True)
    opt.step()
    w.data = w.data.contiguous(memory_format=torch.channels_last)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
