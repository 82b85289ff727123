"""The optimiser step writes parameters and momenta through their addresses: autograd has to hear of it, as it does of torch's own in-place
operations.  On the CPU, with the launching entry of the library replaced by one that does nothing."""
import contextlib

import pytest
import torch

from detectron_pytorch_amd import _lib, muon


class Silent:
    def __init__(self, lib):
        self.lib = lib

    def __getattr__(self, name):
        return (lambda *args: 0) if name == "mi_muon_step" else getattr(self.lib, name)


@pytest.fixture
def silent(hip_lib_path, monkeypatch):
    s = Silent(_lib.lib())
    monkeypatch.setattr(_lib, "lib", lambda: s)
    monkeypatch.setattr(_lib, "require_cuda", lambda t, name: None)
    monkeypatch.setattr(_lib, "current_stream_handle", lambda device: None)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())


def test_a_graph_from_before_the_step_is_refused(silent):
    w = torch.nn.Parameter(torch.randn(4, 6))
    conv = torch.nn.Parameter(torch.randn(4, 3, 2, 2).contiguous(memory_format=torch.channels_last))
    x = torch.randn(5, 4, requires_grad=True)
    opt = muon.Muon([w, conv], lr=0.1)
    w.grad, conv.grad = torch.randn(4, 6), torch.randn(4, 3, 2, 2)
    before = (x @ w).sum() + (conv * conv).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        before.backward()
    versions = [t._version for t in (w, conv)]
    grads = [w.grad._version, conv.grad._version]
    opt.step()
    assert all(t._version > v for t, v in zip((w, conv), versions))
    assert [w.grad._version, conv.grad._version] == grads


def test_momenta_and_parameters_count_gradients_do_not(silent):
    p, g, m = torch.zeros(3, 4), torch.zeros(3, 4), torch.zeros(3, 4)
    muon.muon_step_([p], [g], [m], lr=0.1)
    assert p._version == m._version == 1 and g._version == 0
    with torch.inference_mode():
        q = torch.zeros(3, 4)   # has no version
        muon.muon_step_([q], [q + 1], [torch.zeros(3, 4)], lr=0.1)
    muon.muon_step_([q], [torch.zeros(3, 4)], [m], lr=0.1)
    assert m._version == 2
