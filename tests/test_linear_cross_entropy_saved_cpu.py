"""What the loss hands its backward when autograd's saved tensors are packed and unpacked: looked at on the CPU, with the two launching
entries of the library replaced by ones that write down their arguments."""
import contextlib

import pytest
import torch

from detectron_pytorch_amd import _lib
from detectron_pytorch_amd import linear_cross_entropy as module


class Recorder:
    """The library with its launches written down; sizes come from the library itself."""

    def __init__(self, lib):
        self.lib, self.calls = lib, {}

    def __getattr__(self, name):
        if name not in ("mi_linear_cross_entropy_forward", "mi_linear_cross_entropy_backward"):
            return getattr(self.lib, name)

        def call(*args):
            self.calls[name.rsplit("_", 1)[1]] = args
            return 0

        return call


@pytest.fixture
def recorder(hip_lib_path, monkeypatch):
    r = Recorder(_lib.lib())
    monkeypatch.setattr(_lib, "lib", lambda: r)
    monkeypatch.setattr(_lib, "current_stream_handle", lambda device: None)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    return r


def on_16_bytes(rows, cols, offset, dtype):
    """[rows, cols] whose first element lies `offset` elements behind a multiple of 256 bytes."""
    flat = torch.zeros(rows * cols + 512, dtype=dtype)
    first = (-flat.data_ptr() % 256) // flat.element_size() + offset
    return flat[first:first + rows * cols].view(rows, cols)


def run(recorder, weight, unpack):
    x = torch.zeros(5, weight.size(1), dtype=weight.dtype, requires_grad=True)
    given = []

    def unpacked(t):
        out = unpack(t)
        given.append(out)
        return out

    weight = weight.detach().requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpacked):
        loss = module._LinearCrossEntropy.apply(x, weight, None, torch.zeros(5, dtype=torch.int64), -1, _lib.REDUCTION_MEAN, False)
        torch.autograd.grad(loss, (x, weight), torch.ones(()))
    return given, recorder.calls["backward"]


def test_row_distance_is_that_of_the_unpacked_weight(recorder):
    wide = on_16_bytes(9, 208, 0, torch.bfloat16)
    given, args = run(recorder, wide[:, 8:72], lambda t: t.clone(memory_format=torch.contiguous_format))
    weight = [t for t in given if t is not None and t.shape == (9, 64)][0]
    assert args[1] == weight.data_ptr() and args[2] == weight.stride(0) == 64


def test_a_weight_read_in_place_comes_back_on_16_bytes(recorder):
    """The forward multiplied it where it lay and kept no copy: what the backward reads must allow that too."""
    given, args = run(recorder, on_16_bytes(9, 64, 0, torch.float16),
                      lambda t: on_16_bytes(9, 64, 3, t.dtype).copy_(t) if t.shape == (9, 64) else t)
    assert args[1] % 16 == 0 and args[2] == 64
    saved = [t for t in given if t is not None and t.dtype == torch.uint8][0]
    assert recorder.lib.mi_linear_cross_entropy_saved_bytes(5, 64, 9, _lib.TYPE_F16, args[1], args[2]) <= saved.numel() == args[13]


def test_what_was_kept_comes_back_on_its_alignment(recorder):
    def unpack(t):
        if t is None or t.dtype != torch.uint8:
            return t
        return on_16_bytes(1, t.numel(), 16, torch.uint8).view(-1).copy_(t)

    _, args = run(recorder, on_16_bytes(9, 64, 0, torch.float32), unpack)
    assert args[12] % 64 == 0
