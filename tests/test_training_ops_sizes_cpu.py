"""Sizes that a C int does not hold are refused before they get there (a plain call would take them modulo 2^32)."""
import pytest
import torch

from detectron_pytorch_amd import _lib, linear_cross_entropy, orthogonalize

LONG = 2 ** 32 + 3


def empty(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.fixture(autouse=True)
def any_device(monkeypatch):
    monkeypatch.setattr(_lib, "require_cuda", lambda t, name: None)


def test_loss(hip_lib_path):
    for rows, dim, classes in ((LONG, 4, 5), (4, LONG, 5), (4, 5, LONG)):
        with pytest.raises(ValueError, match="2\\^24"):
            linear_cross_entropy.linear_cross_entropy(empty(rows, dim), empty(classes, dim), None, empty(rows, dtype=torch.int64))


def test_matrices():
    for shape in ((LONG, 4), (4, LONG)):
        with pytest.raises(ValueError, match="2\\^22"):
            orthogonalize.host_arrays([empty(3, 3), empty(*shape)])
    n, rows, cols = orthogonalize.host_arrays([empty(3, 4), empty(2 ** 22, 1)])
    assert n == 2 and list(rows) == [3, 2 ** 22] and list(cols) == [4, 1]
