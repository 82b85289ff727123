"""Gradients of the loss when autograd's saved tensors are packed and unpacked on the way: the same bits as without."""
import pytest
import torch

from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy
from test_linear_cross_entropy_gpu import DEV, TYPES, check, make

pytestmark = pytest.mark.gpu


def weights(w):
    """The same elements on every kind of place: dense, rows apart on 16 bytes, rows apart off them, dense off them."""
    rows, cols = w.shape
    apart = torch.randn(rows, cols + 144, device=DEV).to(w.dtype)
    apart[:, 8:8 + cols] = w
    off = torch.randn(rows, cols + 145, device=DEV).to(w.dtype)
    off[:, 3:3 + cols] = w
    dense_off = torch.zeros(rows * cols + 8, dtype=w.dtype, device=DEV)[3:3 + rows * cols].view(rows, cols)
    dense_off.copy_(w)
    return {"dense": w.clone(), "apart": apart[:, 8:8 + cols], "off": off[:, 3:3 + cols], "dense off": dense_off}


def moved_off(t):
    """A clone that does not start on 16 bytes."""
    flat = torch.zeros(t.numel() + 16, dtype=t.dtype, device=t.device)
    return flat[1:1 + t.numel()].view(t.shape).copy_(t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 72])
def test_hooks_that_move_what_was_saved(dim, dtype):
    x, w, b, y = make(130, dim, 200, dtype)
    for place, weight in weights(w.detach()).items():
        weight = weight.detach().requires_grad_(True)
        want = torch.autograd.grad(linear_cross_entropy(x, weight, b, y), (x, weight, b))
        for unpack in (lambda t: t.clone(memory_format=torch.contiguous_format), moved_off):
            print(place, dim, dtype, unpack, flush=True)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                got = torch.autograd.grad(linear_cross_entropy(x, weight, b, y), (x, weight, b))
            for a, c in zip(got, want):
                assert torch.equal(a, c), place
        with torch.autograd.graph.save_on_cpu():
            got = torch.autograd.grad(linear_cross_entropy(x, weight, b, y), (x, weight, b))
        for a, c in zip(got, want):
            assert torch.equal(a, c), place


@pytest.mark.parametrize("dtype", TYPES)
def test_places_of_a_weight_against_the_formulas(dtype):
    x, w, b, y = make(130, 64, 200, dtype)
    for weight in weights(w.detach()).values():
        check(x, weight.detach().requires_grad_(True), b, y)
