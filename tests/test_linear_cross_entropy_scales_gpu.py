"""The loss and its gradients where factors, gradients or rows are of very different magnitude.  Bounds are those of
test_linear_cross_entropy_gpu.py unless a test says otherwise."""
import pytest
import torch

from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy
from test_linear_cross_entropy_gpu import DEV, TYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale,size", [(1e-35, 1), (1e35, 1), (1e33, 60)])
def test_logits_are_ordinary_where_their_factors_are_not(scale, size):
    x, w, b, y = make(130, 70, 200, torch.float32)
    check((x.detach() * scale).requires_grad_(True), (w.detach() * (size / scale)).requires_grad_(True), b, y)


@pytest.mark.parametrize("scale,grad", [(1e-20, 1e-12), (1e-20, 1e-15), (1e20, 1e12), (1e25, 1e-25)])
def test_gradients_are_ordinary_where_their_factors_are_not(scale, grad):
    x, w, b, y = make(130, 70, 200, torch.float32)
    x, w = (x.detach() * scale).requires_grad_(True), (w.detach() / scale).requires_grad_(True)
    check(x, w, b, y, reduction="sum", grad=torch.tensor(grad, device=DEV))
