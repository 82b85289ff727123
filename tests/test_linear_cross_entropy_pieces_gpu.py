"""Weights that are laid out in pieces: more than 128 MB of float32 ones, or of 16-bit ones whose rows are padded.  Against the formulas of
test_linear_cross_entropy_gpu.py."""
import pytest
import torch

from detectron_pytorch_amd import _lib
from detectron_pytorch_amd.linear_cross_entropy import TYPES as CODES
from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy
from test_linear_cross_entropy_gpu import DEV, check, make

pytestmark = pytest.mark.gpu

LARGE = [(torch.float32, 1024, 40001), (torch.float16, 1001, 70003), (torch.bfloat16, 999, 70003)]


def is_in_pieces(w):
    (classes, dim), dtype = w.shape, CODES[w.dtype]
    size = lambda n: _lib.lib().mi_linear_cross_entropy_saved_bytes(64, dim, n, dtype, w.data_ptr(), dim)  # noqa: E731
    return size(classes) < size(classes // 4)   # nothing of the weights is kept


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype,dim,classes", LARGE)
def test_against_the_formulas(dtype, dim, classes, reduction):
    x, w, b, y = make(90, dim, classes, dtype)
    assert is_in_pieces(w)
    grad = None if reduction == "mean" else torch.linspace(-3, 3, 90, device=DEV)
    check(x, w, b, y, reduction=reduction, grad=grad)


def test_without_bias_and_with_32_bit_labels():
    check(*make(90, 1024, 40001, torch.float32, bias=False, labels=torch.int32))


def test_lowest_class_of_equal_logits_and_nan_across_pieces():
    x, w, _, y = make(70, 1024, 40001, torch.float32, ignored=0.0)
    w = w.detach()
    w[37000:37300] = w[100:400]
    x = w[137].expand(70, 1024).contiguous() * 4
    _, pred = linear_cross_entropy(x, w, None, y, with_pred=True)
    assert bool((pred == 137).all())
    w[38000, 5] = float("nan")
    loss, pred = linear_cross_entropy(x, w, None, y, with_pred=True, reduction="none")
    assert bool((pred == 38000).all()) and bool(torch.isnan(loss).all())


@pytest.mark.parametrize("dtype,dim,classes", LARGE[:2])
def test_saved_tensors_that_move_and_replays(dtype, dim, classes):
    x, w, b, y = make(90, dim, classes, dtype)
    leaves = (x, w, b)
    want = torch.autograd.grad(linear_cross_entropy(*leaves, y), leaves)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)):
        got = torch.autograd.grad(linear_cross_entropy(*leaves, y), leaves)
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    del want
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(linear_cross_entropy(*leaves, y), leaves)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.autograd.grad(linear_cross_entropy(*leaves, y), leaves)
    for turn in range(3):
        with torch.no_grad():
            x.mul_(0.7)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, torch.autograd.grad(linear_cross_entropy(*leaves, y), leaves)):
            assert torch.equal(a, c), turn
