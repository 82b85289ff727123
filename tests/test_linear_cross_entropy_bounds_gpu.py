"""Gradients of the loss, each element within what its own terms allow: a row's own class alone has the rounding of p - 1, every other
probability that of itself, and what is lost below the smallest step of q is 2^-39 of the row's own gradient."""
import pytest
import torch

from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy
from test_linear_cross_entropy_gpu import DEV, FLOOR, HALF_STEP, TYPES, close, make

pytestmark = pytest.mark.gpu


def gradients(x, w, b, y, g):
    """dx, dw, db in float64 for a gradient `g` per row, with their bounds; roundings are counted as in test_linear_cross_entropy_gpu.py."""
    dtype = x.dtype
    x, w, b = x.detach().double(), w.detach().double(), b.detach().double()
    (rows, dim), classes, u = x.shape, w.size(0), HALF_STEP[dtype]
    full = dtype == torch.float32
    z = x @ w.t() + b
    size = x.abs() @ w.abs().t() + b.abs()
    ez = (8 * dim ** 0.5 + 4) * 2.0 ** -24 * size
    if full:
        ez = ez + 2.0 ** -20 * size + dim * 2.0 ** -38 * x.abs().max() * w.abs().max()
    t = z - torch.logsumexp(z, dim=1, keepdim=True)
    p, own = t.exp(), torch.nn.functional.one_hot(y, classes)
    # exp(z - lse): the logit's own error and that of lse, which is a mean of the logits' errors weighed by p, with its own sum's
    rel = ez + (p * ez).sum(dim=1, keepdim=True) + (2 + t.abs().clamp_max(104.0)) * 2.0 ** -21 + 8 * (32 + classes / 64) ** 0.5 * 2.0 ** -24
    g = g.double()[:, None]
    q = (p - own) * g
    eq = g.abs() * (p * rel + own * 2.0 ** -23 + (0.0 if dtype == torch.bfloat16 else 2.0 ** -39)) + ((2.0 ** -21 if full else u) + 2.0 ** -22) * q.abs()

    def product(a, ea, c, terms):
        v, mag = a @ c, a.abs() @ c.abs()
        small = 2.0 ** -38 * c.abs().max() * a.abs().sum(dim=1, keepdim=True) if full else 0.0
        return v, ea @ c.abs() + (8 * terms ** 0.5 * 2.0 ** -24 + (2.0 ** -20 if full else 0.0)) * mag + small + 1.01 * u * v.abs() + FLOOR[dtype]

    db = q.sum(dim=0)
    e_db = eq.sum(dim=0) + 8 * rows ** 0.5 * 2.0 ** -24 * q.abs().sum(dim=0) + 1.01 * u * db.abs() + FLOOR[dtype]
    return product(q, eq, w, classes), product(q.t(), eq.t(), x, rows), (db, e_db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,classes", [(65, 64, 200), (300, 96, 3001), (129, 64, 40001), (700, 513, 1204)])
def test_each_element_by_its_own_terms(rows, dim, classes, dtype):
    x, w, b, y = make(rows, dim, classes, dtype, ignored=0.0)
    got = torch.autograd.grad(linear_cross_entropy(x, w, b, y, reduction="sum"), (x, w, b))
    for t, v, name in zip(got, gradients(x, w, b, y, torch.ones(rows, device=DEV)), ("dx", "dw", "db")):
        close(t, v, name)


@pytest.mark.parametrize("dtype", TYPES)
def test_rare_classes(dtype):
    """Classes whose probabilities are from 1 down to 2^-60 everywhere, through the bias."""
    x, w, b, y = make(200, 64, 600, dtype, ignored=0.0)
    y = y % 100
    b = (b.detach() - torch.linspace(0, 40, 600, device=DEV).to(dtype)).requires_grad_(True)
    got = torch.autograd.grad(linear_cross_entropy(x, w, b, y, reduction="sum"), (x, w, b))
    for t, v, name in zip(got, gradients(x, w, b, y, torch.ones(200, device=DEV)), ("dx", "dw", "db")):
        close(t, v, name)
