"""The loss and its gradients where factors, gradients or rows are of very different magnitude.  Bounds are those of
test_linear_cross_entropy_gpu.py unless a test says otherwise."""
import pytest
import torch

from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy
from test_linear_cross_entropy_gpu import DEV, FLOOR, HALF_STEP, TYPES, check, close, formulas, make

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


def row_gradients(rows, spread):
    """Gradients of single rows from 2^-spread to 2^spread in no order, the ends among them."""
    g = torch.Generator(device=DEV)
    g.manual_seed(spread)
    return torch.linspace(-spread, spread, rows, device=DEV)[torch.randperm(rows, generator=g, device=DEV)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [90, 3001])
def test_a_rows_gradient_does_not_depend_on_the_other_rows(classes, dtype):
    """A power of two times a row's gradient is that power of two times its dx, exactly so but where the type's steps are all alike: there
    either side is off by half of one, and that of a gradient of 1 (fp16: 2^-25) is taken times the power."""
    x, w, b, y = make(150, 72, classes, dtype)
    power = torch.exp2(row_gradients(150, 6 if dtype == torch.float16 else 50).round())
    losses = linear_cross_entropy(x, w, b, y, reduction="none")
    (one,) = torch.autograd.grad(losses, (x,), torch.ones_like(losses), retain_graph=True)
    for wanted in ((x,), (x, w, b)):
        got = torch.autograd.grad(losses, wanted, power, retain_graph=True)[0]
        off = (got.double() - one.double() * power.double()[:, None]).abs()
        assert bool((off <= FLOOR[dtype] * (1 + power.double()[:, None])).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_has_its_own_gradients_accuracy(dtype):
    """dx of a row is its gradient times dx of a gradient of 1, and so is its error's bound, with one more rounding of the product."""
    x, w, b, y = make(200, 64, 1000, dtype)
    g = torch.exp2(row_gradients(200, 5 if dtype == torch.float16 else 50)) * torch.where(torch.rand(200, device=DEV) < 0.5, -1.0, 1.0)
    _, _, (value, bound), _, _, keep = formulas(x, w, b, y, reduction="none", grad=torch.ones(200, device=DEV))
    value, size = value * g.double()[:, None], g.double().abs()[:, None]
    losses = linear_cross_entropy(x, w, b, y, reduction="none")
    for wanted in ((x,), (x, w), (x, w, b)):
        got = torch.autograd.grad(losses, wanted, g, retain_graph=True)[0]
        close(got, (value, size * (bound + 2.0 ** -22 * (value / size).abs()) + FLOOR[dtype]), "dx")
        assert bool((got[~keep] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 0)])
def test_some_gradients_of_weighted_rows(wanted, dtype):
    x, w, b, y = make(130, 64, 300, dtype)
    g = torch.exp2(row_gradients(130, 5))
    want = formulas(x, w, b, y, reduction="none", grad=g)[2:5]
    losses = linear_cross_entropy(x, w, b, y, reduction="none")
    got = torch.autograd.grad(losses, [t for t, f in zip((x, w, b), wanted) if f], g)
    for t, v in zip(got, [v for v, f in zip(want, wanted) if f]):
        close(t, v, str(wanted))


@pytest.mark.parametrize("dtype", TYPES)
def test_row_gradients_that_are_zero_or_no_number(dtype):
    x, w, b, y = make(130, 64, 300, dtype)
    g = torch.ones(130, device=DEV)
    rows = torch.nonzero(y >= 0)[:, 0]
    g[rows[3]] = 0.0
    g[torch.nonzero(y < 0)[:, 0]] = float("nan")     # of rows that do not count
    want = formulas(x, w, b, y, reduction="none", grad=torch.where(y < 0, 0.0, g))
    got = torch.autograd.grad(linear_cross_entropy(x, w, b, y, reduction="none"), (x, w, b), g)
    for t, v in zip(got, want[2:5]):
        close(t, v, "zero")
    assert bool((got[0][rows[3]] == 0).all()) and bool((got[0][y < 0] == 0).all())
    g[rows[5]] = float("inf")
    gx, gw = torch.autograd.grad(linear_cross_entropy(x, w, b, y, reduction="none"), (x, w), g)
    assert not bool(torch.isfinite(gx[rows[5]]).all()) and not bool(torch.isfinite(gw).all())
    others = (y >= 0) & (torch.arange(130, device=DEV) != rows[5])
    assert torch.equal(gx[others], got[0][others])
    zeros = torch.autograd.grad(linear_cross_entropy(x, w, b, y, reduction="none"), (x, w, b), torch.zeros(130, device=DEV))
    assert all(bool((t == 0).all()) for t in zeros)


@pytest.mark.parametrize("dtype", TYPES)
def test_weighted_rows_over_several_pieces(dtype):
    """Rows of very different gradient where dx is added up over pieces of the vocabulary: against the rows by themselves."""
    rows = 16384 if dtype == torch.float32 else 30000
    x, w, b, y = make(rows, 16, 20010, dtype, ignored=0.05)
    power = torch.exp2(row_gradients(rows, 6 if dtype == torch.float16 else 40).round())
    losses = linear_cross_entropy(x, w, b, y, reduction="none")
    (one,) = torch.autograd.grad(losses, (x,), torch.ones_like(losses), retain_graph=True)
    got = torch.autograd.grad(losses, (x, w), power, retain_graph=True)
    off = (got[0].double() - one.double() * power.double()[:, None]).abs()
    assert bool((off <= FLOOR[dtype] * (1 + power.double()[:, None])).all())
    # the same sum over rows, as gradients of the sum of a part of them at a time
    want = torch.zeros(20010, 16, dtype=torch.float64, device=DEV)
    for p in power.unique():
        mine = torch.where(power == p, y, -1)
        want += torch.autograd.grad(linear_cross_entropy(x, w, b, mine, reduction="sum"), (w,))[0].double() * p.double()
    u = 2 * HALF_STEP[dtype] if dtype != torch.float32 else 2.0 ** -18
    assert float((got[1].double() - want).norm() / want.norm()) <= u


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("classes", [70, 3001])
def test_ignored_rows_beside_a_weight_that_is_no_number(classes, reduction, dtype):
    """A row that does not count has a gradient of zero, whatever the other operand holds; the others show it."""
    for value in (float("nan"), float("inf")):
        x, w, b, y = make(200, 64, classes, dtype, ignored=0.4)
        bad = w.detach().clone()
        bad[classes // 2, 11] = value
        bad.requires_grad_(True)
        loss = linear_cross_entropy(x, bad, b, y, reduction=reduction).sum()
        gx, gw, gb = torch.autograd.grad(loss, (x, bad, b))
        rows = y == -1
        # (a row of that class itself, at a logit of -inf: q = -1, -1 times inf)
        assert bool((gx[rows] == 0).all()) and not bool(torch.isfinite(gx[~rows]).all(dim=1).any())
        none = torch.full_like(y, -1)
        for t in torch.autograd.grad(linear_cross_entropy(x, bad, b, none, reduction=reduction).sum(), (x, bad, b)):
            assert bool((t == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_row_gradients_at_the_two_ends_of_a_float(dtype):
    """A row whose gradient is nothing beside the others' leaves no trace in the sum over rows."""
    x, w, b, y = make(130, 64, 300, dtype, ignored=0.0)
    g = torch.full((130,), 2.0 ** 20, device=DEV)
    g[40], g[41], g[42] = 2.0 ** -145, 2.0 ** -120, -2.0 ** -100
    want = formulas(x, w, b, y, reduction="none", grad=g)
    losses = linear_cross_entropy(x, w, b, y, reduction="none")
    for wanted in ((0, 1, 2), (1,), (1, 2), (0,)):
        got = torch.autograd.grad(losses, [(x, w, b)[k] for k in wanted], g, retain_graph=True)
        for k, t in zip(wanted, got):
            close(t, want[2 + k], "%s of %s" % (k, wanted))
        if 0 in wanted:
            assert float(got[0][40:43].abs().max()) < 2.0 ** -90
