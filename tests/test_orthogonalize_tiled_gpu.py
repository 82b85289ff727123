"""The hard cases of orthogonalize where the products run on tiles of 22-bit pairs (short side above 64, or a long side above 16384), and
the border between that way and the one of short sides.

Tolerances.  ITERATION (test_orthogonalize_gpu.py) holds for matrices without a wide gap in their spectrum.  Where there is one, an error of
the first products along directions that the matrix does not have grows by the first coefficient a in each step that follows: at most
3 products a step with 2^-21 each, their sum over the steps a geometric one of a^steps (1 + 1/a + ...) <= 1.5 a^steps.
"""
import pytest
import torch

from detectron_pytorch_amd.muon import muon_step_
from detectron_pytorch_amd.orthogonalize import COEFFICIENTS, orthogonalize, orthogonalize_many
from test_orthogonalize_gpu import DEV, ITERATION, TYPES, close, formula, gradient, reference_step

pytestmark = pytest.mark.gpu


def noise(coefficients=COEFFICIENTS, steps=5):
    return 3 * 1.5 * 2.0 ** -21 * coefficients[0] ** steps


SIDES = [(40, 60), (200, 300), (300, 200), (130, 1000), (1100, 1030)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(1, 16384), (1, 16385), (16385, 1), (3, 20000), (20000, 64), (64, 16384), (64, 16385), (33, 40001), (65, 65),
                                 (65, 20000), (1, 1 << 20)])
def test_border_between_the_two_ways(m, n, dtype):
    g = gradient(m, n, dtype)
    close(orthogonalize(g), formula(g), dtype, "%d x %d" % (m, n))


@pytest.mark.parametrize("m,n", SIDES)
def test_zero(m, n):
    for dtype in TYPES:
        assert bool((orthogonalize(torch.zeros(m, n, dtype=dtype, device=DEV)) == 0).all())


@pytest.mark.parametrize("m,n", SIDES)
def test_rank_one(m, n):
    g = gradient(m, 1, torch.float32) @ gradient(1, n, torch.float32)
    close(orthogonalize(g), formula(g), torch.float32, "rank one", noise())


@pytest.mark.parametrize("m,n", SIDES)
def test_repeated_and_zero_rows_and_columns(m, n):
    g = gradient(m, n, torch.float32)
    g[1::2] = g[0::2][:g[1::2].size(0)]
    g[10] = 0
    g[:, 3] = 0
    close(orthogonalize(g), formula(g), torch.float32, "repeated rows", noise())


@pytest.mark.parametrize("m,n", SIDES)
def test_rows_of_very_different_size(m, n):
    """One direction of 2^-20 of the others and less, as embeddings of rare entries have."""
    g = gradient(m, n, torch.float32)
    g[5] *= 2.0 ** -20
    g[:, 7] *= 2.0 ** -30
    close(orthogonalize(g), formula(g), torch.float32, "scaled", noise())


@pytest.mark.parametrize("m,n", SIDES)
def test_one_value(m, n):
    g = torch.zeros(m, n, device=DEV)
    g[m - 1, n - 1] = -3.0
    out = orthogonalize(g)
    close(out, formula(g), torch.float32, "one value")
    out[m - 1, n - 1] = 0
    assert bool((out == 0).all())


@pytest.mark.parametrize("m,n", SIDES)
def test_smaller_than_eps(m, n):
    g = gradient(m, n, torch.float32)
    g = g / g.norm() * 1e-3
    close(orthogonalize(g, eps=1.0), formula(g, eps=1.0), torch.float32, "eps")


@pytest.mark.parametrize("m,n", SIDES)
def test_not_a_number_stays_in_its_matrix(m, n):
    for bad in (float("nan"), float("inf"), float("-inf")):
        mats = [gradient(m, n, torch.float32, seed=k) for k in range(3)]
        mats[1][m // 2, n // 3] = bad
        outs = orthogonalize_many(mats)
        assert bool(torch.isnan(outs[1]).any())
        for k in (0, 2):
            close(outs[k], formula(mats[k]), torch.float32, "the other matrix")


@pytest.mark.parametrize("m,n", SIDES)
@pytest.mark.parametrize("coefficients,steps", [((1.5, -0.5, 0.0), 12), ((2.0, -1.5, 0.5), 12), ((1.875, -1.25, 0.375), 12),
                                                ((3.86, -11.9, 7.42), 5), ((4.96, -8.2, 2.74), 5), ((4.99, -6.09, 1.49), 5),
                                                ((0.0, 1.0, 0.0), 3), ((-1.5, 0.5, 0.0), 5)])
def test_other_coefficients(coefficients, steps, m, n):
    """Two or three iterations share a pass over the long side where n is a multiple of m, so these are products of several factors."""
    g = gradient(m, n, torch.float32)
    close(orthogonalize(g, steps=steps, coefficients=coefficients), formula(g, steps, coefficients), torch.float32, str(coefficients),
          max(4 * ITERATION, noise(coefficients, steps) if steps <= 5 else 0))


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
def test_other_steps(steps):
    for m, n in SIDES[1:] + [(80, 4000)]:
        g = gradient(m, n, torch.float32)
        close(orthogonalize(g, steps=steps), formula(g, steps), torch.float32, "%d steps" % steps, ITERATION * max(1, steps / 5))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    g = gradient(400, 700, dtype)
    views = [g[3:250, 7:300], g.t(), g[::2, ::3], g[:0], g[1:301, 1:302], g[:, 5:90], g.view(-1)[1:1 + 200 * 300].view(200, 300)]
    for v, o in zip(views, orthogonalize_many(views)):
        assert o.shape == v.shape
        if v.numel():
            close(o, formula(v), dtype, "view %s" % (tuple(v.shape),))


@pytest.mark.parametrize("dtype", TYPES)
def test_any_magnitude(dtype):
    for s in {torch.float32: (1e-36, 1e-20, 1e20, 1e36), torch.bfloat16: (1e-36, 1e36), torch.float16: (1e-3, 1e3)}[dtype]:
        h = (gradient(150, 220, torch.float32) * s).to(dtype)
        close(orthogonalize(h, eps=1e-44), formula(h, eps=1e-44), dtype, "%g" % s)


@pytest.mark.parametrize("dtype", TYPES)
def test_step_of_large_and_small_matrices(dtype):
    """Both ways in one step, one of the matrices without a gradient's value, one of them off 16 bytes."""
    shapes = [(200, 300), (30, 70), (300, 200), (1, 20000), (150, 150)]
    ps = [gradient(m, n, dtype, 1) for m, n in shapes]
    off = torch.zeros(150 * 150 + 8, dtype=dtype, device=DEV)[1:1 + 150 * 150].view(150, 150)
    off.copy_(ps[4])
    ps[4] = off
    ms = [torch.zeros(m, n, device=DEV) for m, n in shapes]
    u = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    for turn in range(3):
        gs = [gradient(m, n, dtype, 3 + turn) for m, n in shapes]
        gs[2].zero_()
        want = [reference_step(p, g, m, 0.05, 0.9, 0.1, True) for p, g, m in zip(ps, gs, ms)]
        muon_step_(ps, gs, ms, lr=0.05, momentum=0.9, weight_decay=0.1)
        for p, m, (wp, wm) in zip(ps, ms, want):
            scale = 0.05 * max(1.0, p.size(0) / p.size(1)) ** 0.5
            # a row alone: the iteration's error is all in one direction, as large as its norm
            bound = (u + 2.0 ** -23) * wp.abs() + scale * (4 * ITERATION) + 2.0 ** -25
            assert bool(((p.double() - wp).abs() <= bound).all())
            assert bool(((m.double() - wm).abs() <= 2.0 ** -22 * (wm.abs() + 0.1)).all())


@pytest.mark.parametrize("m,n", SIDES)
@pytest.mark.parametrize("coefficients,steps", [((2.75, 0.02, 0.0), 1), ((3.9, -1.3, 0.1), 2), ((3.9, -1.3, 0.1), 4)])
def test_singular_values_near_the_largest_that_is_stored(coefficients, steps, m, n):
    """A single direction starts at 1 and comes to 2.7 after one step: its square fills 91 % of the stored form's range."""
    g = torch.zeros(m, n, device=DEV)
    g[3, 4] = 5.0
    close(orthogonalize(g, steps=steps, coefficients=coefficients), formula(g, steps, coefficients), torch.float32, "one value")
    g = gradient(m, 1, torch.float32) @ gradient(1, n, torch.float32)
    close(orthogonalize(g, steps=steps, coefficients=coefficients), formula(g, steps, coefficients), torch.float32, "rank one",
          max(ITERATION, noise(coefficients, steps)))


@pytest.mark.parametrize("m,n", SIDES)
def test_a_weight_is_rounded_once(m, n):
    """Half a step of the new weight, and the decay's own rounding (half a step of a number in [0.5, 1)); what the iteration is off by is
    small beside that for weights around 100 and a rate of 2e-4."""
    p, g, mom = 100 * gradient(m, n, torch.float32, 1) / 1e-2, gradient(m, n, torch.float32, 2), torch.zeros(m, n, device=DEV)
    want, _ = reference_step(p, g, mom, 2e-4, 0.95, 0.5, True)
    muon_step_([p], [g], [mom], lr=2e-4, weight_decay=0.5)
    bound = (2.0 ** -24 + 1.01 * 2.0 ** -25) * want.abs() + 2e-4 * max(1.0, m / n) ** 0.5 * 4 * ITERATION
    assert bool(((p.double() - want).abs() <= bound).all())
