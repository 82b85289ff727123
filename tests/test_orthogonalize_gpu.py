"""Orthogonalised matrices and the optimiser step against the formulas in 64 bits.

Tolerances.  The iteration's products carry 22 bits; an error e |X| of one of its forms reaches the result through the remaining
steps, at most a^steps = 485 times along the smallest singular directions, and in the 2-norm by a few times for matrices
without a wide gap in their spectrum.  15 products with 2^-21 each and a factor of 8 between the norms: 6e-5 of the result's
norm.  Rounding to the type adds half a step of each element.
"""
import math

import pytest
import torch

from detectron_pytorch_amd.muon import Muon, muon_step_
from detectron_pytorch_amd.orthogonalize import COEFFICIENTS, orthogonalize, orthogonalize_many

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ITERATION = 15 * 8 * 2.0 ** -21


def formula(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = g.double() if g.size(0) <= g.size(1) else g.double().t()
    x = x / torch.linalg.matrix_norm(x).clamp_min(eps)
    for _ in range(steps):
        gram = x @ x.t()
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x if g.size(0) <= g.size(1) else x.t()


def close(got, want, dtype, what, iteration=ITERATION):
    assert torch.isfinite(got).all(), what
    off = torch.linalg.vector_norm(got.double() - want)
    allowed = (iteration + HALF_STEP[dtype]) * torch.linalg.vector_norm(want) + want.numel() ** 0.5 * 2.0 ** -25
    assert float(off) <= float(allowed), "%s: off by %.3g where %.3g is allowed" % (what, float(off), float(allowed))


def gradient(m, n, dtype, seed=0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + 31 * m + n)
    r = max(1, min(m, n) // 8)
    g = torch.randn(m, r, generator=gen, device=DEV) @ torch.randn(r, n, generator=gen, device=DEV) / math.sqrt(r)
    return (1e-2 * (g + torch.randn(m, n, generator=gen, device=DEV))).to(dtype)


SIZES = [(1, 1), (1, 2), (1, 300), (300, 1), (2, 2), (3, 5), (16, 16), (31, 33), (33, 31), (64, 64), (65, 64), (64, 257),
         (127, 130), (200, 1000), (1000, 200), (129, 4001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SIZES)
def test_against_the_formula(m, n, dtype):
    g = gradient(m, n, dtype)
    before = g.clone()
    out = orthogonalize(g)
    assert out.shape == g.shape and out.dtype == dtype and torch.equal(g, before)
    close(out, formula(g), dtype, "%d x %d" % (m, n))


@pytest.mark.parametrize("m,n", [(1500, 1500), (600, 9000), (5000, 700)])
def test_large_tiles_and_slices(m, n):
    for dtype in (torch.float32, torch.bfloat16):
        g = gradient(m, n, dtype)
        close(orthogonalize(g), formula(g), dtype, "%d x %d" % (m, n))


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 10])
def test_other_steps(steps):
    for m, n in ((50, 70), (70, 400)):
        g = gradient(m, n, torch.float32)
        close(orthogonalize(g, steps=steps), formula(g, steps), torch.float32, "%d steps" % steps, ITERATION * max(1, steps / 5))


def test_other_coefficients():
    g = gradient(60, 100, torch.float32)
    for c in ((1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)):
        close(orthogonalize(g, steps=12, coefficients=c), formula(g, 12, c), torch.float32, str(c), 4 * ITERATION)


def test_many_of_different_sizes():
    mats = [gradient(m, n, torch.float32, seed=k) for k in range(3) for m, n in SIZES]        # more than one table
    outs = orthogonalize_many(mats)
    for g, o in zip(mats, outs):
        close(o, formula(g), torch.float32, str(tuple(g.shape)))
    again = orthogonalize_many(mats)
    for a, b in zip(outs, again):
        assert torch.equal(a, b)


def test_any_magnitude():
    for dtype, scales in ((torch.float32, (1e-30, 1e-12, 1e12, 1e30)), (torch.bfloat16, (1e-30, 1e30)), (torch.float16, (1e-3, 1e3))):
        g = gradient(70, 90, torch.float32)
        for s in scales:
            h = (g * s).to(dtype)
            close(orthogonalize(h, eps=1e-38), formula(h, eps=1e-38), dtype, "%g" % s)


def test_zero_rank_one_and_repeated_rows():
    assert bool((orthogonalize(torch.zeros(40, 60, device=DEV)) == 0).all())
    g = torch.randn(50, 1, device=DEV) @ torch.randn(1, 80, device=DEV)
    close(orthogonalize(g), formula(g), torch.float32, "rank one", 20 * ITERATION)   # all other directions are noise
    g = gradient(40, 90, torch.float32)
    g[1::2] = g[0::2]
    g[10] = 0
    close(orthogonalize(g), formula(g), torch.float32, "repeated rows", 20 * ITERATION)


def test_smaller_than_eps_stays_small():
    g = gradient(30, 50, torch.float32)
    g = g / g.norm() * 1e-3
    close(orthogonalize(g, eps=1.0), formula(g, eps=1.0), torch.float32, "eps")


def test_not_a_number_stays_one():
    for bad in (float("nan"), float("inf")):
        mats = [gradient(40, 70, torch.float32), gradient(65, 30, torch.float32)]
        mats[0][3, 4] = bad
        outs = orthogonalize_many(mats)
        assert bool(torch.isnan(outs[0]).any())
        close(outs[1], formula(mats[1]), torch.float32, "the other matrix")


def test_strides_and_empty_matrices():
    g = gradient(90, 130, torch.bfloat16)
    views = [g[3:50, 7:100], g.t(), g[::2, ::3], g[:0], g[:, :0]]
    for v, o in zip(views, orthogonalize_many(views)):
        assert o.shape == v.shape
        if v.numel():
            close(o, formula(v), torch.bfloat16, "view")


def test_result_is_near_orthogonal():
    """Singular values from 0.02 of the norm on land in [0.6, 1.3] after five steps (p has no fixed point there, only a band)."""
    g = torch.randn(100, 400, device=DEV)
    s = torch.linalg.svdvals(orthogonalize(g).double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


def reference_step(p, g, m, lr, momentum=0.95, weight_decay=0.0, nesterov=True):
    m = momentum * m.double() + g.double()
    u = g.double() + momentum * m if nesterov else m
    scale = math.sqrt(max(1.0, p.size(0) / p.size(1)))
    return (1 - lr * weight_decay) * p.double() - lr * scale * formula(u), m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nesterov,weight_decay", [(True, 0.0), (False, 0.1)])
def test_step_against_the_formula(nesterov, weight_decay, dtype):
    shapes = [(30, 70), (70, 30), (1, 50), (128, 128), (9, 600)]
    ps = [gradient(m, n, dtype, 1) for m, n in shapes]
    ms = [gradient(m, n, torch.float32, 2) for m, n in shapes]
    lr = 0.05
    for turn in range(3):
        gs = [gradient(m, n, dtype, 3 + turn) for m, n in shapes]
        want = [reference_step(p, g, m, lr, 0.9, weight_decay, nesterov) for p, g, m in zip(ps, gs, ms)]
        muon_step_(ps, gs, ms, lr=lr, momentum=0.9, weight_decay=weight_decay, nesterov=nesterov)
        for p, m, (wp, wm) in zip(ps, ms, want):
            off = (p.double() - wp).abs()
            scale = lr * math.sqrt(max(1.0, p.size(0) / p.size(1)))
            # a row or column alone: the iteration's error is all in one direction, as large as its norm
            bound = (HALF_STEP[dtype] + 2.0 ** -23) * wp.abs() + scale * (4 * ITERATION) + 2.0 ** -25
            assert bool((off <= bound).all())
            assert bool(((m.double() - wm).abs() <= 2.0 ** -22 * (wm.abs() + 0.1)).all())


def test_captured_and_replayed():
    shapes = [(30, 70), (70, 30), (128, 200)]
    start = [gradient(m, n, torch.float32, 1) for m, n in shapes]
    gs = [gradient(m, n, torch.float32, 2) for m, n in shapes]
    held = [t.clone() for t in start]
    ms = [torch.zeros_like(t) for t in start]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        muon_step_([t.clone() for t in held], gs, [m.clone() for m in ms], lr=0.02)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step_(held, gs, ms, lr=0.02)
    eager, em = [t.clone() for t in start], [torch.zeros_like(t) for t in start]
    for t, s in zip(held, start):
        t.copy_(s)
    for m in ms:
        m.zero_()
    for turn in range(4):
        for g in gs:
            g.mul_(-0.7)
        graph.replay()
        torch.cuda.synchronize()
        muon_step_(eager, gs, em, lr=0.02)
        for a, b in zip(held + ms, eager + em):
            assert torch.equal(a, b)


def test_on_another_stream():
    g = gradient(300, 500, torch.float32)
    want = orthogonalize(g)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = orthogonalize(g)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


def test_optimizer_over_a_module():
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3), torch.nn.ReLU(), torch.nn.Conv2d(8, 6, 3), torch.nn.Flatten(),
                              torch.nn.Linear(6 * 16, 5)).to(DEV)
    net[2] = net[2].to(memory_format=torch.channels_last)
    opt = Muon(net.parameters(), lr=0.02, sgd_lr=0.1, weight_decay=0.01)
    momenta = {}
    for _ in range(3):
        opt.zero_grad()
        net(torch.randn(2, 3, 8, 8, device=DEV)).square().sum().backward()
        want = {}
        for p in net.parameters():
            m = momenta.get(p, torch.zeros_like(p)).double()
            if p.dim() >= 2:
                flat, gflat = p.detach().reshape(p.size(0), -1), p.grad.reshape(p.size(0), -1)
                w, m = reference_step(flat, gflat, m.reshape(flat.shape), 0.02, 0.95, 0.01)
                w, m = w.reshape(p.shape), m.reshape(p.shape)
            else:
                m = 0.9 * m + p.grad.double() + 0.01 * p.detach().double()
                w = p.detach().double() - 0.1 * m
            want[p], momenta[p] = w, m.float()
        opt.step()
        for p in net.parameters():
            assert float((p.detach().double() - want[p]).abs().max()) <= 1e-3 * 0.02 + 2.0 ** -22 * float(want[p].abs().max())
    net[0] = net[0].to(memory_format=torch.channels_last)      # in the middle of training
    opt.zero_grad()
    net(torch.randn(2, 3, 8, 8, device=DEV)).square().sum().backward()
    p = net[0].weight
    w, _ = reference_step(p.detach().reshape(8, -1), p.grad.reshape(8, -1), momenta[p].reshape(8, -1), 0.02, 0.95, 0.01)
    opt.step()
    assert float((p.detach().reshape(8, -1).double() - w).abs().max()) <= 1e-3 * 0.02 + 2.0 ** -22
    saved = opt.state_dict()
    other = Muon(net.parameters(), lr=0.02, sgd_lr=0.1, weight_decay=0.01)
    other.load_state_dict(saved)
    for p in net.parameters():
        assert torch.equal(other.state[p]["momentum_buffer"], opt.state[p]["momentum_buffer"])
