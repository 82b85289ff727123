"""What the classifier loss, the orthogonalisation and the optimiser step refuse: checked without a GPU."""
import ctypes

import pytest
import torch

from detectron_pytorch_amd import _lib
from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy
from detectron_pytorch_amd.muon import Muon, _check_apart, as_matrix, muon_step_
from detectron_pytorch_amd.orthogonalize import orthogonalize, orthogonalize_many, polynomial

NULL = ctypes.c_void_p(0)
SOME = ctypes.c_void_p(4096)   # an address that a refused call never touches


def ints(*v):
    return (ctypes.c_int * len(v))(*v)


def floats(*v):
    return (ctypes.c_float * len(v))(*v)


def test_cpu_tensors_are_refused(hip_lib_path):
    with pytest.raises(NotImplementedError):
        linear_cross_entropy(torch.zeros(2, 3), torch.zeros(4, 3), None, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(NotImplementedError):
        orthogonalize(torch.zeros(2, 3))
    with pytest.raises(NotImplementedError):
        muon_step_([torch.zeros(2, 3)], [torch.zeros(2, 3)], [torch.zeros(2, 3)], lr=0.1)
    assert orthogonalize_many([]) == []
    assert muon_step_([], [], [], lr=0.1) is None
    with pytest.raises(ValueError):
        muon_step_([torch.zeros(2, 3)], [], [], lr=0.1)


def test_coefficients_are_three():
    assert list(polynomial([1, 2.5, -3])) == [1.0, 2.5, -3.0]
    for bad in ((), (1.0, 2.0), (1.0, 2.0, 3.0, 4.0)):
        with pytest.raises(ValueError):
            polynomial(bad)


def test_optimizer_arguments():
    p = torch.nn.Parameter(torch.zeros(3, 4))
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(sgd_lr=-0.1), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            Muon([p], **bad)
    Muon([p]).step()   # no gradient: nothing to do


def test_biases_take_the_sgd_step():
    torch.manual_seed(0)
    ours, theirs = (torch.nn.Parameter(torch.randn(7)) for _ in range(2))
    theirs.data.copy_(ours.data)
    a = Muon([ours], lr=0.3, sgd_lr=0.1, weight_decay=0.01)
    b = torch.optim.SGD([theirs], lr=0.1, momentum=0.9, weight_decay=0.01)
    for _ in range(4):
        g = torch.randn(7)
        ours.grad, theirs.grad = g.clone(), g.clone()
        a.step()
        b.step()
        assert torch.allclose(ours, theirs, rtol=0, atol=2.0 ** -20)


def test_momenta_stay_float32_through_a_checkpoint():
    p = torch.nn.Parameter(torch.randn(7).bfloat16())
    opt = Muon([p], lr=0.3)
    p.grad = torch.randn(7).bfloat16() / 3
    opt.step()
    opt.step()
    buf = opt.state[p]["momentum_buffer"]
    assert buf.dtype == torch.float32
    q = torch.nn.Parameter(p.detach().clone())
    other = Muon([q], lr=0.3)
    other.load_state_dict(opt.state_dict())
    assert other.state[q]["momentum_buffer"].dtype == torch.float32
    assert torch.equal(other.state[q]["momentum_buffer"], buf) and other.state[q]["momentum_buffer"] is not buf
    q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert torch.equal(p, q)


def test_momentum_follows_the_parameters_memory_format():
    w = torch.nn.Parameter(torch.randn(4, 3, 2, 2))
    opt = Muon([w], orthogonalize=False)
    w.grad = torch.randn(4, 3, 2, 2)
    opt.step()
    before = opt.state[w]["momentum_buffer"].clone()
    w.data = w.data.contiguous(memory_format=torch.channels_last)
    assert torch.equal(opt._momentum(w), before) and opt._momentum(w).stride() == w.stride()
    empty = torch.nn.Parameter(torch.zeros(0, 5))
    empty.grad = torch.zeros(0, 5)
    Muon([empty]).step()
    assert as_matrix(empty).shape == (0, 0)


def test_as_matrix():
    w = torch.arange(2 * 3 * 4 * 5.0).view(2, 3, 4, 5)
    assert torch.equal(as_matrix(w), w.view(2, 60)) and as_matrix(w).data_ptr() == w.data_ptr()
    c = w.contiguous(memory_format=torch.channels_last)
    assert as_matrix(c).is_contiguous() and as_matrix(c).data_ptr() == c.data_ptr()
    assert torch.equal(as_matrix(c), w.permute(0, 2, 3, 1).reshape(2, 60))
    assert as_matrix(w.transpose(0, 1)) is None


def test_tensors_of_a_step_share_no_memory():
    flat, grad = torch.zeros(24), torch.zeros(24)
    a, b, c = flat[:8], flat[8:16], flat[15:24]
    _check_apart([b, a], [grad[:8], grad[4:12], torch.zeros(1).expand(8)])   # gradients may share memory among themselves
    _check_apart([a, torch.zeros(0), flat[3:3]], [flat[8:]])
    for written, read in (([a, a], []), ([b, c], []), ([c, b], []), ([flat, b], []), ([b], [flat[9:10]]), ([b], [flat]),
                          ([flat], [b]), ([a, b], [flat.view(2, 12).t()])):
        with pytest.raises(ValueError):
            _check_apart(written, read)


def test_loss_arguments_at_the_boundary(hip_lib_path):
    h = _lib.lib()

    def forward(x=SOME, w=SOME, y=SOME, rows=4, dim=8, classes=5, dtype=0, xs=8, ws=8, reduction=1, loss=SOME, saved=SOME,
                saved_bytes=1 << 30, room=SOME, room_bytes=1 << 30):
        return h.mi_linear_cross_entropy_forward(x, xs, w, ws, NULL, y, 1, rows, dim, classes, dtype, -1, reduction, loss, NULL,
                                                 saved, saved_bytes, room, room_bytes, NULL)

    for bad in (dict(x=NULL), dict(w=NULL), dict(y=NULL), dict(loss=NULL), dict(saved=NULL), dict(room=NULL), dict(rows=0),
                dict(rows=-1), dict(rows=1 << 25), dict(dim=0), dict(classes=0), dict(classes=1 << 25),
                dict(rows=1 << 24, classes=1 << 24), dict(rows=1 << 19, classes=1 << 18), dict(dtype=3),
                dict(dtype=-1), dict(xs=7), dict(ws=7), dict(ws=1 << 23), dict(reduction=3), dict(reduction=-1),
                dict(saved=ctypes.c_void_p(4100)), dict(room=ctypes.c_void_p(4100))):
        assert forward(**bad) == 1 and b"linear_cross_entropy" in h.mi_last_error(), bad
    for bad in (dict(saved_bytes=16), dict(room_bytes=16)):
        assert forward(**bad) == 3 and b"needed" in h.mi_last_error(), bad
    assert h.mi_linear_cross_entropy_backward(NULL, SOME, 8, NULL, 4, 8, 5, 0, 1, NULL, NULL, NULL, SOME, 1 << 30, SOME, 1 << 30,
                                              NULL) == 1
    assert h.mi_linear_cross_entropy_backward(SOME, SOME, 8, NULL, 4, 8, 5, 0, 1, NULL, NULL, NULL, SOME, 1 << 30, SOME, 8,
                                              NULL) == 3
    for gx, gw in ((ctypes.c_void_p(4104), NULL), (NULL, ctypes.c_void_p(4098))):
        assert h.mi_linear_cross_entropy_backward(SOME, SOME, 8, NULL, 4, 8, 5, 0, 1, gx, gw, NULL, SOME, 1 << 30, SOME, 1 << 30,
                                                  NULL) == 1
    assert h.mi_linear_cross_entropy_saved_bytes(0, 8, 5, 0, SOME, 8) == 0
    # 16-bit weights that can be multiplied where they lie are not kept a second time
    in_place = h.mi_linear_cross_entropy_saved_bytes(4, 64, 5000, 2, ctypes.c_void_p(4096), 64)
    assert in_place < 64 * 5000 < h.mi_linear_cross_entropy_saved_bytes(4, 64, 5000, 2, ctypes.c_void_p(4098), 64)


def test_workspace_stays_bounded(hip_lib_path):
    h = _lib.lib()
    # 1 GB of q for one piece of the vocabulary and an eighth of that around it, whatever the vocabulary
    for classes in (20000, 160000, 1600000):
        assert h.mi_linear_cross_entropy_workspace_bytes(8192, 64, classes, 2, _lib.PASS_BACKWARD) < (1152 << 20)


def test_matrix_arguments_at_the_boundary(hip_lib_path):
    h = _lib.lib()
    one = (ctypes.c_void_p * 1)(4096)
    none = (ctypes.c_void_p * 1)(0)
    usual = floats(3.4445, -4.7750, 2.0315)

    def call(count=1, a=one, b=one, rows=ints(4), cols=ints(6), dtype=0, steps=5, c=usual, eps=1e-7, room=SOME, size=1 << 30):
        return h.mi_orthogonalize(count, a, b, rows, cols, dtype, steps, c, eps, room, size, NULL)

    for bad in (dict(count=0), dict(rows=ints(0)), dict(cols=ints(-3)), dict(rows=ints(1 << 23)), dict(a=none), dict(b=none),
                dict(rows=ints(70000), cols=ints(70000)), dict(dtype=4), dict(steps=0), dict(steps=65), dict(eps=0.0),
                dict(room=NULL), dict(room=ctypes.c_void_p(4104)), dict(c=NULL)):
        assert call(**bad) == 1 and h.mi_last_error(), bad
    assert call(size=64) == 3
    for c in (floats(40.0, 0.0, 0.0), floats(3.0, 3.0, 3.0), floats(1.0, -900.0, 0.0), floats(float("nan"), 0.0, 0.0)):
        assert call(c=c) == 4 and b"coefficients" in h.mi_last_error()
    # the range of the iteration, found by sampling its singular values: taken or refused as that says, but for a narrow strip
    g = torch.Generator().manual_seed(0)
    seen = set()
    for _ in range(300):
        c = (torch.rand(3, generator=g) * 12 - 6).tolist()
        c = floats(*c)
        s, x, f = torch.linspace(0, 1, 4001, dtype=torch.float64), 0.0, 0.0
        for _ in range(3):
            factor = c[0] + c[1] * s ** 2 + c[2] * s ** 4
            top = float((s * factor).abs().max())
            x, f = max(x, top), max(f, float(factor.abs().max()))
            s = torch.linspace(0, top, 4001, dtype=torch.float64)
        if abs(max(x / 2.8, f / 60.0) - 1) > 0.01:
            rc = call(c=c, steps=3, size=64)
            seen.add(rc)
            assert rc == (3 if max(x / 2.8, f / 60.0) < 1 else 4), list(c)
    assert seen == {3, 4}
    assert h.mi_muon_step(1, one, one, NULL, ints(4), ints(6), 0, 0.1, 0.9, 1, 0.0, 5, usual, 1e-7, SOME, 1 << 30, NULL) == 1
    assert h.mi_muon_step(1, one, one, none, ints(4), ints(6), 0, 0.1, 0.9, 1, 0.0, 5, usual, 1e-7, SOME, 1 << 30, NULL) == 1
    assert h.mi_orthogonalize_workspace_bytes(1, ints(0), ints(3)) == 0
