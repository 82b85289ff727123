"""Orthogonalised matrices by Newton-Schulz products -- host side of mi_orthogonalize.

    orthogonalize(g)            one matrix [m, n]
    orthogonalize_many([...])   matrices of any sizes, one type, every stage of all of them in one launch

X = G / max(|G|_F, eps), then `steps` times X <- a X + b (X X^T) X + c (X X^T)^2 X (on G^T when G has more rows than
columns): the singular vectors of G with singular values near 1, what an orthogonalised weight update applies
(muon.Muon).  float32, float16 or bfloat16 matrices; products carry 22 bits and accumulate in float32, and only the result
is rounded to the type.
"""
import ctypes

import torch

from . import _lib

TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # steep at 0, within (0.68, 1.21) after five steps from there on
STEPS = 5
EPS = 1e-7


def check_matrices(mats, what):
    """The matrices' common device and type; raises for what mi_orthogonalize does not take."""
    for t in mats:
        _lib.require_cuda(t, what)
        if t.dim() != 2 or t.dtype not in TYPES or t.dtype != mats[0].dtype or t.device != mats[0].device:
            raise ValueError("%s must be 2-D float32, float16 or bfloat16 tensors of one type on one device, got %s %s on %s"
                             % (what, t.dtype, tuple(t.shape), t.device))
    return mats[0].device, TYPES[mats[0].dtype]


def host_arrays(mats):
    """(count, rows, cols) of non-empty matrices as the C side takes them."""
    n = len(mats)
    for t in mats:
        if max(t.shape) > 1 << 22:   # (checked here too: a C int takes sizes modulo 2^32)
            raise ValueError("matrices have sides of up to 2^22, got %s" % (tuple(t.shape),))
    return n, (ctypes.c_int * n)(*[t.size(0) for t in mats]), (ctypes.c_int * n)(*[t.size(1) for t in mats])


def pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def polynomial(coefficients):
    """(a, b, c) as the C side takes them."""
    coefficients = [float(c) for c in coefficients]
    if len(coefficients) != 3:
        raise ValueError("coefficients are (a, b, c), got %d numbers" % len(coefficients))
    return (ctypes.c_float * 3)(*coefficients)


def workspace_for(count, rows, cols, device):
    n = _lib.lib().mi_orthogonalize_workspace_bytes(count, rows, cols)
    if n == 0:
        _lib.check(1, "mi_orthogonalize_workspace_bytes")
    return torch.empty((n,), dtype=torch.uint8, device=device)


@torch.no_grad()
def orthogonalize_many(mats, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS):
    """The orthogonalised matrices, in the order and of the shapes given.  Asynchronous on the current stream; capturable."""
    mats = list(mats)
    if not mats:
        return []
    dev, dtype = check_matrices(mats, "matrices")
    outs = [torch.empty(t.shape, dtype=t.dtype, device=dev) for t in mats]
    full = [(t.contiguous(), o) for t, o in zip(mats, outs) if t.numel()]
    if not full:
        return outs
    ins, results = [t for t, _ in full], [o for _, o in full]
    count, rows, cols = host_arrays(ins)
    with torch.cuda.device(dev):
        workspace = workspace_for(count, rows, cols, dev)
        rc = _lib.lib().mi_orthogonalize(count, pointers(ins), pointers(results), rows, cols, dtype, int(steps),
                                         polynomial(coefficients), float(eps), workspace.data_ptr(), workspace.numel(),
                                         _lib.current_stream_handle(dev))
    _lib.check(rc, "mi_orthogonalize")
    return outs


def orthogonalize(g, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS):
    """The orthogonalised matrix `g` [m, n], in its type."""
    return orthogonalize_many([g], steps, coefficients, eps)[0]
