"""How much memory the loss asks for, from the library's own size functions."""
import ctypes

import pytest

from detectron_pytorch_amd import _lib

MB = 1 << 20
F32, F16, BF16 = _lib.TYPE_F32, _lib.TYPE_F16, _lib.TYPE_BF16


def sizes(rows, dim, classes, dtype):
    h = _lib.lib()
    kept = h.mi_linear_cross_entropy_saved_bytes(rows, dim, classes, dtype, ctypes.c_void_p(4096), dim)
    forward = h.mi_linear_cross_entropy_workspace_bytes(rows, dim, classes, dtype, _lib.PASS_FORWARD_PRED)
    backward = h.mi_linear_cross_entropy_workspace_bytes(rows, dim, classes, dtype, _lib.PASS_BACKWARD)
    assert kept and forward and backward
    return kept, forward, backward


@pytest.mark.parametrize("rows,dim,classes,dtype", [
    (8192, 4096, 50021, BF16), (8192, 4096, 50021, F32), (1024, 4096, 50021, BF16), (1024, 1024, 200000, F16),
    (4096, 1001, 250000, F16), (16384, 16, 20010, F32), (30000, 64, 20010, BF16), (300, 64, 1 << 18, BF16), (100000, 128, 1000, F32)])
def test_less_than_float32_logits(hip_lib_path, rows, dim, classes, dtype):
    """What is kept for the backward and the larger workspace, together, where there are logits of 200 MB and more."""
    kept, forward, backward = sizes(rows, dim, classes, dtype)
    logits = 4 * rows * classes
    assert logits > 2e8 and kept + max(forward, backward) < logits


@pytest.mark.parametrize("rows,dim,classes,dtype", [
    (512, 4096, 50000, F32), (1, 4096, 1 << 24, F32), (7, 1 << 14, 1 << 20, F32), (64, 1001, 1 << 20, F16), (1024, 1024, 81, F32),
    (777, 1001, 5003, F16), (8192, 4096, 50021, BF16), (8192, 4096, 50021, F32), (1 << 20, 64, 81, BF16), (100000, 1024, 100, F16)])
def test_bounds(hip_lib_path, rows, dim, classes, dtype):
    """Laid-out features, 128 MB of laid-out weights; q of 256 MB or as much as dx in float32 would be, 32 MB of slices or dx in
    float32, a weight gradient's slices of 32 MB, and sums of an eighth of q (the forward: 12 bytes for every 32 logits)."""
    kept, forward, backward = sizes(rows, dim, classes, dtype)
    rows_p, dim_p = -rows % 64 + rows, -dim % 64 + dim
    dx = 4 * rows * dim
    small = MB + 32 * rows_p
    assert kept <= rows_p * dim_p * (4 if dtype == F32 else 2) + 128 * MB + small
    assert forward <= 128 * MB + 12 * rows_p * (classes / 32 + 8) + small
    assert backward <= 1.125 * (256 * MB + dx) + max(32 * MB, dx) + 32 * MB + 128 * MB + small


def test_a_longer_vocabulary_takes_no_more(hip_lib_path):
    for dtype in (F32, F16, BF16):
        some = [sizes(2048, 1024, classes, dtype) for classes in (200000, 400000, 1600000)]
        for kept, _, backward in some[1:]:
            assert kept == some[0][0] and backward <= 1.25 * some[0][2]
