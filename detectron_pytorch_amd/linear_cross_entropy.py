"""Softmax cross entropy of a linear classifier without its logits in memory -- host side of mi_linear_cross_entropy_*.

`F.cross_entropy(F.linear(x, weight, bias), labels)` keeps [rows, classes] logits, their softmax and their gradient; at a
detector's 81 classes that is nothing, over a long list of classes it is most of the head's memory and traffic.  The HIP
kernels form the logits tile by tile on the matrix cores, in the forward and again in the backward, and keep per row
the log of the sum of exponentials only (reference of the plain form: lib/modeling/fast_rcnn_heads.py:39,57).  Memory: a copy of the
features, float32 or padded weights laid out anew (up to 128 MB, kept; more of them piece by piece), and in the backward a piece of
the softmax, up to 256 MB, with partial sums: 0.45 GB where float32 logits of 8192 rows and 50021 classes take 1.64.  At a few
dozen MB of logits there is nothing to save.

    loss = linear_cross_entropy(x, weight, bias, labels)                    # differentiable in x, weight, bias
    loss, pred = linear_cross_entropy(x, weight, bias, labels, with_pred=True)

x [rows, dim], weight [classes, dim], bias [classes] or None: all float32, all float16 or all bfloat16, on one GPU; labels int32
or int64 [rows].  Sums, softmax statistics and the loss are float32.  float32 products carry 22 bits of each factor down to 2^-18 of
the largest finite magnitude of its tensor, and one bit less per halving below that (an infinite factor makes its logits NaN).
Gradients take probabilities with the bits of their type (float32: 22) and as zero below 2^-39 (float32, float16).  With
reduction='none' that holds for each row of x's gradient by itself; in the weight's gradient, parts below 2^-38 of the largest row's are lost.
"""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib

TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
MOST_STRIDE = 1 << 22   # rows further apart are brought together first
REDUCTIONS = {"none": _lib.REDUCTION_NONE, "mean": _lib.REDUCTION_MEAN, "sum": _lib.REDUCTION_SUM}


def _check(x, weight, bias, labels, reduction):
    device, dtype = x.device, x.dtype
    for t, name in ((x, "x"), (weight, "weight"), (labels, "labels"), (bias, "bias")):
        if t is not None:
            _lib.require_cuda(t, name)
            if t.device != device:
                raise ValueError("linear_cross_entropy takes tensors on one device")
    if x.dim() != 2 or weight.dim() != 2 or x.size(1) != weight.size(1):
        raise ValueError("linear_cross_entropy takes x [rows, dim] and weight [classes, dim], got %s and %s"
                         % (tuple(x.shape), tuple(weight.shape)))
    if weight.numel() == 0:
        raise ValueError("linear_cross_entropy needs at least one class and one feature, got weight %s" % (tuple(weight.shape),))
    if max(x.size(0), weight.size(0)) > 1 << 24 or x.size(1) > 1 << 20:   # (checked here too: a C int takes sizes modulo 2^32)
        raise ValueError("linear_cross_entropy takes up to 2^24 rows and classes and 2^20 features, got x %s and weight %s"
                         % (tuple(x.shape), tuple(weight.shape)))
    if dtype not in TYPES or weight.dtype != dtype:
        raise ValueError("linear_cross_entropy takes float32, float16 or bfloat16 x and weight of one type, got %s and %s"
                         % (dtype, weight.dtype))
    if bias is not None and (bias.dtype != dtype or bias.shape != weight.shape[:1]):
        raise ValueError("bias must be %s [%d], got %s %s" % (dtype, weight.size(0), bias.dtype, tuple(bias.shape)))
    if (labels.dtype is not torch.int64 and labels.dtype is not torch.int32) or labels.shape != x.shape[:1]:
        raise ValueError("labels must be int32 or int64 [%d], got %s %s" % (x.size(0), labels.dtype, tuple(labels.shape)))
    if reduction not in REDUCTIONS:
        raise ValueError("reduction must be 'none', 'mean' or 'sum', got %r" % (reduction,))


def _rows(t):
    """`t` with contiguous rows that do not overlap, and the distance between them."""
    rows, cols = t.shape
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and not cols <= t.stride(0) <= MOST_STRIDE):
        t = t.contiguous()
    return t, (t.stride(0) if rows > 1 else cols)


def _unpacked(ctx, weight, bias, saved):
    """The saved tensors as the backward reads them, and the distance of the weight's rows.  Hooks on saved tensors
    (torch.autograd.graph.saved_tensors_hooks, save_on_cpu) may give back others: of other strides, at another address."""
    if (weight.data_ptr(), weight.stride(), saved.data_ptr()) == ctx.places and (bias is None or bias.is_contiguous()):
        return weight, ctx.w_stride, bias, saved
    weight, stride = _rows(weight)
    needed = _lib.lib().mi_linear_cross_entropy_saved_bytes(*ctx.shape, weight.data_ptr(), stride)
    if needed > saved.numel():   # the forward read it where it lay and kept no copy, which this place does not allow
        weight, stride = weight.clone(memory_format=torch.contiguous_format), weight.size(1)
    if saved.data_ptr() % 256 or not saved.is_contiguous():
        saved = saved.clone(memory_format=torch.contiguous_format)
    return weight, stride, None if bias is None else bias.contiguous(), saved


class _LinearCrossEntropy(Function):
    """`.apply(x, weight, bias_or_None, labels, ignore_index, reduction, with_pred)`; pred is not differentiable."""

    @staticmethod
    def forward(ctx, x, weight, bias, labels, ignore_index, reduction, with_pred):
        (x, x_stride), (weight, w_stride), labels = _rows(x), _rows(weight), labels.contiguous()
        bias = None if bias is None else bias.contiguous()
        rows, dim = x.shape
        classes, dtype, dev = weight.size(0), TYPES[x.dtype], x.device
        lib = _lib.lib()
        ctx.shape, ctx.reduction = (rows, dim, classes, dtype), reduction
        if rows == 0:   # nothing to launch
            ctx.save_for_backward(weight, bias, None)
            loss = torch.zeros((0,) if reduction == _lib.REDUCTION_NONE else (), dtype=torch.float32, device=dev)
            pred = torch.empty((0,), dtype=torch.int64, device=dev)
            ctx.mark_non_differentiable(pred)
            return (loss, pred) if with_pred else loss
        with torch.cuda.device(dev):
            loss = torch.empty((rows,) if reduction == _lib.REDUCTION_NONE else (), dtype=torch.float32, device=dev)
            pred = torch.empty((rows,), dtype=torch.int64, device=dev) if with_pred else None
            saved = torch.empty((lib.mi_linear_cross_entropy_saved_bytes(rows, dim, classes, dtype, weight.data_ptr(),
                                                                         w_stride),), dtype=torch.uint8, device=dev)
            ws_bytes = lib.mi_linear_cross_entropy_workspace_bytes(
                rows, dim, classes, dtype, _lib.PASS_FORWARD_PRED if with_pred else _lib.PASS_FORWARD)
            workspace = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
            rc = lib.mi_linear_cross_entropy_forward(
                x.data_ptr(), x_stride, weight.data_ptr(), w_stride, None if bias is None else bias.data_ptr(),
                labels.data_ptr(), int(labels.dtype == torch.int64), rows, dim, classes, dtype, ignore_index, reduction,
                loss.data_ptr(), pred.data_ptr() if with_pred else None, saved.data_ptr(), saved.numel(), workspace.data_ptr(),
                ws_bytes, _lib.current_stream_handle(dev))
        _lib.check(rc, "mi_linear_cross_entropy_forward")
        ctx.places, ctx.w_stride = (weight.data_ptr(), weight.stride(), saved.data_ptr()), w_stride
        ctx.save_for_backward(weight, bias, saved)
        if with_pred:
            ctx.mark_non_differentiable(pred)
            return loss, pred
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        weight, bias, saved = ctx.saved_tensors
        rows, dim, classes, dtype = ctx.shape
        dev = weight.device
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        if rows == 0:
            return (torch.zeros((0, dim), dtype=weight.dtype, device=dev) if want_x else None,
                    torch.zeros((classes, dim), dtype=weight.dtype, device=dev) if want_w else None,
                    torch.zeros((classes,), dtype=weight.dtype, device=dev) if want_b else None, None, None, None, None)
        lib = _lib.lib()
        with torch.cuda.device(dev):
            weight, w_stride, bias, saved = _unpacked(ctx, weight, bias, saved)
            grad_loss = grad_loss.contiguous().float()
            grad_x = torch.empty((rows, dim), dtype=weight.dtype, device=dev) if want_x else None
            grad_w = torch.empty((classes, dim), dtype=weight.dtype, device=dev) if want_w else None
            grad_b = torch.empty((classes,), dtype=weight.dtype, device=dev) if want_b else None
            ws_bytes = lib.mi_linear_cross_entropy_workspace_bytes(rows, dim, classes, dtype, _lib.PASS_BACKWARD)
            workspace = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
            rc = lib.mi_linear_cross_entropy_backward(
                grad_loss.data_ptr(), weight.data_ptr(), w_stride, None if bias is None else bias.data_ptr(), rows, dim,
                classes, dtype, ctx.reduction, grad_x.data_ptr() if want_x else None, grad_w.data_ptr() if want_w else None,
                grad_b.data_ptr() if want_b else None, saved.data_ptr(), saved.numel(), workspace.data_ptr(), ws_bytes,
                _lib.current_stream_handle(dev))
        _lib.check(rc, "mi_linear_cross_entropy_backward")
        return grad_x, grad_w, grad_b, None, None, None, None


def linear_cross_entropy(x, weight, bias, labels, ignore_index=-1, reduction="mean", with_pred=False):
    """Cross entropy of softmax(x weight^T + bias) against `labels`, float32.

    Rows with label `ignore_index` (the framework's padding rows: -1) count nowhere and get a zero gradient, whatever x holds
    there and the weight anywhere; 'mean' runs over the other rows and is 0 when there are none.  A label that is neither ignored nor a class makes
    its row's loss NaN.  `with_pred`: also the class of the largest logit per row (int64, lowest index of equal ones, -1
    for ignored rows).  The backward is captured into a graph or run eagerly like the forward: no host synchronisation."""
    _check(x, weight, bias, labels, reduction)
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index must be a label's value, got %r" % (ignore_index,))
    return _LinearCrossEntropy.apply(x, weight, bias, labels, int(ignore_index), REDUCTIONS[reduction], bool(with_pred))
