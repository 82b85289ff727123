"""Optimiser with momentum and orthogonalised updates for weight matrices -- host side of mi_muon_step.

    muon_step_(params, grads, momenta, lr=...)   one step of a list of matrices, in place
    Muon(params, lr=...)                         the torch.optim.Optimizer around it (rcnn.train.make_optimizer: SOLVER.TYPE)

Per matrix:  M <- mu M + G,  U = G + mu M (nesterov) or M,
             W <- (1 - lr weight_decay) W - lr sqrt(max(1, rows / cols)) orthogonalize(U).
A convolution's weight [out, in, kh, kw] is the matrix [out, in kh kw].  What is no matrix (biases) takes the momentum SGD step
of torch.optim.SGD, with its own learning rate.
"""
import torch

from . import _lib
from .orthogonalize import COEFFICIENTS, EPS, STEPS, check_matrices, host_arrays, pointers, polynomial, workspace_for


def _check_apart(written, read):
    """Refuses tensors of `written` (contiguous) that share memory with one another or with one of `read`."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), True) for t in written if t.numel()]
    for t in read:
        if t.numel():
            last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
            spans.append((t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size(), False))
    spans.sort()
    end, end_written = 0, 0   # of what came before
    for first, behind, is_written in spans:
        if first < (end if is_written else end_written):
            raise ValueError("a parameter or momentum shares memory with another tensor of the step")
        end = max(end, behind)
        if is_written:
            end_written = max(end_written, behind)


@torch.no_grad()
def muon_step_(params, grads, momenta, lr, momentum=0.95, weight_decay=0.0, nesterov=True, steps=STEPS,
               coefficients=COEFFICIENTS, eps=EPS):
    """One step of contiguous matrices `params` (float32, float16 or bfloat16) with `grads` of their type and shapes and
    float32 `momenta`, which are updated too.  Asynchronous on the current stream; capturable (the numbers are the
    captured ones)."""
    params, grads, momenta = list(params), list(grads), list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError("muon_step_ takes as many gradients and momenta as parameters")
    if not params:
        return
    dev, dtype = check_matrices(params, "params")
    for p, g, m in zip(params, grads, momenta):
        _lib.require_cuda(g, "grads")
        _lib.require_cuda(m, "momenta")
        if g.shape != p.shape or m.shape != p.shape or g.dtype != p.dtype or m.dtype != torch.float32:
            raise ValueError("a gradient has its parameter's shape and type, a momentum its shape in float32")
        if g.device != dev or m.device != dev:
            raise ValueError("muon_step_ takes tensors on one device")
        if not (p.is_contiguous() and m.is_contiguous()):
            raise ValueError("parameters and momenta are updated in place: they must be contiguous")
    _check_apart(params + momenta, grads)
    full = [(p, g.contiguous(), m) for p, g, m in zip(params, grads, momenta) if p.numel()]
    if not full:
        return
    ps, gs, ms = zip(*full)
    count, rows, cols = host_arrays(ps)
    with torch.cuda.device(dev):
        workspace = workspace_for(count, rows, cols, dev)
        rc = _lib.lib().mi_muon_step(count, pointers(ps), pointers(gs), pointers(ms), rows, cols, dtype, float(lr),
                                     float(momentum), int(nesterov), float(weight_decay), int(steps),
                                     polynomial(coefficients), float(eps), workspace.data_ptr(), workspace.numel(),
                                     _lib.current_stream_handle(dev))
    _lib.check(rc, "mi_muon_step")
    # written through their addresses: a backward over a graph from before the step has to see it, as after torch's own optimisers
    torch.autograd.graph.increment_version([t for t in ps + ms if not t.is_inference()])


def as_matrix(t):
    """A dense parameter of two or more dimensions as a contiguous matrix [out, rest] over the same memory, None for other
    layouts.  A channels-last weight is the matrix with its columns in memory order: orthogonalisation does not depend on the
    order of columns."""
    rows = t.size(0)
    cols = t.numel() // rows if rows else 0
    if t.is_contiguous():
        return t.view(rows, cols)
    if t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last):
        return t.permute(0, 2, 3, 1).reshape(rows, cols)
    return None


def _same_order(t, like):
    """Whether `t` lies in memory as `like` does (dimensions of one element aside)."""
    return (t.is_contiguous() and like.is_contiguous()) or t.stride() == like.stride()


def _is_captured(p):
    return p.is_cuda and torch.cuda.is_current_stream_capturing()


class Muon(torch.optim.Optimizer):
    """Parameters of two or more dimensions take the orthogonalised step with `lr`, the others momentum SGD with `sgd_lr`
    (lr when None) and `sgd_momentum`.  Per group as usual: {"params": ..., "lr": ..., "sgd_lr": ..., "weight_decay": ...};
    "orthogonalize": False keeps a group's matrices on SGD too.  Momenta are float32, whatever the parameter's type.  A step can be
    captured into a graph after one that ran (which made the momenta)."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, sgd_lr=None, sgd_momentum=0.9,
                 steps=STEPS, coefficients=COEFFICIENTS, eps=EPS, orthogonalize=True):
        if lr < 0 or (sgd_lr is not None and sgd_lr < 0) or weight_decay < 0 or not 0 <= momentum < 1 or not 0 <= sgd_momentum < 1:
            raise ValueError("learning rates and weight decay are at least 0, momenta in [0, 1)")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, sgd_lr=sgd_lr,
                                      sgd_momentum=sgd_momentum, steps=steps, coefficients=tuple(coefficients), eps=eps,
                                      orthogonalize=orthogonalize))

    def _momentum(self, p):
        state = self.state[p]
        buf = state.get("momentum_buffer")
        if buf is not None and _same_order(buf, p):
            return buf
        if _is_captured(p):   # every replay would make it anew
            raise RuntimeError("a step of Muon is captured after one that ran: momenta are made outside of a graph")
        if buf is None:
            buf = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        else:   # the parameter was given another memory format
            buf = torch.empty_like(p, dtype=torch.float32).copy_(buf)
        state["momentum_buffer"] = buf
        return buf

    def load_state_dict(self, state_dict):
        """As torch's, which gives states their parameter's type; momenta keep their own."""
        super().load_state_dict(state_dict)
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], saved["params"]):
                buf = state_dict["state"].get(key, {}).get("momentum_buffer")
                if buf is not None:
                    self.state[p]["momentum_buffer"] = torch.empty_like(p, dtype=torch.float32).copy_(buf)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            matrices, others = {}, {}
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("Muon does not take sparse gradients")
                if group["orthogonalize"] and p.dim() >= 2:
                    if as_matrix(p) is None:
                        raise ValueError("Muon updates dense parameters (contiguous or channels-last), got strides %s"
                                         % (p.stride(),))
                    grad = p.grad if _same_order(p.grad, p) else torch.empty_like(p).copy_(p.grad)
                    mats = matrices.setdefault((p.device, p.dtype), ([], [], []))
                    for to, t in zip(mats, (p, grad, self._momentum(p))):
                        to.append(as_matrix(t))
                else:
                    for to, t in zip(others.setdefault((p.device, p.dtype), ([], [], [])), (p, p.grad, self._momentum(p))):
                        to.append(t)
            for params, grads, momenta in matrices.values():
                muon_step_(params, grads, momenta, lr=group["lr"], momentum=group["momentum"],
                           weight_decay=group["weight_decay"], nesterov=group["nesterov"], steps=group["steps"],
                           coefficients=group["coefficients"], eps=group["eps"])
            for params, grads, momenta in others.values():
                _sgd_step_(params, grads, momenta, group["lr"] if group["sgd_lr"] is None else group["sgd_lr"],
                           group["sgd_momentum"], group["weight_decay"])
        return loss


def _sgd_step_(params, grads, momenta, lr, momentum, weight_decay):
    """torch.optim.SGD's momentum step (coupled weight decay, no dampening) of a list, with float32 momenta."""
    grads = [g.float() for g in grads]
    torch._foreach_mul_(momenta, momentum)
    torch._foreach_add_(momenta, grads)
    if weight_decay:
        torch._foreach_add_(momenta, [p.float() for p in params], alpha=weight_decay)
    if params[0].dtype in (torch.float32, torch.float64):
        torch._foreach_add_(params, momenta, alpha=-lr)
    else:   # rounded once
        for p, m in zip(params, momenta):
            p.copy_(p.float() - lr * m)
