"""Optimizer of matrix-shaped parameters: updates orthogonalised by Newton-Schulz products (Muon).

``newton_schulz`` orthogonalises a matrix, a stack of matrices or a list of them; ``Muon`` is the optimizer, whose whole step
over all matrices of a model - momentum, orthogonalisation, decay and update - is one call of the library
(step_newton_schulz).  The reference trains with Adam and SGD only (classifier_stgcn_real_only/utils/processor.py:240-255)."""
import math

import torch

from . import _lib

STEPS = 5
EPS = 1e-7


def _run(items, dtype, device, steps, eps, momentum=0.0, nesterov=False, lr=0.0, decay=0.0):
    arr = (_lib.NsItem * len(items))(*items)
    nb = _lib.query("step_newton_schulz_ws_bytes", arr, len(items))
    if not nb:
        raise _lib.StepHipError("newton_schulz: %s" % _lib.load().step_last_error().decode())
    ws = torch.empty(nb, dtype=torch.uint8, device=device)
    _lib.call("step_newton_schulz", arr, len(items), dtype, steps, eps, momentum, int(nesterov), lr, decay, ws, nb)


def _checked(steps, eps):
    if not isinstance(steps, int) or not 1 <= steps <= 100:
        raise _lib.StepHipError("newton_schulz: 1 to 100 steps, got %r" % (steps,))
    if not float(eps) >= 0.0:
        raise _lib.StepHipError("newton_schulz: eps %r" % (eps,))
    return steps, float(eps)


def newton_schulz(g, steps=STEPS, eps=EPS):
    """The Newton-Schulz orthogonalisation of g (..., m, n), or of every tensor of a list: from X = g / (|g|_F + eps), `steps`
    times X <- a X + (b A + c A A) X with A = X X^T and (a, b, c) = (3.4445, -4.7750, 2.0315) (on the transpose where m > n),
    which drives all singular values towards 1.  float32, bfloat16 or float16; the result has g's shape and type and is
    rounded once: the products are held to fp32's accuracy for every type.  A zero matrix stays zero.  Not differentiable.
    The tensors of a list have one type and one device; small matrices of a list (min(m, n) <= 64) share their launches."""
    steps, eps = _checked(steps, eps)
    many = isinstance(g, (list, tuple))
    gs = list(g) if many else [g]
    if not gs:
        return []
    outs, items, keep = [], [], []
    for t in gs:
        if not isinstance(t, torch.Tensor) or t.dim() < 2:
            raise _lib.StepHipError("newton_schulz: matrices (..., m, n) wanted, got %s" % (
                tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__,))
        if t.dtype not in _lib.DTYPES:
            raise _lib.StepHipError("newton_schulz: float32, bfloat16 or float16 wanted, got %s" % t.dtype)
        if t.dtype != gs[0].dtype or t.device != gs[0].device:
            raise _lib.StepHipError("newton_schulz: a list has one type and one device, got %s on %s and %s on %s" % (
                gs[0].dtype, gs[0].device, t.dtype, t.device))
        if t.numel() > 0 and (max(t.shape[-2:]) > 1 << 21 or t.numel() // (t.shape[-2] * t.shape[-1]) > 1 << 24):
            raise _lib.StepHipError("newton_schulz: %s: 2^21 rows or columns and 2^24 matrices at most" % (tuple(t.shape),))
    for t in gs:
        if not t.is_cuda:
            raise _lib.StepHipError("step_amd kernels need tensors on the GPU (got device %s); there is no CPU path" % t.device)
        c = t.detach().contiguous()
        o = torch.empty_like(c)
        outs.append(o)
        if not c.numel():
            continue
        m, n = c.shape[-2:]
        keep.append(c)
        items.append((c.data_ptr(), o.data_ptr(), None, None, c.numel() // (m * n), m, n, 1.0))
    if items:
        _run(items, _lib.DTYPES[gs[0].dtype], gs[0].device, steps, eps)
    return outs if many else outs[0]


class Muon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates for the matrices of a model, Adam for everything else.

    For a parameter of two axes or more, as the matrix (shape[0], all others):

        buf <- momentum buf + grad,   u = grad + momentum buf (nesterov) or buf,   o = newton_schulz(u)
        p   <- p (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) o

    Parameters of one axis (biases, norms' weights) and those of a group with ``matrices=False`` take Adam steps with decoupled
    decay at ``adam_lr`` (default: lr), ``adam_betas``, ``adam_eps``.  All parameters are fp32, contiguous and on one GPU per
    step; those without a gradient are left alone.  The matrices' step is one library call, three launches for all matrices
    with a side of at most 64.  It may be captured into a graph once every matrix has had a step (lr and the other options are
    then those of the capture); Adam's part may not."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=STEPS, eps=EPS, adam_lr=None,
                 adam_betas=(0.9, 0.999), adam_eps=1e-8):
        if not lr >= 0.0 or not weight_decay >= 0.0 or not 0.0 <= momentum < 1.0:
            raise ValueError("lr %r, weight_decay %r, momentum %r" % (lr, weight_decay, momentum))
        if adam_lr is not None and not adam_lr >= 0.0:
            raise ValueError("adam_lr %r" % (adam_lr,))
        _checked(steps, eps)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, eps=eps,
                                      adam_lr=adam_lr, adam_betas=adam_betas, adam_eps=adam_eps, matrices=True))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            mats, rest = [], []
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise _lib.StepHipError("Muon: sparse gradients are not supported")
                (mats if group["matrices"] and p.dim() >= 2 and p.numel() else rest).append(p)
            if mats:
                self._step_matrices(group, mats)
            if rest:
                self._step_rest(group, rest)
        return loss

    def _step_matrices(self, group, mats):
        dev = mats[0].device
        for p in mats:
            g = p.grad
            if p.dtype is not torch.float32 or g.dtype is not torch.float32:
                raise _lib.StepHipError("Muon keeps fp32 parameters, got %s (gradient %s)" % (p.dtype, g.dtype))
            if not p.is_cuda:
                raise _lib.StepHipError("step_amd kernels need tensors on the GPU (got device %s); there is no CPU path" % p.device)
            if p.device != dev or g.device != dev:
                raise _lib.StepHipError("Muon: the parameters of a group lie on %s and %s" % (dev, p.device))
            if not p.is_contiguous():
                raise _lib.StepHipError("Muon: non-contiguous parameter of shape %s" % (tuple(p.shape),))
        if len({p.data_ptr() for p in mats}) != len(mats):       # two updates of one matrix at a time
            raise _lib.StepHipError("Muon: a group holds a parameter twice")
        items, keep, written = [], [], []
        for p in mats:
            state = self.state[p]
            buf = state.get("momentum_buffer")
            if buf is None:
                if torch.cuda.is_current_stream_capturing():     # (a replay would clear it again)
                    raise _lib.StepHipError("Muon: take one step before a capture, which makes the momentum buffers")
                buf = state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            elif buf.dtype is not torch.float32 or buf.shape != p.shape or buf.device != dev or not buf.is_contiguous():
                raise _lib.StepHipError("Muon: momentum buffer %s %s does not fit its parameter" % (buf.dtype, tuple(buf.shape)))
            g = p.grad.contiguous()
            m = p.shape[0]
            n = p.numel() // m
            if max(m, n) > 1 << 21:
                raise _lib.StepHipError("Muon: a parameter of shape %s: 2^21 rows or columns at most" % (tuple(p.shape),))
            keep.append(g)
            written += (p, buf)
            items.append((g.data_ptr(), None, buf.data_ptr(), p.data_ptr(), 1, m, n, math.sqrt(m / n) if m > n else 1.0))
        _run(items, 0, dev, group["steps"], group["eps"], group["momentum"], group["nesterov"], group["lr"], group["weight_decay"])
        # written behind torch's back: caches and saved tensors go by the version
        torch.autograd.graph.increment_version(written)

    def _step_rest(self, group, rest):
        lr = group["lr"] if group["adam_lr"] is None else group["adam_lr"]
        b1, b2 = group["adam_betas"]
        if rest[0].is_cuda and torch.cuda.is_current_stream_capturing():
            raise _lib.StepHipError("Muon: Adam's corrections are counted on the host: only the matrices' step can be captured")
        grads, firsts, seconds = [p.grad for p in rest], [], []
        for p in rest:
            state = self.state[p]
            if "step" not in state:
                state["step"] = 0
                state["exp_avg"], state["exp_avg_sq"] = torch.zeros_like(p), torch.zeros_like(p)
            state["step"] += 1
            firsts.append(state["exp_avg"])
            seconds.append(state["exp_avg_sq"])
        if group["weight_decay"]:
            torch._foreach_mul_(rest, 1 - lr * group["weight_decay"])
        torch._foreach_lerp_(firsts, grads, 1 - b1)
        torch._foreach_mul_(seconds, b2)
        torch._foreach_addcmul_(seconds, grads, grads, 1 - b2)
        roots = torch._foreach_sqrt(seconds)
        torch._foreach_div_(roots, [math.sqrt(1 - b2 ** self.state[p]["step"]) for p in rest])
        torch._foreach_add_(roots, group["adam_eps"])
        torch._foreach_addcdiv_(rest, firsts, roots, [-lr / (1 - b1 ** self.state[p]["step"]) for p in rest])
