"""Training losses on the GPU.

The CVAE's with the reference's names and argument order:
``between_frame_loss(gait1, gait2, thres)`` (generator_cvae/utils/losses.py:7-42) and
``vae_loss(x_in, x_out, mean, lsig, beta)`` (generator_cvae/utils/processor_stgcn.py:34-40).
One HIP launch computes the value and every gradient (step_vae_loss); the reference spends
O(B*T*V*C) scalar mse_loss calls (~16 s per iteration in its logs) on the same number.

``policy_loss``: the clipped policy objective with a KL term over rows of logits, for fine-tuning a model on ratings of its
answers.  The reference has no counterpart."""
import torch

from . import _lib


class _VaeLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x_in, x_out, mean, lsig, beta):
        if x_in.dim() == 5:
            if x_in.shape[4] != 1:
                raise _lib.StepHipError("vae_loss expects M == 1 gaits (N,C,T,V,1)")
        elif x_in.dim() != 4:
            raise _lib.StepHipError("vae_loss expects (N,C,T,V[,1]) gaits, got %s" % (tuple(x_in.shape),))
        if x_in.shape != x_out.shape:
            raise _lib.StepHipError("x_in %s and x_out %s differ in shape" % (tuple(x_in.shape), tuple(x_out.shape)))
        N, C, T, V = x_in.shape[:4]
        xi = x_in.detach().float().contiguous()
        xo = x_out.detach().float().contiguous()
        dev = xo.device
        have_z = mean is not None
        Z = mean.shape[1] if have_z else 0
        m = mean.detach().float().contiguous() if have_z else None
        s = lsig.detach().float().contiguous() if have_z else None
        loss = torch.empty(3, dtype=torch.float32, device=dev)
        d_xo = torch.empty_like(xo)
        d_m = torch.empty_like(m) if have_z else None
        d_s = torch.empty_like(s) if have_z else None
        nb = _lib.query("step_vae_loss_ws_bytes", N)
        ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=dev)
        _lib.call("step_vae_loss", xi, xo, m, s, float(beta), loss, d_xo, d_m, d_s, N, C, T, V, Z, ws, nb)
        ctx.save_for_backward(d_xo, d_m, d_s)
        ctx.shape = tuple(x_out.shape)
        ctx.parts = loss
        return loss[0].clone()

    @staticmethod
    def backward(ctx, g):
        d_xo, d_m, d_s = ctx.saved_tensors
        need = ctx.needs_input_grad
        gxo = (d_xo * g).view(ctx.shape) if need[1] else None
        gxi = (-(d_xo * g)).view(ctx.shape) if need[0] else None
        gm = d_m * g if (need[2] and d_m is not None) else None
        gs = d_s * g if (need[3] and d_s is not None) else None
        return gxi, gxo, gm, gs, None


def between_frame_loss(gait1, gait2, thres=0.01):
    """losses.py:7-42 (``thres`` is unused in the reference as well)"""
    return _VaeLossFn.apply(gait1, gait2, None, None, 0.0)


def vae_loss(x_in, x_out, mean, lsig, beta=1.):
    """processor_stgcn.py:34-40: between_frame_loss(x_in, x_out) + beta * KLD"""
    return _VaeLossFn.apply(x_in, x_out, mean, lsig, beta)


class _PolicyLossFn(torch.autograd.Function):
    """The forward leaves the gradient for an upstream gradient of 1 behind (value and gradient take one pass over the
    logits); the backward hands it out, or computes it again from the logits where the upstream gradient is not 1 - on
    the device, with one rounding - or where a retained graph asks a second time.  A graph that holds the backward without its
    forward is replayed when the forward's memory may long be something else's: there it is computed anew from the caller's tensors,
    and where one of them had to be copied, whose copy is not the caller's to keep, refused."""

    @staticmethod
    def forward(ctx, logits, actions, old_logp, advantages, ref_logp, mask, clip_low, clip_high, beta, copied):
        classes = logits.shape[-1]
        rows = logits.numel() // classes
        z = logits.contiguous()
        loss = z.new_empty((), dtype=torch.float32)
        stats = z.new_empty(3, dtype=torch.float32)
        logp = z.new_empty(logits.shape[:-1], dtype=torch.float32)
        need = ctx.needs_input_grad[0]
        grad = torch.empty_like(z) if need else None
        ctx.mark_non_differentiable(logp, stats)
        ctx.config = (clip_low, clip_high, beta)
        nb = _lib.size("step_policy_loss_ws_bytes", rows, classes)
        ws = z.new_empty(nb, dtype=torch.uint8)
        if not rows:
            loss.zero_(), stats.zero_()
        else:
            _lib.call("step_policy_loss", z, actions, old_logp, advantages, ref_logp, mask, clip_low, clip_high, beta, None, 0,
                      loss, stats, logp, grad, rows, classes, _lib.DTYPES[z.dtype], ws, nb)
        if need:
            ctx.save_for_backward(z, actions, old_logp, advantages, ref_logp, mask)
            ctx.grad, ctx.ws, ctx.capture = grad, ws, _lib.capture(z.device)
            ctx.copied = copied or not logits.is_contiguous()
        return loss, logp, stats

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, g, _logp, _stats):
        z, actions, old_logp, advantages, ref_logp, mask = ctx.saved_tensors
        grad, ctx.grad = ctx.grad, None
        capture = _lib.capture(z.device)
        first = grad is not None and capture == ctx.capture
        ws = ctx.ws
        if not first:
            if ctx.copied and capture is not None and ctx.capture is None:
                raise _lib.StepHipError("policy_loss: a backward captured without its forward reads the forward's arguments at every "
                                        "replay: contiguous logits, int64 actions, fp32 and bool of one value a row wanted")
            grad, ws = torch.empty_like(z), torch.empty_like(ws)
        rows = z.numel() // z.shape[-1]
        if rows:
            _lib.call("step_policy_loss", z, actions, old_logp, advantages, ref_logp, mask, *ctx.config, g.contiguous(),
                      int(first), None, None, None, grad, rows, z.shape[-1], _lib.DTYPES[z.dtype], ws, ws.numel())
        return (grad,) + (None,) * 9


def policy_loss(logits, actions, old_logp, advantages, ref_logp=None, mask=None, clip=0.2, beta=0.0):
    """Clipped policy loss with a KL term: (loss, logp, stats).

    logits (..., classes) float32, bfloat16 or float16; per row, i.e. of shape logits.shape[:-1] or broadcast to it:
    actions (integers), old_logp (log probability of the action when it was drawn), advantages, ref_logp (the reference
    model's, for the KL term) and mask (bool; False: the row does not count and is not read).  With
    logp = log_softmax(logits)[action], rho = exp(logp - old_logp):

        loss = mean over the mask of  -min(rho A, clamp(rho, 1 - low, 1 + high) A) + beta (exp(d) - d - 1),  d = ref_logp - logp

    (0 where the mask leaves nothing); ``clip`` is low = high or the pair (low, high).  The loss is differentiable in the
    logits alone.  logp (the rows' log probabilities, 0 where masked) and stats = [policy part, KL, share of clipped rows] are
    fp32 and carry no gradient.  An action outside [0, classes) in a live row makes the loss NaN.  The gradient (of the logits'
    type, rounded once) is made in the forward already and takes the logits' size in memory until the backward.  A backward
    captured into a graph without its forward reads logits, actions and the rows' values at each replay, as they are then: it
    takes contiguous logits, int64 actions, fp32 and bool of the shape logits.shape[:-1] alone, which stay the caller's."""
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1 or logits.shape[-1] < 1:
        raise _lib.StepHipError("policy_loss: logits (..., classes) wanted")
    if logits.dtype not in _lib.DTYPES:
        raise _lib.StepHipError("policy_loss: float32, bfloat16 or float16 logits wanted, got %s" % logits.dtype)
    if logits.shape[-1] > 1 << 30:
        raise _lib.StepHipError("policy_loss: %d classes, 2^30 at most" % logits.shape[-1])
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    low, high, beta = float(low), float(high), float(beta)
    if not (0.0 <= low <= 1.0 and high >= 0.0):
        raise _lib.StepHipError("policy_loss: clip (%r, %r): 0 <= low <= 1 and high >= 0 wanted" % (low, high))
    lead = logits.shape[:-1]
    where = logits.get_device()
    copied = False

    def per_row(t, name, kinds, to):
        nonlocal copied
        if not isinstance(t, torch.Tensor) or t.dtype not in kinds:
            raise _lib.StepHipError("policy_loss: %s: a tensor of %s wanted, got %s" % (
                name, " / ".join(str(k)[6:] for k in kinds), getattr(t, "dtype", type(t).__name__)))
        if t.get_device() != where or t.is_meta != logits.is_meta:
            raise _lib.StepHipError("policy_loss: %s is on %s, logits on %s" % (name, t.device, logits.device))
        if t.dtype is to and t.shape == lead and not t.requires_grad and t.is_contiguous():
            return t
        try:
            r = t.detach().to(to).expand(lead).contiguous()
            copied = copied or r.data_ptr() != t.data_ptr()
            return r
        except RuntimeError:
            raise _lib.StepHipError("policy_loss: %s %s does not fit logits %s" % (name, tuple(t.shape), tuple(logits.shape))) from None

    floats = (torch.float32, torch.float64, torch.bfloat16, torch.float16)
    actions = per_row(actions, "actions", (torch.int64, torch.int32), torch.int64)
    old_logp = per_row(old_logp, "old_logp", floats, torch.float32)
    advantages = per_row(advantages, "advantages", floats, torch.float32)
    ref_logp = per_row(ref_logp, "ref_logp", floats, torch.float32) if ref_logp is not None else None
    mask = per_row(mask, "mask", (torch.bool,), torch.bool) if mask is not None else None
    if not logits.is_cuda:
        raise _lib.StepHipError("step_amd kernels need tensors on the GPU (got device %s); there is no CPU path" % logits.device)
    return _PolicyLossFn.apply(logits, actions, old_logp, advantages, ref_logp, mask, low, high, beta, copied)
