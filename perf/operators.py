"""The training operators of a model's norm, objective and update, as cases that can be timed.

    layer_norm     step_amd.ops.layer_norm       layer norm, forward and backward
    policy         step_amd.losses.policy_loss   clipped policy loss with a KL term, value and gradient
    newton_schulz  step_amd.optim.newton_schulz  the orthogonalised update of a matrix or a stack of matrices
    muon           step_amd.optim.Muon           one step over the weights of a classifier

With `own` false, run() computes them from elementary torch operations; with `own` true it makes the calls that a
user of step_amd makes.  exact() is the same in 64 bits, from the definitions."""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

LN_EPS = 1e-5
CLIP, BETA = 0.2, 0.04
A, B, C = 3.4445, -4.7750, 2.0315       # the quintic of the Newton-Schulz step
STEPS, NS_EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the hybrid classifier's head (64 pooled + 29 affective features) at the training batch of 4096 gaits
        {"name": "ln_head", "op": "layer_norm", "rows": 4096, "cols": 93, "dtype": "f32", "backward": True},
        # one token while answering: nothing but latency
        {"name": "ln_token", "op": "layer_norm", "rows": 1, "cols": 4096, "dtype": "bf16", "backward": False},
        # a training batch of 16k tokens: the memory's rate
        {"name": "ln_batch", "op": "layer_norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "backward": True},
        # rows that no wide load is aligned to
        {"name": "ln_odd", "op": "layer_norm", "rows": 9001, "cols": 2187, "dtype": "f16", "backward": True},
        # the four emotions of the classifier, a training batch of gaits
        {"name": "policy_emotions", "op": "policy", "rows": 4096, "classes": 4, "dtype": "f32", "kl": False, "padded": False},
        # answers of a language model, padded to one length
        {"name": "policy_tokens", "op": "policy", "rows": 8192, "classes": 32000, "dtype": "bf16", "kl": True, "padded": True},
        # an odd vocabulary in 32 bits
        {"name": "policy_odd", "op": "policy", "rows": 1021, "classes": 50257, "dtype": "f32", "kl": True, "padded": True},
        # a vocabulary larger than one block of threads holds in registers
        {"name": "policy_wide", "op": "policy", "rows": 640, "classes": 140001, "dtype": "bf16", "kl": True, "padded": False},
        # a step over every matrix of the 3-32-64-64 classifier with 75 taps: many small matrices at once
        {"name": "muon_classifier", "op": "muon", "widths": "32,64,64", "taps": 75, "dtype": "f32"},
        # the 75-tap temporal convolution of a 256-channel block
        {"name": "ns_wide_block", "op": "newton_schulz", "batch": 1, "m": 256, "n": 19200, "dtype": "f32"},
        # a stack of tall matrices whose sizes fit no tile
        {"name": "ns_tall_stack", "op": "newton_schulz", "batch": 3, "m": 4101, "n": 1030, "dtype": "bf16"},
        # a square projection of a large model
        {"name": "ns_square", "op": "newton_schulz", "batch": 1, "m": 4096, "n": 4096, "dtype": "f32"},
    ]


def _spread(rng, lo, hi):
    """a whole number whose logarithm is evenly spread"""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("layer_norm", "layer_norm", "policy", "policy", "newton_schulz", "newton_schulz", "muon"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "layer_norm":
        cols = _spread(rng, 3, 16384)
        rows = _spread(rng, 1, min(65536, 16384 * 4096 // cols))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "backward": rng.random() < 0.7}
    if op == "policy":
        classes = _spread(rng, 2, 150000)
        rows = _spread(rng, 1, min(65536, 100000000 // classes))
        return {"op": op, "rows": rows, "classes": classes, "dtype": dtype, "kl": rng.random() < 0.7, "padded": rng.random() < 0.7}
    if op == "muon":
        widths = ",".join(str(_spread(rng, 16, 128)) for _ in range(3))
        return {"op": op, "widths": widths, "taps": rng.choice((9, 25, 75)), "dtype": "f32"}
    m = _spread(rng, 2, 4096)
    n = _spread(rng, 2, min(19200, 4096 * 4096 // m))
    batch = rng.choice((1, 1, 2, 5)) if 5 * m * n <= 4096 * 4096 else 1
    m, n = (m, n) if rng.random() < 0.5 else (n, m)
    return {"op": op, "batch": batch, "m": m, "n": n, "dtype": dtype}


def _matrices(case):
    """the weights of a classifier's three blocks (graph, temporal and residual convolutions) and of its last layer"""
    taps, cin, shapes = case["taps"], 3, []
    for i, w in enumerate(int(x) for x in case["widths"].split(",")):
        shapes += [(3 * w, cin, 1, 1), (w, w, taps, 1)]
        if i < 2:
            shapes.append((w, cin, 1, 1))
        cin = w
    return shapes + [(4, cin, 1, 1)]


def _ns_flops(m, n):
    r, c = min(m, n), max(m, n)
    return STEPS * (3 * r * r * c + r ** 3)          # two of the three products are symmetric


def work(case):
    if case["op"] == "layer_norm":
        e, s = case["rows"] * case["cols"], BYTES[case["dtype"]]
        if case["backward"]:
            return {"bytes": 4 * e * s + 4 * case["cols"] * s, "flops": 20 * e}
        return {"bytes": 2 * e * s + 2 * case["cols"] * s, "flops": 8 * e}
    if case["op"] == "policy":
        e = case["rows"] * case["classes"]
        # a padded row is not read: its gradient is zero
        return {"bytes": ((0.8 if case["padded"] else 1) + 1) * e * BYTES[case["dtype"]] + 24 * case["rows"], "flops": 10 * e}
    if case["op"] == "muon":
        mats = [(s[0], s[1] * s[2] * s[3]) for s in _matrices(case)]
        return {"bytes": 20 * sum(m * n for m, n in mats), "flops": sum(_ns_flops(m, n) for m, n in mats)}
    e = case["batch"] * case["m"] * case["n"]
    return {"bytes": 2 * e * BYTES[case["dtype"]], "flops": case["batch"] * _ns_flops(case["m"], case["n"])}


# ----------------------------------------------------------------------------------------------- the inputs
def _momentum(shape, g):
    """a matrix such as an update has before it is orthogonalised: some directions that fall off, over noise"""
    m, n = shape[-2:]
    r = max(1, min(m, n) // 4)
    fall = torch.arange(1, r + 1, device=DEVICE) ** -0.5
    low = torch.matmul(torch.randn(*shape[:-2], m, r, device=DEVICE, generator=g) * fall, torch.randn(*shape[:-2], r, n, device=DEVICE, generator=g))
    return 1e-3 * (low + 0.5 * torch.randn(shape, device=DEVICE, generator=g))


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=DEVICE, generator=g)

    if case["op"] == "layer_norm":
        rows, cols = case["rows"], case["cols"]
        scale = torch.exp(0.5 * randn(rows, 1))             # activations: rows of different size, features off zero
        x = (randn(rows, cols) * scale + 0.3 * randn(cols)).to(dtype)
        w, b = (1 + 0.2 * randn(cols)).to(dtype), (0.1 * randn(cols)).to(dtype)
        dy = randn(rows, cols).to(dtype) if case["backward"] else None
        if case["backward"]:
            x, w, b = (t.requires_grad_(True) for t in (x, w, b))
        return {"case": case, "x": x, "w": w, "b": b, "dy": dy}

    if case["op"] == "policy":
        rows, classes = case["rows"], case["classes"]
        logits = (2.0 * randn(rows, classes)).to(dtype)
        noise = torch.empty(rows, classes, device=DEVICE).exponential_(generator=g)
        actions = (logits.float() - noise.log_()).argmax(1)           # drawn from the model itself
        del noise
        logp = logits.float().gather(1, actions[:, None])[:, 0] - torch.logsumexp(logits.float(), 1)
        old, ref = logp + 0.15 * randn(rows), logp + 0.3 * randn(rows)
        mask = None
        if case["padded"]:
            mask = torch.rand(rows, device=DEVICE, generator=g) < 0.8
        return {"case": case, "logits": logits.requires_grad_(True), "actions": actions, "old": old, "adv": randn(rows),
                "ref": ref if case["kl"] else None, "mask": mask}

    if case["op"] == "muon":
        params = []
        for s in _matrices(case):
            p = torch.nn.Parameter(randn(*s) / math.sqrt(s[1] * s[2]))
            p.grad = _momentum((s[0], s[1] * s[2] * s[3]), g).view(s)
            params.append(p)
        return {"case": case, "params": params}

    return {"case": case, "g": _momentum((case["batch"], case["m"], case["n"]), g).to(dtype)}


# ------------------------------------------------------------------------------------------- the plain forms
def _plain_layer_norm(x, w, b, dy):
    xf, wf = x.detach().float(), w.detach().float()
    d = xf - xf.mean(1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + LN_EPS)
    xhat = d * rstd
    y = (xhat * wf + b.detach().float()).to(x.dtype)
    if dy is None:
        return y
    dyf = dy.float()
    t = dyf * wf
    dx = rstd * (t - t.mean(1, keepdim=True) - xhat * (t * xhat).mean(1, keepdim=True))
    return y, dx.to(x.dtype), (dyf * xhat).sum(0).to(w.dtype), dyf.sum(0).to(b.dtype)


def _plain_policy(logits, actions, old, adv, ref, mask):
    z = logits.detach().float()
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    at = actions[:, None]
    # a row's few values in 64 bits: its ratio may lie next to the border of the clipping
    logp = (z.gather(1, at).double() - top.double() - torch.log(total.double()))[:, 0]
    old, adv, ref = old.double(), adv.double(), None if ref is None else ref.double()
    ratio = torch.exp(logp - old)
    one, two = ratio * adv, ratio.clamp(1 - CLIP, 1 + CLIP) * adv
    live = torch.ones_like(adv, dtype=torch.bool) if mask is None else mask
    count = live.sum().clamp(min=1)
    zero = torch.zeros_like(adv)
    obj = -torch.minimum(one, two)
    slope = torch.where(one <= two, -one, zero)
    kl = zero
    if ref is not None:
        kl = torch.exp(ref - logp) - (ref - logp) - 1
        slope = slope + BETA * (1 - torch.exp(ref - logp))
    clipped = (one > two).double()
    stats = torch.stack([torch.where(live, t, zero).sum() for t in (obj, kl, clipped)]) / count
    slope = torch.where(live, slope / count, zero).float()[:, None]
    grad = torch.where(live[:, None], e / total * -slope, 0.0)
    grad.scatter_add_(1, at, slope)
    return (stats[0] + BETA * stats[1]).float(), torch.where(live, logp, zero).float(), stats.float(), grad.to(logits.dtype)


def _plain_newton_schulz(g):
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + NS_EPS)
    for _ in range(STEPS):
        p = x @ x.mT.contiguous()
        x = A * x + (B * p + C * (p @ p)) @ x
    return (x.mT if tall else x).contiguous().to(g.dtype)


def _plain_muon(state):
    bufs = state.setdefault("bufs", [torch.zeros_like(p) for p in state["params"]])
    with torch.no_grad():
        for p, buf in zip(state["params"], bufs):
            buf.mul_(MOMENTUM).add_(p.grad)
            u = (p.grad + MOMENTUM * buf).flatten(1)
            o = _plain_newton_schulz(u).view_as(p) * math.sqrt(max(1.0, u.shape[0] / u.shape[1]))
            p.mul_(1 - LR * DECAY).add_(o, alpha=-LR)
    return [p.detach() for p in state["params"]], bufs


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    if op == "layer_norm":
        return _plain_layer_norm(state["x"], state["w"], state["b"], state["dy"])
    if op == "policy":
        return _plain_policy(state["logits"], state["actions"], state["old"], state["adv"], state["ref"], state["mask"])
    if op == "muon":
        return _plain_muon(state)
    return _plain_newton_schulz(state["g"])


# ----------------------------------------------------------------------------------------- the framework's calls
def _own(state, op):
    from step_amd import losses, ops, optim
    if op == "layer_norm":
        y = ops.layer_norm(state["x"], state["w"], state["b"], LN_EPS)
        if state["dy"] is None:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (state["x"], state["w"], state["b"]), state["dy"])
    if op == "policy":
        loss, logp, stats = losses.policy_loss(state["logits"], state["actions"], state["old"], state["adv"], state["ref"],
                                               state["mask"], clip=CLIP, beta=BETA)
        (grad,) = torch.autograd.grad(loss, state["logits"])
        return loss.detach(), logp, stats, grad
    if op == "muon":
        if "opt" not in state:
            state["opt"] = optim.Muon(state["params"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY)
        state["opt"].step()
        return [p.detach() for p in state["params"]], [state["opt"].state[p]["momentum_buffer"] for p in state["params"]]
    return optim.newton_schulz(state["g"], steps=STEPS, eps=NS_EPS)


# -------------------------------------------------------------------------------------------- in 64 bits
def _exact_newton_schulz(g):
    x = g.double()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + NS_EPS)
    for _ in range(STEPS):
        if x.shape[-2] <= x.shape[-1]:
            s = x @ x.mT.contiguous()
            x3 = s @ x
            x5 = s @ x3
        else:
            s = x.mT.contiguous() @ x
            x3 = x @ s
            x5 = x3 @ s
        x = A * x + B * x3 + C * x5
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "layer_norm":
        x, w, b = (state[k].detach().double().requires_grad_(case["backward"]) for k in ("x", "w", "b"))
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        y = (x - mean) / torch.sqrt(var + LN_EPS) * w + b
        if not case["backward"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), state["dy"].double())
    if case["op"] == "policy":
        z = state["logits"].detach().double().requires_grad_(True)
        logp = torch.log_softmax(z, 1).gather(1, state["actions"][:, None])[:, 0]
        ratio, adv = torch.exp(logp - state["old"].double()), state["adv"].double()
        one, two = ratio * adv, torch.where(ratio > 1 + CLIP, 1 + CLIP, torch.where(ratio < 1 - CLIP, 1 - CLIP, ratio)) * adv
        rows = torch.arange(len(adv), device=z.device) if state["mask"] is None else state["mask"].nonzero()[:, 0]
        count = max(1, len(rows))
        d = state["ref"].double() - logp if state["ref"] is not None else torch.zeros_like(logp)
        kl = torch.expm1(d) - d
        stats = torch.stack([t[rows].sum() / count for t in (-torch.minimum(one, two), kl, (two < one).double())])
        loss = stats[0] + BETA * stats[1]
        (grad,) = torch.autograd.grad(loss, z)
        lp = torch.zeros_like(adv)
        lp[rows] = logp.detach()[rows]
        return loss.detach(), lp, stats.detach(), grad
    if case["op"] == "muon":
        params, bufs = [], []
        for p in state["params"]:
            g = p.grad.double().flatten(1)                       # the first step: the momentum is the gradient
            o = _exact_newton_schulz((1 + MOMENTUM) * g).view_as(p) * max(1.0, g.shape[0] / g.shape[1]) ** 0.5
            params.append(p.detach().double() * (1 - LR * DECAY) - LR * o)
            bufs.append(p.grad.double())
        return params, bufs
    return _exact_newton_schulz(state["g"])
