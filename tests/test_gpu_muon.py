"""GPU: step_amd.optim (newton_schulz, Muon) against the iteration in 64 bits.

Tolerances, relative to the result in the 2-norm (a result's singular values are all about 1).  u = 2^-24, h the half step of the
result's type.  min(m, n) <= 64 is taken in fp64: the final rounding h, and 1e-9 for everything before it.  Larger ones: a step
rounds each of three products (operands of 22 bits or more: 2^-23 each; fp32 sums: their roundings are independent and grow with the
square root of the terms, 2^-24 sqrt(K) at K <= 600: under 2^-19.4 of the terms' size) - under 1.5e-6 a product with K = 600 - and an
error is multiplied by at most 1.7 = max |p'| / (p / s) where the singular values have come near 1, which is in the last two or three
steps: 3 x 1.5e-6 x (1 + 1.7 + 1.7^2 + ...) <= 1.3e-5 x 2.  Tested at 2.5e-5; inputs have a condition that the fp32 iteration bears."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = torch.device("cuda:0")
U = 2.0 ** -24
A, B, C = 3.4445, -4.7750, 2.0315
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def orthogonalised(g, steps=5, eps=1e-7):
    x = g.double()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    for _ in range(steps):
        s = x @ x.mT.contiguous()
        y = s @ x
        x = A * x + B * y + C * (s @ y)
    return x.mT if tall else x


def matrices(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    m, n = shape[-2:]
    r = max(1, min(m, n) // 4)
    low = torch.randn(*shape[:-2], m, r, generator=g) @ torch.randn(*shape[:-2], r, n, generator=g) / math.sqrt(r)
    return (1e-3 * (low + torch.randn(*shape, generator=g))).to(dtype).to(D)


def tolerance(m, n, dtype):
    h = torch.finfo(dtype).eps / 2
    return h + (1e-9 if min(m, n) <= 64 else 2.5e-5)


def close(got, ref, tol, what=""):
    assert torch.isfinite(got).all(), what
    off = float((got.double() - ref).norm() / ref.norm())
    assert off <= tol, "%s: %.3e > %.1e" % (what, off, tol)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (4, 64), (16, 16), (17, 33), (33, 17), (64, 64), (64, 600), (601, 63), (64, 4800), (96, 3),
          (65, 65), (65, 64), (66, 300), (129, 127), (128, 128), (300, 131), (200, 600), (513, 257)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_newton_schulz(m, n, dtype):
    from step_amd import optim
    g = matrices(m, n, seed=m * n, dtype=dtype)
    o = optim.newton_schulz(g)
    assert o.shape == g.shape and o.dtype == dtype and o.data_ptr() != g.data_ptr()
    close(o, orthogonalised(g), tolerance(m, n, dtype), (m, n))


@pytest.mark.parametrize("shape", [(3, 20, 50), (2, 2, 70, 90), (5, 130, 66), (40, 8, 8), (1500, 5, 4)])
def test_stacks(shape):
    from step_amd import optim
    g = matrices(*shape)
    o = optim.newton_schulz(g)
    close(o, orthogonalised(g), tolerance(*shape[-2:], torch.float32))
    flat, one = g.reshape(-1, *shape[-2:]), o.reshape(-1, *shape[-2:])
    close(optim.newton_schulz(flat[-1]), orthogonalised(flat[-1]), tolerance(*shape[-2:], torch.float32))
    close(one[-1], orthogonalised(flat[-1]), tolerance(*shape[-2:], torch.float32))


def test_lists():
    """more small matrices than one launch takes, large ones and stacks among them, an empty one"""
    from step_amd import optim
    shapes = [(3 + i % 40, 5 + 3 * i % 70) for i in range(60)] + [(100, 80), (2, 9, 9), (0, 4), (70, 500)]
    gs = [matrices(*s, seed=i) if 0 not in s else torch.empty(s, device=D) for i, s in enumerate(shapes)]
    outs = optim.newton_schulz(gs)
    assert len(outs) == len(gs) and optim.newton_schulz([]) == []
    for g, o in zip(gs, outs):
        assert o.shape == g.shape
        if g.numel():
            close(o, orthogonalised(g), tolerance(*g.shape[-2:], torch.float32), tuple(g.shape))


@pytest.mark.parametrize("m,n", [(48, 200), (90, 140)])
@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_steps(m, n, steps):
    from step_amd import optim
    g = matrices(m, n)
    # one step more may multiply by 1.7 again
    close(optim.newton_schulz(g, steps=steps), orthogonalised(g, steps), tolerance(m, n, torch.float32) * (1 if steps < 6 else 5))


@pytest.mark.parametrize("m,n", [(30, 90), (120, 100)])
def test_scale_zero_inf_and_nan(m, n):
    from step_amd import optim
    g = matrices(m, n)
    ref = orthogonalised(g)
    for s in (1e-30, 1e-12, 1e12, 1e30):                     # the norm is taken in fp64
        got = optim.newton_schulz(g * s, eps=0.0)
        close(got, orthogonalised(g * s, eps=0.0), tolerance(m, n, torch.float32), s)
    assert not optim.newton_schulz(torch.zeros(m, n, device=D)).any()
    tiny = optim.newton_schulz(g * 1e-9)                      # eps counts
    close(tiny, orthogonalised(g * 1e-9), tolerance(m, n, torch.float32))
    for bad in (float("nan"), float("inf")):
        b = g.clone()
        b[3, 4] = bad
        o = optim.newton_schulz(torch.stack([g, b, g]))
        assert bool(o[1].isnan().all())
        close(o[0], ref, tolerance(m, n, torch.float32))
        close(o[2], ref, tolerance(m, n, torch.float32))


def test_strides_bits_and_views():
    from step_amd import optim
    g = matrices(90, 130)
    o = optim.newton_schulz(g)
    assert torch.equal(o, optim.newton_schulz(g))
    close(optim.newton_schulz(g.t()), orthogonalised(g).t(), 2.5e-5 + U)
    wide = torch.zeros(90, 140, device=D)
    wide[:, 3:133] = g
    assert torch.equal(o, optim.newton_schulz(wide[:, 3:133]))
    flat = torch.zeros(90 * 130 + 1, device=D)
    flat[1:] = g.reshape(-1)
    assert torch.equal(o, optim.newton_schulz(flat[1:].view(90, 130)))
    s = matrices(12, 40)
    assert torch.equal(optim.newton_schulz(s), optim.newton_schulz(s.t().contiguous().t()))


# ----------------------------------------------------------------------------------------------- the optimizer
def plain_step(p, buf, g, lr, mu, nesterov, decay):
    buf = mu * buf + g
    u = g + mu * buf if nesterov else buf
    o = orthogonalised(u.flatten(1)).view_as(p)
    m = p.shape[0]
    n = p.numel() // m
    return p * (1 - lr * decay) - lr * math.sqrt(max(1.0, m / n)) * o, buf


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_against_the_formula(nesterov):
    """three steps; after each the parameter is taken from the kernels, so that errors do not add up.  Bounds: the update's own
    tolerance, the momentum's two roundings (2 u of its terms), whose effect on an update is at most its condition, and the
    parameter's three roundings"""
    from step_amd import optim
    shapes = [(16, 8, 9, 1), (96, 3, 1, 1), (64, 64), (70, 10, 9, 1), (4, 64, 1, 1)]
    params = [torch.nn.Parameter(matrices(s[0], int(torch.tensor(s[1:]).prod()), seed=i).view(s) * 100) for i, s in enumerate(shapes)]
    skipped = torch.nn.Parameter(torch.ones(3, 3, device=D))
    opt = optim.Muon(params + [skipped], lr=0.03, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    bufs = [torch.zeros(s, dtype=torch.float64, device=D) for s in shapes]
    for step in range(3):
        for i, p in enumerate(params):
            p.grad = matrices(p.shape[0], p.numel() // p.shape[0], seed=100 * step + i).view(p.shape)
        before = [p.detach().double() for p in params]
        version = [p._version for p in params]
        opt.step()
        for i, p in enumerate(params):
            ref, buf = plain_step(before[i], bufs[i], p.grad.double(), 0.03, 0.9, nesterov, 0.1)
            got = opt.state[p]["momentum_buffer"]
            assert float((got.double() - buf).abs().max()) <= 3 * U * float((bufs[i].abs() + p.grad.abs()).max())
            change = (ref - before[i]).norm()
            off = (p.detach().double() - ref).norm()
            assert float(off) <= 5e-5 * float(change) + 3 * U * float(before[i].norm()), (step, i)
            bufs[i] = got.double()
            assert p._version > version[i]
    assert torch.equal(skipped, torch.ones(3, 3, device=D)) and skipped not in opt.state


def test_muon_adam_part_and_groups():
    """one-axis parameters and `matrices=False` groups take torch's own AdamW steps"""
    from step_amd import optim
    g = torch.Generator().manual_seed(0)
    vals = [torch.randn(s, generator=g) for s in ((5,), (3, 4, 4), ())]
    ours = [torch.nn.Parameter(v.to(D)) for v in vals]
    theirs = [torch.nn.Parameter(v.to(D)) for v in vals]
    opt = optim.Muon([{"params": ours, "matrices": False}], lr=0.01, weight_decay=0.02, adam_betas=(0.8, 0.9))
    ref = torch.optim.AdamW(theirs, lr=0.01, weight_decay=0.02, betas=(0.8, 0.9))
    for _ in range(4):
        for a, b in zip(ours, theirs):
            a.grad = torch.randn(a.shape, generator=g).to(D)
            b.grad = a.grad.clone()
        opt.step(), ref.step()
    for a, b in zip(ours, theirs):
        assert float((a - b).detach().abs().max()) <= 1e-6


def test_muon_state_dict_and_closure():
    from step_amd import optim

    def make():
        torch.manual_seed(1)
        return [torch.nn.Parameter(torch.randn(20, 30, device=D)), torch.nn.Parameter(torch.randn(20, device=D))]

    def run(opt, params, n, at):
        for k in range(n):
            for i, p in enumerate(params):
                p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * (at + k) + i)).to(D)
            assert float(opt.step(lambda: torch.tensor(2.0))) == 2.0

    p, q = make(), make()
    a, b = optim.Muon(p, lr=0.1), optim.Muon(q, lr=0.5)
    run(a, p, 2, 0)
    with torch.no_grad():
        for x, y in zip(q, p):
            x.copy_(y)
    b.load_state_dict(copy.deepcopy(a.state_dict()))          # (torch hands the tensors themselves over)
    run(a, p, 2, 2), run(b, q, 2, 2)
    assert all(torch.equal(x, y) for x, y in zip(p, q))


def test_captured_steps():
    """the step of small and large matrices, and a plain call beside it with a workspace of its own, replayed"""
    from step_amd import optim
    params = [torch.nn.Parameter(matrices(*s, seed=i)) for i, s in enumerate([(30, 50), (100, 90)])]
    grads = [matrices(*p.shape, seed=7) for p in params]
    extra = matrices(80, 70)
    for p, g in zip(params, grads):
        p.grad = g
    opt = optim.Muon(params, lr=0.02)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
        optim.newton_schulz(extra)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    with torch.cuda.graph(other):
        o = optim.newton_schulz(extra)
    for k in range(4):
        start = [(p.detach().clone(), opt.state[p]["momentum_buffer"].clone()) for p in params]
        for g, p in zip(grads, params):
            g.copy_(matrices(*p.shape, seed=20 + k))
        extra.copy_(matrices(80, 70, seed=k))
        torch.cuda.synchronize()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        after = [(p.detach().clone(), opt.state[p]["momentum_buffer"].clone()) for p in params]
        with torch.no_grad():
            for p, (v, b) in zip(params, start):
                p.copy_(v)
                opt.state[p]["momentum_buffer"].copy_(b)
        opt.step()
        for p, (v, b) in zip(params, after):
            assert torch.equal(p, v) and torch.equal(opt.state[p]["momentum_buffer"], b), k
        assert torch.equal(o, optim.newton_schulz(extra))
        torch.cuda.synchronize()


def test_two_streams_at_once():
    from step_amd import optim
    gs = [matrices(100, 140, seed=1), matrices(60, 400, seed=2)]
    want = [optim.newton_schulz(g) for g in gs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(optim.newton_schulz(gs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in (0, 1) for o in got[i])


def test_inference_caches_see_a_step():
    """the eval forward keeps packed weights by the parameters' versions: a step must be seen by the next eval forward"""
    from step_amd import optim
    from step_amd.net.classifier_real_and_synth import Classifier
    torch.manual_seed(0)
    m = Classifier(3, 4, {"strategy": "spatial"}).to(D).eval()
    x = 0.3 * torch.randn(3, 3, 75, 16, 1, device=D)
    with torch.no_grad():
        before, _ = m(x)
        m(x)
    opt = optim.Muon([p for p in m.parameters() if p.dim() == 4], lr=0.1)
    out, _ = m(x)
    torch.nn.functional.cross_entropy(out, torch.tensor([0, 1, 2], device=D)).backward()
    opt.step()
    with torch.no_grad():
        after, _ = m(x)
        fresh = Classifier(3, 4, {"strategy": "spatial"}).to(D).eval()
        fresh.load_state_dict(m.state_dict())
        want, _ = fresh(x)
    assert torch.equal(after, want) and not torch.equal(after, before)


# The products' tiles are 256 x 128, 128 x 128, 128 x 64 or 64 x 64, whole, split along the contraction, or both, by a count of
# their times: these shapes take each of them.  l >= 2 r may take up to three steps together.  Tolerance: the above with the
# contraction K = max(m, n), whose sums' roundings grow with its root.
@pytest.mark.parametrize("shape,dtype", [
    ((513, 3590), torch.float32), ((3590, 513), torch.bfloat16), ((2970, 2409), torch.float32), ((1781, 2810), torch.float32),
    ((1781, 2810), torch.float16), ((3048, 3035), torch.float32), ((3048, 3035), torch.bfloat16), ((3712, 2152), torch.float32),
    ((5, 2261, 1905), torch.float32), ((556, 2099), torch.float16), ((2012, 2601), torch.bfloat16), ((2012, 2601), torch.float32),
    ((449, 1941), torch.float16), ((150, 9001), torch.float32), ((9001, 130), torch.float32), ((9, 269, 2656), torch.bfloat16),
    ((8, 1157, 416), torch.float32), ((3, 1801, 600), torch.float32), ((1030, 65, 70), torch.float32)])   # (1024 at a time)
def test_larger(shape, dtype):
    from step_amd import optim
    m, n = shape[-2:]
    g = matrices(*shape, seed=m, dtype=dtype)
    tol = torch.finfo(dtype).eps / 2 + 2.5e-5 * max(1.0, math.sqrt(max(m, n) / 600))
    close(optim.newton_schulz(g), orthogonalised(g), tol, shape)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 8])
def test_steps_taken_together(steps):
    """three steps together cost the smallest singular values up to 2e-5 more; a step more may multiply by 1.7"""
    from step_amd import optim
    for m, n in ((70, 300), (901, 110), (170, 9001), (3000, 400)):
        g = matrices(m, n)
        close(optim.newton_schulz(g, steps=steps), orthogonalised(g, steps), tolerance(m, n, torch.float32) * (2 if steps < 6 else 5), (m, n))


def test_muon_refuses_what_it_cannot_do():
    from step_amd import optim
    p = torch.nn.Parameter(matrices(20, 30))
    alias = torch.nn.Parameter(p.detach())                    # the same memory
    for q in (p, alias):
        q.grad = matrices(20, 30, seed=1)
    before = p.detach().clone()
    with pytest.raises(optim._lib.StepHipError, match="twice"):
        optim.Muon([p, alias]).step()
    assert torch.equal(p, before)
    fresh, bias = optim.Muon([p]), optim.Muon([p, torch.nn.Parameter(torch.zeros(3, device=D))])
    bias.param_groups[0]["params"][1].grad = torch.ones(3, device=D)
    bias.step()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for opt, what in ((fresh, "one step before"), (bias, "counted on the host")):
        # (inside the capture, so that it ends in order)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(optim._lib.StepHipError, match=what):
                opt.step()
            p.detach().add_(0.0)
    torch.cuda.synchronize()
    assert not fresh.state.get(p)


@pytest.mark.parametrize("m,n", [(1690, 71), (10000, 100), (90, 12000), (6000, 130), (7000, 160), (300, 3000)])
def test_no_less_exact_than_fp32_products(m, n):
    """half as far again as the iteration with torch's own fp32 products at most: what 22 to 24 bits an operand, fp32 sums and the
    steps taken together may cost beside plain fp32"""
    from step_amd import optim
    g = matrices(m, n, seed=m)
    ref, plain = orthogonalised(g), orthogonalised32(g)
    off = [float((t.double() - ref).norm() / ref.norm()) for t in (optim.newton_schulz(g), plain)]
    assert off[0] <= 1.5 * off[1] + 2e-7, off


def orthogonalised32(g):
    x = g / (torch.linalg.vector_norm(g) + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.mT.contiguous() if tall else x
    for _ in range(5):
        s = x @ x.mT.contiguous()
        x = A * x + (B * s + C * (s @ s)) @ x
    return x.mT if tall else x


# What a size below eps may cost.  X_0 = g / (|g| + eps) is small by any power there, and so are the first steps' results, which grow
# by a = 3.4445 each: the tolerance is relative and the same as for any other size, since nothing in the formula is less exact there.
# References: the result's type rounds them where it has no such small numbers (half a unit of its smallest one, 2^-150 in fp32).
@pytest.mark.parametrize("m,n", [(30, 90), (120, 100), (300, 1300), (9001, 170), (2000, 600)])
def test_sizes_far_below_eps(m, n):
    from step_amd import optim
    g = matrices(m, n, seed=3)
    g = g / g.norm()
    for e in (-7, -9, -11, -12, -13, -15, -18, -25, -34):
        for steps in (1, 5, 7):
            t = g * 10.0 ** e
            close(optim.newton_schulz(t, steps=steps), orthogonalised(t, steps), tolerance(m, n, torch.float32) * (1 if steps < 6 else 5), (e, steps))
    for eps in (1e-3, 1.0, 1e20, 1e-30):
        for e in (-3, -8, -30):
            t = g * 10.0 ** e
            ref = orthogonalised(t, 5, float(torch.tensor(eps)))
            if float(ref.norm()) > 1e-30:
                close(optim.newton_schulz(t, eps=eps), ref, tolerance(m, n, torch.float32), (e, eps))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_stack_of_sizes(dtype):
    """each matrix of a stack has its own size: one among ordinary ones and zeros"""
    from step_amd import optim
    sizes = [1.0, 1e-4, 3e-7, 2e-6, 0.0, 1e-5]
    eps = 1e-4
    for m, n in ((100, 140), (20, 140), (90, 2700)):
        g = torch.stack([matrices(m, n, seed=i).div_(matrices(m, n, seed=i).norm()) * s for i, s in enumerate(sizes)]).to(dtype)
        o = optim.newton_schulz(g, eps=eps)
        ref = orthogonalised(g, 5, eps)
        for i, s in enumerate(sizes):
            if not g[i].any():                                # (fp16 holds nothing of the smallest)
                assert not o[i].any()
                continue
            # 16 bits: half a unit of the smallest number beside the relative rounding, in every element
            tiny = math.sqrt(m * n) * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 / float(ref[i].norm())
            close(o[i], ref[i], tolerance(m, n, dtype) + tiny, (m, n, s))


@pytest.mark.parametrize("m,n", [(30, 90), (120, 100)])
def test_zero_without_eps(m, n):
    """a zero matrix stays zero whatever eps is; the smallest numbers do not count as zeros"""
    from step_amd import optim
    assert not optim.newton_schulz(torch.zeros(2, m, n, device=D), eps=0.0).any()
    p = torch.nn.Parameter(torch.ones(m, n, device=D))
    p.grad = torch.zeros_like(p)
    optim.Muon([p], eps=0.0, lr=0.1).step()
    assert torch.equal(p, torch.ones_like(p))
    g = matrices(m, n) * 1e-36                                # subnormal elements among them: what fp32 holds of them is the input
    close(optim.newton_schulz(g, eps=0.0), orthogonalised(g, eps=0.0), tolerance(m, n, torch.float32))


def kinds(m, n):
    """low rank and noise, noise alone, singular values over a range of 30 and of 1000"""
    gen = torch.Generator().manual_seed(m + n)
    r, l = min(m, n), max(m, n)
    u, v = (torch.linalg.qr(torch.randn(k, r, generator=gen).to(D).double())[0] for k in (r, l))
    yield matrices(m, n, seed=m)
    yield torch.randn(m, n, generator=gen).to(D)
    for condition in (30.0, 1000.0):
        x = (u * condition ** -torch.linspace(0, 1, r, device=D, dtype=torch.float64)) @ v.t().contiguous()
        yield (x if m <= n else x.t()).float().contiguous()


@pytest.mark.parametrize("m,n", [(6000, 160), (160, 8000), (7000, 192), (192, 10000), (224, 6000), (256, 9000), (300, 10000), (340, 3000),
                                 (500, 6000), (1000, 3000), (1400, 3000), (200, 200)])
def test_as_exact_as_fp32_products_on_all_kinds(m, n):
    """root 2 times the error of the iteration with torch's own fp32 products at most.  Of an error's three parts - the operands'
    rounding, the sums' and the results' - the first is 2^-23 for two halves of 11 bits where fp32 has 2^-24, the others are fp32's
    (root of (4 + 1 + 1) / 3); it is these that the smallest singular values multiply, on both sides alike"""
    from step_amd import optim
    for i, g in enumerate(kinds(m, n)):
        ref = orthogonalised(g)
        off = [float((t.double() - ref).norm() / ref.norm()) for t in (optim.newton_schulz(g), orthogonalised32(g))]
        assert off[0] <= math.sqrt(2) * off[1], (i, off)


def test_more_small_matrices_than_a_launch_takes():
    """stacks and lists that are divided: each launch has a matrix of many blocks' work beside a stack, or more matrices than one
    launch may have blocks of 256 to 1024 threads"""
    from step_amd import optim
    g = matrices(1000000, 4, 4, seed=1)
    o = optim.newton_schulz(g)
    for at in (slice(0, 5), slice(4090, 4100), slice(999990, None)):
        close(o[at], orthogonalised(g[at]), tolerance(4, 4, torch.float32))
    ref = orthogonalised(g)
    per = (o.double() - ref).norm(dim=(1, 2)) / ref.norm(dim=(1, 2))
    assert float(per.max()) <= tolerance(4, 4, torch.float32)
    g = matrices(5000, 33, 70, seed=2)
    o = optim.newton_schulz(g)
    close(o, orthogonalised(g), tolerance(33, 70, torch.float32))
    same = optim.newton_schulz(g[:1].expand(5000, 33, 70))    # one matrix is one result, wherever it lies in a stack
    assert torch.equal(same, same[:1].expand(5000, 33, 70))


def test_a_long_matrix_beside_a_stack():
    from step_amd import optim
    long, wide = (torch.randn(*s, generator=torch.Generator(D).manual_seed(i), device=D) for i, s in enumerate([(64, 1 << 21), (1 << 21, 3)]))
    stack = matrices(512, 8, 8, seed=3)
    outs = optim.newton_schulz([long, stack, wide])
    for g, o in zip((long, stack, wide), outs):
        close(o, orthogonalised(g), tolerance(1, 1, torch.float32), tuple(g.shape))


@pytest.mark.parametrize("shape,dtype", [((3, 2101, 530), torch.bfloat16), ((256, 9600), torch.float32), ((1781, 1810), torch.float16), ((70, 9, 33), torch.float32)])
def test_the_same_bits_on_any_stream_and_memory(shape, dtype):
    """split tiles, steps taken together, stacks: called again beside other work, in memory that held something else"""
    from step_amd import optim
    g = matrices(*shape, dtype=dtype)
    want = optim.newton_schulz(g)
    side = torch.cuda.Stream()
    for k in range(6):
        junk = torch.full((1 << 26,), float("nan"), device=D)
        del junk
        stream = side if k % 2 else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = optim.newton_schulz(g)
        if k % 2:
            optim.newton_schulz(g)                            # on the other stream meanwhile
        torch.cuda.synchronize()
        assert torch.equal(got, want), k
