"""GPU: step_amd.losses.policy_loss against the definition in 64 bits.

Tolerances.  u = 2^-24.  An element's exponent is off by at most 3 u times its size in base 2 (two roundings of the fused
operations, one of the row's maximum), v_exp_f32 by one unit (2 u), the sum by its chain of additions (at most 160: 128 values a
thread, then a tree of 16 and 6): the logarithm of the sum is off by L = (3 range + 164) u with range = the spread of the row's
logits (in base 2) that weigh anything, at most 40.  The log probability adds its own rounding.  A ratio is off by L relatively,
the gradient's coefficient as well, a probability by 2 L; the loss, an average, by the average of |A| rho L, and its rounding.
The gradient is rounded once to the logits' type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = torch.device("cuda:0")
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
LSE = (3 * 40 + 164) * U


def reference(logits, actions, old, adv, ref, mask, low, high, beta):
    """the loss, log probabilities, statistics and gradient in 64 bits, by autograd, and the size of what they add up"""
    z = logits.detach().double().requires_grad_(True)
    classes = z.shape[-1]
    zr, a = z.reshape(-1, classes), actions.reshape(-1)
    live = torch.ones(len(a), dtype=torch.bool, device=z.device) if mask is None else mask.reshape(-1)
    rows = live.nonzero()[:, 0]
    old, adv = old.reshape(-1).double()[rows], adv.reshape(-1).double()[rows]
    lp = torch.log_softmax(zr[rows], 1).gather(1, a[rows][:, None])[:, 0]
    rho = torch.exp(lp - old)
    o1, o2 = rho * adv, rho.clamp(1 - low, 1 + high) * adv
    d = ref.reshape(-1).double()[rows] - lp if ref is not None else torch.zeros_like(lp)
    kl = torch.exp(d) - d - 1
    n = max(1, len(rows))
    parts = [t.sum() / n for t in (-torch.minimum(o1, o2), kl, (o1 > o2).double())]
    loss = parts[0] + beta * parts[1]
    (g,) = torch.autograd.grad(loss, z) if len(rows) else (torch.zeros_like(z),)
    logp = torch.zeros(len(a), dtype=torch.float64, device=z.device)
    logp[rows] = lp.detach()
    size = float(((rho * adv).abs().sum() + beta * ((torch.exp(d) - 1).abs().sum() + kl.sum())) / n) if len(rows) else 0.0
    slope = torch.zeros(len(a), dtype=torch.float64, device=z.device)
    slope[rows] = (((rho * adv).abs() + beta * (torch.exp(d) + 1)) / n).detach()
    return loss.detach(), logp.view(actions.shape), torch.stack(parts).detach(), g, size, slope


def inputs(lead, classes, dtype, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    z = (scale * torch.randn(*lead, classes, generator=g)).to(dtype)
    a = torch.randint(0, classes, lead, generator=g)
    lp = torch.log_softmax(z.double(), -1).gather(-1, a[..., None])[..., 0]
    old = (lp + 0.2 * torch.randn(lead, generator=g)).float()
    ref = (lp + 0.3 * torch.randn(lead, generator=g)).float()
    adv = torch.randn(lead, generator=g)
    mask = torch.rand(lead, generator=g) < 0.7
    return [t.to(D) for t in (z, a, old, adv, ref, mask)]


def check(z, a, old, adv, ref, mask, clip=0.2, beta=0.05, upstream=None):
    from step_amd import losses
    low, high = clip if isinstance(clip, tuple) else (clip, clip)
    leaf = z.detach().clone().requires_grad_(True)
    loss, logp, stats = losses.policy_loss(leaf, a, old, adv, ref, mask, clip=clip, beta=beta)
    (loss if upstream is None else upstream * loss).backward()
    rl, rlp, rs, rg, size, slope = reference(z, a, old, adv, ref, mask, low, high, beta)
    assert loss.dtype == torch.float32 and logp.shape == a.shape and leaf.grad.dtype == z.dtype
    assert abs(float(loss) - float(rl)) <= LSE * size + 2 * U * abs(float(rl)), (float(loss), float(rl))
    assert bool(((logp.double() - rlp).abs() <= LSE + 2 * U * rlp.abs()).all())
    assert float((stats.double() - rs).abs().max()) <= LSE * (size / max(beta, 1e-9) if beta else size) + 2 * U * float(rs.abs().max())
    if upstream is not None:
        rg, slope = rg * upstream, slope * abs(upstream)
    classes = z.shape[-1]
    p = torch.softmax(z.double().reshape(-1, classes), 1)
    onehot = torch.zeros_like(p).scatter_(1, a.reshape(-1, 1).clamp(0, classes - 1), 1.0)
    bound = (slope[:, None] * (p * (4 * LSE + 4 * U) + onehot * (4 * LSE + 4 * U))).view_as(rg)
    fi = torch.finfo(z.dtype)
    lim = bound + fi.eps / 2 * (rg.abs() + bound) + fi.smallest_normal * fi.eps
    off = (leaf.grad.double() - rg).abs()
    assert bool((off <= lim).all()), float((off / lim).max())
    return loss, logp, stats, leaf.grad


# classes about every border of the choice of threads per row (8 / 64 / 256 / 1024, 1 to 16 packs), odd ones among them
CLASSES = [1, 2, 4, 5, 31, 33, 63, 97, 255, 256, 257, 511, 513, 1000, 2047, 4095, 4097, 8000, 8193, 16383, 16400, 32000, 50257, 65535, 65540,
           131072, 131079, 140001]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_value_and_gradient(classes, dtype):
    check(*inputs((11 if classes < 5000 else 3,), classes, dtype, seed=classes))


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 4096, 20001])
def test_rows_of_four_emotions(rows):
    z, a, old, adv, ref, mask = inputs((rows,), 4, torch.float32, seed=rows)
    check(z, a, old, adv, ref, mask)
    check(z, a, old, adv, None, None)


@pytest.mark.parametrize("clip,beta", [(0.2, 0.0), ((0.1, 0.3), 0.5), ((1.0, 1e9), 0.04), (0.0, 0.04)])
def test_clip_and_beta(clip, beta):
    z, a, old, adv, ref, mask = inputs((6, 50), 77, torch.float32)
    check(z, a, old, adv, ref, mask, clip=clip, beta=beta)


@pytest.mark.parametrize("dtype", TYPES)
def test_upstream_gradient_and_a_retained_graph(dtype):
    from step_amd import losses
    args = inputs((40,), 300, dtype)
    check(*args, upstream=1024.0)                             # a loss scale: one rounding, nothing lost below fp16's range
    check(*args, upstream=-0.3)
    leaf = args[0].clone().requires_grad_(True)
    loss, _, _ = losses.policy_loss(leaf, *args[1:], beta=0.05)
    grads = [torch.autograd.grad(loss, leaf, torch.tensor(s, device=D), retain_graph=True)[0] for s in (1.0, 1.0, 2.0, 1.0)]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[3])
    assert len({g.data_ptr() for g in grads}) == 4            # each call's gradient is its own
    _, _, _, two = check(*args, upstream=2.0)
    assert torch.equal(two, grads[2])


def test_masks():
    from step_amd import losses
    z, a, old, adv, ref, mask = inputs((64,), 501, torch.float32)
    none = torch.zeros_like(mask)
    loss, logp, stats, grad = check(z, a, old, adv, ref, none)
    assert float(loss) == 0.0 and not logp.any() and not stats.any() and not grad.any()
    # what stands in a masked row - logits, action, log probabilities - is never looked at
    want = check(z, a, old, adv, ref, mask)
    z2, a2, old2, adv2, ref2 = z.clone(), a.clone(), old.clone(), adv.clone(), ref.clone()
    out = ~mask
    z2[out], a2[out], old2[out], adv2[out], ref2[out] = float("nan"), -100, float("inf"), float("nan"), float("-inf")
    leaf = z2.requires_grad_(True)
    got = losses.policy_loss(leaf, a2, old2, adv2, ref2, mask, beta=0.05)
    got[0].backward()
    for p, q in zip(got + (leaf.grad,), want):
        assert torch.equal(p, q)


def test_forbidden_classes_and_actions_out_of_range():
    from step_amd import losses
    z, a, old, adv, ref, _ = inputs((30,), 120, torch.float32)
    z[:, 60:] = float("-inf")                                 # classes that may not be chosen
    a = a % 60
    lp = torch.log_softmax(z.double(), 1).gather(1, a[:, None])[:, 0]
    check(z, a, (lp + 0.1).float(), adv, (lp - 0.1).float(), None)
    for bad in (-1, 120, 1 << 40, -(1 << 40)):
        b = a.clone()
        b[3] = bad
        leaf = z.clone().requires_grad_(True)
        loss, logp, _ = losses.policy_loss(leaf, b, old, adv, ref)
        loss.backward()
        assert bool(loss.isnan()) and bool(logp[3].isnan()) and int(logp.isnan().sum()) == 1
        assert bool(leaf.grad[3].isnan().any()) and bool(leaf.grad[4].isfinite().all())


def test_nan_logits_are_not_hidden():
    from step_amd import losses
    z, a, old, adv, ref, _ = inputs((8,), 90, torch.float32)
    z[2, 5] = float("nan")
    z[5] = float("-inf")                                      # a row that allows nothing
    loss, logp, _ = losses.policy_loss(z, a, old, adv, ref)
    assert bool(loss.isnan()) and logp.isnan().tolist() == [False, False, True, False, False, True, False, False]


def test_broadcast_strides_types_and_no_gradient():
    from step_amd import losses
    z, a, old, adv, ref, mask = inputs((6, 20), 130, torch.bfloat16)
    per_answer = adv[:, :1]                                   # one advantage an answer
    check(z, a, old, per_answer.expand(6, 20), ref, mask)
    want = losses.policy_loss(z, a, old, per_answer.expand(6, 20).contiguous(), ref, mask, beta=0.05)
    got = losses.policy_loss(z, a.int(), old.double(), per_answer, ref, mask, beta=0.05)
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and not got[0].requires_grad
    wide = torch.randn(6, 20, 140, device=D).to(torch.bfloat16)
    check(wide[..., 5:135], a, old, adv, ref, mask)           # strided rows
    flat = torch.randn(6 * 20 * 130 + 1, device=D)
    check(flat[1:].view(6, 20, 130), a, old, adv, ref, mask)  # rows that start off 16 bytes
    check(z[0, 0], a[0, 0], old[0, 0], adv[0, 0], None, None)  # one row without leading axes
    old.requires_grad_(True)
    leaf = z.clone().requires_grad_(True)
    losses.policy_loss(leaf, a, old, adv)[0].backward()
    assert old.grad is None and leaf.grad is not None
    e = torch.empty(0, 7, device=D, requires_grad=True)
    loss, logp, _ = losses.policy_loss(e, torch.empty(0, dtype=torch.int64, device=D), torch.empty(0, device=D), torch.empty(0, device=D))
    loss.backward()
    assert float(loss) == 0.0 and logp.shape == (0,) and e.grad.shape == (0, 7)


def test_logits_changed_before_the_backward_are_refused():
    from step_amd import losses
    z, a, old, adv, _, _ = inputs((6,), 30, torch.float32)
    x = z.clone().requires_grad_(True)
    y = x * 1.0
    loss, _, _ = losses.policy_loss(y, a, old, adv)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_gradient_against_differences():
    """along a direction; away from the clipping's borders (clip 1e3) the loss is smooth.  Error: fp32 noise of two losses
    over 2 h (LSE / h = 1.7e-5 / 1e-2) plus h^2"""
    from step_amd import losses
    z, a, old, adv, ref, mask = inputs((50,), 40, torch.float32)
    leaf = z.clone().requires_grad_(True)
    f = lambda t: losses.policy_loss(t, a, old, adv, ref, mask, clip=(1.0, 1e3), beta=0.3)[0]  # noqa: E731
    f(leaf).backward()
    v = torch.randn(50, 40, generator=torch.Generator().manual_seed(3)).to(D)
    h = 1e-2
    num = (float(f(z + h * v)) - float(f(z - h * v))) / (2 * h)
    scale = float((leaf.grad.double() * v.double()).abs().sum())
    assert abs(num - float((leaf.grad.double() * v.double()).sum())) <= 5e-3 * scale + 5e-3


def test_the_same_bits_every_time_and_captured():
    from step_amd import losses
    z, a, old, adv, ref, mask = inputs((700,), 1003, torch.bfloat16)
    zs = z.clone().requires_grad_(True)

    def step():
        loss, logp, stats = losses.policy_loss(zs, a, old, adv, ref, mask, beta=0.05)
        return loss, logp, stats, torch.autograd.grad(loss, zs)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        with torch.no_grad():
            zs.copy_(inputs((700,), 1003, torch.bfloat16, seed=seed)[0])
            mask.copy_(inputs((700,), 1003, torch.bfloat16, seed=seed)[5])
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step()):
            assert torch.equal(p, q), seed
        torch.cuda.synchronize()


def test_offsets_beyond_32_bits():
    from step_amd import losses
    classes = 32000
    rows = (1 << 31) // classes + 5
    z = torch.zeros(rows, classes, dtype=torch.bfloat16, device=D)
    tail, a4, old4, adv4, _, _ = inputs((4,), classes, torch.bfloat16)
    z[-4:] = tail
    mask = torch.zeros(rows, dtype=torch.bool, device=D)
    mask[-4:] = True
    a, old, adv = torch.zeros(rows, dtype=torch.int64, device=D), torch.zeros(rows, device=D), torch.zeros(rows, device=D)
    a[-4:], old[-4:], adv[-4:] = a4, old4, adv4
    leaf = z.requires_grad_(True)
    loss, logp, _ = losses.policy_loss(leaf, a, old, adv, mask=mask)
    (grad,) = torch.autograd.grad(loss, leaf)
    small, slp, _, sgrad = check(tail, a4, old4, adv4, None, None, beta=0.0)
    assert torch.equal(loss, small) and torch.equal(logp[-4:], slp) and torch.equal(grad[-4:], sgrad)
    assert not grad[-6:-4].any() and not grad[0].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [4, 100, 4000, 70003, 140001])
def test_the_lowest_values_as_masks(classes, dtype):
    """classes shut out with the type's lowest value, which times log2 e is beyond fp32; a row that shuts out all of them is
    uniform, by the definition"""
    z, a, old, adv, ref, _ = inputs((5,), classes, dtype, seed=classes)
    lowest = torch.finfo(dtype).min
    z[1, 1:] = lowest
    a[1] = 0
    z[2] = lowest
    z[3, : classes // 2] = lowest
    z[4, -1] = torch.finfo(dtype).max
    a[3:] = classes - 1
    lp = torch.log_softmax(z.double(), 1).gather(1, a[:, None])[:, 0]
    check(z, a, (lp + 0.1).float(), adv, (lp - 0.1).float(), None)


def test_a_captured_backward_without_its_forward(monkeypatch):
    """the forward ran eagerly, its gradient's memory is not the graph's: a backward under capture takes memory of its own and
    computes the gradient anew"""
    from step_amd import losses
    z, a, old, adv, ref, mask = inputs((60,), 333, torch.bfloat16)
    leaf = z.clone().requires_grad_(True)
    loss = losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)[0]
    held = loss.grad_fn.grad.data_ptr()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    (captured,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert captured.data_ptr() != held
    monkeypatch.undo()
    again = losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)[0]
    held = again.grad_fn.grad.data_ptr()
    (want,) = torch.autograd.grad(again, leaf)
    assert want.data_ptr() == held and torch.equal(captured, want)


@pytest.mark.parametrize("classes", [300, 140001])
@pytest.mark.parametrize("masked", [True, False])
def test_a_graph_of_the_backward_alone(classes, masked):
    """the forward ran eagerly and is gone, its memory taken for something else, when the graph is replayed: each replay is the gradient
    of the caller's tensors as they are then"""
    from step_amd import losses
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        z, a, old, adv, ref, mask = inputs((90,), classes, torch.bfloat16)
        mask = mask if masked else None
        leaf, up = z.requires_grad_(True), torch.ones((), device=D)
        loss = losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)[0]
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            (grad,) = torch.autograd.grad(loss, leaf, up)
        del loss
        torch.cuda.synchronize()
        taken = [torch.full((n,), float("nan"), device=D) for n in [64] * 50 + [1 << 14] * 50 + [1 << 22] * 8]   # what the forward gave back
        for k, scale in enumerate((1.0, 2.0, 1.0, 0.5)):
            fresh = inputs((90,), classes, torch.bfloat16, seed=10 + k)
            with torch.no_grad():
                for t, f in zip((leaf, a, old, adv, ref, mask), fresh):
                    if t is not None:
                        t.copy_(f)
                up.fill_(scale)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            again = losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)[0]
            (want,) = torch.autograd.grad(again, leaf, up)
            assert torch.equal(grad, want), (k, scale)
            torch.cuda.synchronize()
        assert all(bool(t.isnan().all()) for t in taken)


def test_a_graph_of_the_backward_alone_takes_no_copies():
    from step_amd import losses
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        z, a, old, adv, some, _ = inputs((40,), 50, torch.float32)
        leaf = z.requires_grad_(True)
        for args in ((a.int(), old, adv), (a, old.double(), adv), (a, old, adv[:1])):
            loss = losses.policy_loss(leaf, *args)[0]
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                with pytest.raises(losses._lib.StepHipError, match="captured without its forward"):
                    torch.autograd.grad(loss, leaf, retain_graph=True)
                some.add_(1.0)                                # (so that the graph holds something)
            side.synchronize()
            torch.autograd.grad(loss, leaf)                   # eagerly it has no such needs


def test_forward_and_backward_in_two_graphs():
    """the backward's graph replayed more often than the forward's, with other upstream gradients"""
    from step_amd import losses
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        z, a, old, adv, ref, mask = inputs((70,), 700, torch.float32)
        a = a.int()                                           # a copy is made, in the forward's graph
        leaf, up = z.requires_grad_(True), torch.ones((), device=D)
        losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)
        side.synchronize()
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first, stream=side):
            loss = losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)[0]
        with torch.cuda.graph(second, stream=side, pool=first.pool()):
            (grad,) = torch.autograd.grad(loss, leaf, up)
        for seed, scales in ((5, (1.0, 2.0, 1.0)), (6, (3.0, 1.0)), (7, (1.0,))):
            with torch.no_grad():
                for t, f in zip((leaf, a, old, adv, ref, mask), inputs((70,), 700, torch.float32, seed=seed)):
                    t.copy_(f)
            first.replay()
            for scale in scales:
                up.fill_(scale)
                second.replay()
                torch.cuda.synchronize()
                again = losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)[0]
                (want,) = torch.autograd.grad(again, leaf, up)
                assert torch.equal(loss, again) and torch.equal(grad, want), (seed, scale)
                grad.zero_()                                  # the caller's to change
                torch.cuda.synchronize()


def test_an_eager_backward_of_a_captured_forward():
    """its gradient is not the graph's memory, which the next replay writes again"""
    from step_amd import losses
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        z, a, old, adv, ref, mask = inputs((70,), 700, torch.float32)
        leaf = z.requires_grad_(True)
        losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)[0]
        graph.replay()
        (grad,) = torch.autograd.grad(loss, leaf)
        (want,) = torch.autograd.grad(losses.policy_loss(leaf, a, old, adv, ref, mask, beta=0.05)[0], leaf)
        assert torch.equal(grad, want)
        adv.neg_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want)


@pytest.mark.parametrize("classes", [5, 300, 4000, 20000, 70003, 140001])
def test_small_probabilities_of_fp32_rows(classes):
    """gradients of classes far below the maximum, which is 0 so that no difference is rounded.  In units of u: the exponential 2, the
    exponent's correction 2 (an fp32 ln 2 times at most 46), roundings of its two products, the scale, its sum and division 6, the
    sum's smallest terms (127 a thread at most, under 8e-10 each) 2: 12 u of each element"""
    from step_amd import losses
    g = torch.Generator().manual_seed(classes)
    rows = max(3, 60000 // classes)
    z = (-32 + 11 * torch.rand(rows, classes, generator=g)).to(D)
    a = torch.randint(0, classes, (rows,), generator=g).to(D)
    z[torch.arange(rows), a] = 0
    old, adv = (0.05 * torch.randn(rows, generator=g)).to(D), torch.randn(rows, generator=g).to(D)
    leaf = z.requires_grad_(True)
    (grad,) = torch.autograd.grad(losses.policy_loss(leaf, a, old, adv)[0], leaf)
    _, _, _, ref, _, _ = reference(z, a, old, adv, None, None, 0.2, 0.2, 0.0)
    others = torch.ones_like(z, dtype=torch.bool)
    others[torch.arange(rows), a] = False
    off = (grad.double() - ref).abs()[others] / ref.abs()[others]
    assert float(off[ref[others] != 0].max()) <= 12 * U, float(off[ref[others] != 0].max()) / U


@pytest.mark.parametrize("rows,classes,dtype", [(20000, 7, torch.float32), (20000, 613, torch.float32), (20000, 613, torch.bfloat16), (20000, 4000, torch.float32),
                                                (8000, 20000, torch.float32), (8000, 50257, torch.float32), (4000, 100003, torch.float32),
                                                (4000, 140001, torch.bfloat16)])
def test_log_probabilities_have_no_bias(rows, classes, dtype):
    """the mean of the signed errors.  A row's error has no sign of its own: the result's rounding, uniform within 2^-21 for a log
    probability under 16 (a standard deviation of 2.8e-7), and the sum's, under 2 u; over the rows 3e-7 / root of rows, of which
    four, and 2e-9.  (The exponential of the hardware leans by up to 1e-8, which leaves two of the four.)"""
    from step_amd import losses
    g = torch.Generator(D).manual_seed(classes)
    z = (2 * torch.randn(rows, classes, device=D, generator=g)).to(dtype)
    a = torch.randint(0, classes, (rows,), device=D, generator=g)
    zero = torch.zeros(rows, device=D)
    _, logp, _ = losses.policy_loss(z, a, zero, zero)
    bias = []
    for k in range(0, rows, 1000):
        part = z[k:k + 1000].double()
        bias.append((logp[k:k + 1000].double() - (part.gather(1, a[k:k + 1000, None])[:, 0] - torch.logsumexp(part, 1))).sum())
    bias = float(sum(bias)) / rows
    assert abs(bias) <= 4 * 3e-7 / rows ** 0.5 + 2e-9, bias


def test_a_loss_whose_terms_cancel():
    """65536 rows whose terms cancel to 1e-4 of their size: the loss is good to 1e-5, that is to 1e-9 of the terms (a row's ratio is off
    by u at random, of the mean over the rows four standard deviations are 9.3e-10, and its one rounding is 6e-12)"""
    from step_amd import losses
    g = torch.Generator(D).manual_seed(1)
    rows, classes = 65536, 372
    z = 2 * torch.randn(rows, classes, device=D, generator=g)
    a = torch.randint(0, classes, (rows,), device=D, generator=g)
    lp = torch.log_softmax(z.double(), 1).gather(1, a[:, None])[:, 0]
    old = (lp + 0.05 * torch.randn(rows, device=D, generator=g)).float()
    adv = torch.randn(rows, device=D, generator=g)
    rho = torch.exp(lp - old.double())
    adv = adv - (rho.clamp(0.8, 1.2) * adv.double()).mean().float() + 1e-4     # (ratios within the clipping: terms rho A)
    loss, _, stats = losses.policy_loss(z, a, old, adv)
    terms = torch.minimum(rho * adv.double(), rho.clamp(0.8, 1.2) * adv.double())
    want, size = -float(terms.mean()), float(terms.square().mean().sqrt())
    assert abs(want) <= 1e-3 * size
    assert abs(float(loss) - want) <= 4 * U / rows ** 0.5 * size + U * abs(want), (float(loss), want)
