"""GPU: step_amd.ops.layer_norm against the definition in 64 bits.

Tolerances.  u = 2^-24 is fp32's half step, h the half step of the tensors' type (fp32 2^-24, bf16 2^-8, fp16 2^-11, relative to
the value).  A result is rounded once to its type: h |ref|.  Before that, sums over a row have chains of at most 64 additions
(32 values a thread, then a tree), so a mean is off by at most 64 u times the mean of the absolute values, a sum over rows of
length R by (R + 64) u times the sum of the absolute values; every other operation adds a few u.  `K` u with K = 80 covers the
chain and those.  The bounds are per element, in the terms that the formula adds up."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = torch.device("cuda:0")
U, K = 2.0 ** -24, 80
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def formula(x, w, b, dy, eps):
    """y, dx, dw, db in 64 bits and the bounds of their errors before the final rounding"""
    x, dy = x.double(), dy.double()
    w = torch.ones_like(x[0]) if w is None else w.double()
    b = torch.zeros_like(x[0]) if b is None else b.double()
    C = x.shape[1]
    mu = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mu) * r
    e_xh = K * U * (x.abs().mean(1, keepdim=True) * r + xh.abs() + 1e-30)        # of the mean, then relative
    t = dy * w
    m1, m2 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
    dx = r * (t - m1 - xh * m2)
    e_m2 = K * U * (t * xh).abs().mean(1, keepdim=True) + (t.abs() * e_xh).mean(1, keepdim=True)
    e_dx = r * (K * U * (t.abs() + t.abs().mean(1, keepdim=True) + (xh * m2).abs()) + e_xh * m2.abs() + xh.abs() * e_m2)
    R = x.shape[0]
    e_dw = (R + 64) * U * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)
    e_db = (R + 64) * U * dy.abs().sum(0)
    return (xh * w + b, dx, (dy * xh).sum(0), dy.sum(0)), (e_xh * w.abs() + 4 * U * (xh * w).abs() + 2 * U * b.abs(), e_dx, e_dw, e_db)


def within(got, ref, bound, what):
    assert torch.isfinite(got).all(), what
    # below a type's normal numbers a rounding is half of its smallest number
    lim = bound + half_step(got.dtype) * (ref.abs() + bound) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double() - ref).abs()
    assert bool((off <= lim).all()), "%s: %.3e over its bound" % (what, float((off / lim).max()))


def inputs(rows, cols, dtype, wdtype, seed=0, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(rows, 1, generator=g)) + offset).to(dtype).to(D)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(wdtype).to(D)
    b = (0.2 * torch.randn(cols, generator=g)).to(wdtype).to(D)
    dy = torch.randn(rows, cols, generator=g).to(dtype).to(D)
    return x, w, b, dy


def check(x, w, b, dy, eps=1e-5):
    from step_amd import ops
    leaves = [t.clone().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    y.backward(dy)
    C = x.shape[-1]
    refs, bounds = formula(x.reshape(-1, C), w, b, dy.reshape(-1, C), eps)
    got = [y.detach().reshape(-1, C), leaves[0].grad.reshape(-1, C)] + [t.grad if t is not None else None for t in leaves[1:]]
    for name, a, r, e in zip(("y", "dx", "dw", "db"), got, refs, bounds):
        if a is not None:
            within(a, r, e, name)


# sizes about every border of the choice of threads per row: 8 / 64 / 256 / 1024 threads, packs of 16 bytes and single elements
SHAPES = [(1, 1), (3, 2), (5, 16), (33, 17), (600, 31), (7, 64), (4096, 93), (9, 127), (11, 128), (5, 129), (3, 512), (2, 513), (70, 1000),
          (2, 1024), (3, 2048), (2, 2187), (5, 4096), (2, 4104), (3, 8192), (2, 8193), (2, 16384), (3, 16385), (2, 20000), (1, 40001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_gradients(rows, cols, dtype):
    check(*inputs(rows, cols, dtype, dtype, seed=rows + cols))


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_fp32_weights_beside_16_bit_rows(dtype):
    check(*inputs(37, 200, dtype, torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_without_weight_or_bias(dtype):
    x, w, b, dy = inputs(19, 136, dtype, dtype)
    check(x, None, None, dy)
    check(x, w, None, dy)
    check(x, None, b, dy)


def test_leading_axes_strides_and_offsets():
    x, w, b, dy = inputs(24, 120, torch.float32, torch.float32)
    check(x.view(2, 3, 4, 120), w, b, dy.view(2, 3, 4, 120))
    check(x[0], w, b, dy[0])
    wide = torch.randn(24, 140, device=D)
    check(wide[:, 3:123], w, b, dy)                          # strided rows
    flat = torch.randn(24 * 120 + 1, device=D)
    check(flat[1:].view(24, 120), w, b, dy)                  # rows that start off 16 bytes
    check(x.t().contiguous().t(), w, b, dy)                  # transposed storage
    check(x[:1].expand(24, 120), w, b, dy)                   # one row, many times
    check(x, w, b, torch.ones((), device=D).expand(24, 120))  # a broadcast gradient


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_far_from_zero_and_constant_rows(dtype):
    offset = 1000.0 if dtype == torch.float32 else 50.0
    check(*inputs(9, 300, dtype, dtype, offset=offset))
    x, w, b, dy = inputs(4, 300, dtype, dtype)
    x[1] = 7.0                                               # no variance: eps alone
    x[2] = 0.0
    check(x, w, b, dy)


def test_a_row_is_the_same_in_any_batch_and_every_time():
    from step_amd import ops
    x, w, b, dy = inputs(5000, 200, torch.bfloat16, torch.bfloat16)
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y[4321:4322], ops.layer_norm(x[4321:4322], w, b))
    grads = []
    for _ in range(2):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        ops.layer_norm(*leaves).backward(dy)
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(p, q) for p, q in zip(*grads))


def test_nan_and_inf_stay_in_their_rows():
    from step_amd import ops
    x, w, b, _ = inputs(6, 250, torch.float32, torch.float32)
    clean = ops.layer_norm(x, w, b)
    x[2, 7], x[4, 0] = float("nan"), float("inf")
    y = ops.layer_norm(x, w, b)
    assert bool(y[2].isnan().all()) and bool(y[4].isnan().any())
    for r in (0, 1, 3, 5):
        assert torch.equal(y[r], clean[r])


def test_partial_gradients_and_empty_batches():
    from step_amd import ops
    x, w, b, dy = inputs(12, 40, torch.float32, torch.float32)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(ops.layer_norm(x, w, b), (w,), dy)
    refs, bounds = formula(x, w.detach(), b, dy, 1e-5)
    within(dw, refs[2], bounds[2], "dw")
    x0 = torch.empty(0, 40, device=D, requires_grad=True)
    y = ops.layer_norm(x0, w, b)
    y.sum().backward()
    assert y.shape == (0, 40) and x0.grad.shape == (0, 40) and float(w.grad.abs().max()) == 0.0


def test_gradient_against_differences():
    """loss = <dy, y>: the central difference along a direction, whose error is the fp32 noise of two losses over 2 h (about
    1e-6 sqrt(n) / 2h) plus h^2 of the third derivative"""
    from step_amd import ops
    x, w, b, dy = inputs(8, 96, torch.float32, torch.float32)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.layer_norm(x, w, b), (x,), dy)
    v = torch.randn(8, 96, generator=torch.Generator().manual_seed(9)).to(D)
    h = 1e-2
    loss = lambda t: float((ops.layer_norm(t, w, b).double() * dy.double()).sum())  # noqa: E731
    num = (loss(x.detach() + h * v) - loss(x.detach() - h * v)) / (2 * h)
    ref = float((dx.double() * v.double()).sum())
    scale = float((dx.double().abs() * v.double().abs()).sum())
    assert abs(num - ref) <= 5e-3 * scale


def test_captured_and_on_another_stream():
    from step_amd import ops
    x, w, b, dy = inputs(300, 264, torch.bfloat16, torch.bfloat16)
    xs, dys = x.clone(), dy.clone()
    leaves = [xs.requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]

    def step():
        y = ops.layer_norm(*leaves)
        return (y,) + torch.autograd.grad(y, leaves, dys)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ref = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        with torch.no_grad():
            xs.copy_(inputs(300, 264, torch.bfloat16, torch.bfloat16, seed=seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        ref = step()
        for p, q in zip(out, ref):
            assert torch.equal(p, q), seed
        torch.cuda.synchronize()


def test_offsets_beyond_32_bits():
    from step_amd import ops
    rows, cols = (1 << 31) // 4096 + 3, 4096                 # 2^31 + 12288 elements
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=D)
    tail, w, b, dy = inputs(4, cols, torch.bfloat16, torch.bfloat16)
    x[-4:] = tail
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y[-4:], ops.layer_norm(tail, w, b))
    assert torch.equal(y[0], b)


def test_hybrid_classifier_with_a_layer_norm_head():
    """logits of one gait do not change with its batch, training takes a batch of one, every parameter gets a gradient"""
    from step_amd.net.classifier_hybrid import Classifier
    torch.manual_seed(0)
    m = Classifier(3, 29, 4, {"strategy": "spatial"}, head_norm="layer").to(D)
    assert {k for k in m.state_dict() if k.startswith("data_bn2")} == {"data_bn2.weight", "data_bn2.bias"}
    xa, xg = torch.randn(5, 29, device=D), 0.3 * torch.randn(5, 3, 75, 16, 1, device=D)
    m.eval()
    with torch.no_grad():
        out = m(xa, xg)
        one = m(xa[3:4], xg[3:4])
    # what stands before the head is the same arithmetic for a gait, in tiles that the batch may move
    assert float((out[3] - one[0]).abs().max()) <= 1e-5 * float(out.abs().max())
    m.train()
    torch.nn.functional.cross_entropy(m(xa[:1], xg[:1]), torch.tensor([2], device=D)).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


@pytest.mark.parametrize("rows,cols,dtype", [(3, 1 << 26, torch.float32), (1, (1 << 28) - 3, torch.bfloat16), (2, (1 << 27) + 1, torch.float16)])
def test_the_longest_rows(rows, cols, dtype, monkeypatch):
    """up to the 2^28 columns that layer_norm takes: the weights' gradients are joined by fewer blocks than there are columns.  A
    thread's chain of additions is cols / 1024 long here, all in one direction at worst"""
    import sys
    monkeypatch.setattr(sys.modules[__name__], "K", K + cols / 1024)
    g = torch.Generator(D).manual_seed(cols)
    x, dy = (torch.randn(rows, cols, generator=g, device=D).to(dtype) for _ in range(2))
    w, b = ((1 + 0.3 * torch.randn(cols, generator=g, device=D)).to(dtype) for _ in range(2))
    check(x, w, b, dy)
    torch.cuda.empty_cache()
