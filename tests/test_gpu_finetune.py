"""GPU: the layer norm, the policy loss and the orthogonalised update together, as a training program has them."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
D = torch.device("cuda:0")


def test_one_step_of_norm_loss_and_update():
    """a step of a two-layer head (layer norm, product, policy loss, Muon) against the same in 64 bits.  fp32 throughout: the
    gradients are held to 1e-4 of their largest (a product's fp32 sums and the operators' own bounds), the updates to 2e-3 of
    theirs (an orthogonalisation enlarges its input's error by its condition)"""
    from step_amd import losses, ops, optim
    g = torch.Generator().manual_seed(5)
    N, F, H, Cls = 256, 93, 48, 4
    x = torch.randn(N, F, generator=g)
    w1, w2 = torch.randn(H, F, generator=g) / F ** 0.5, torch.randn(Cls, H, generator=g) / H ** 0.5
    nw, nb = 1 + 0.1 * torch.randn(F, generator=g), 0.1 * torch.randn(F, generator=g)
    a = torch.randint(0, Cls, (N,), generator=g)
    adv, noise = torch.randn(N, generator=g), 0.1 * torch.randn(N, generator=g)

    def forward(x, nw, nb, w1, w2, norm):
        return torch.tanh(norm(x, nw, nb) @ w1.t()) @ w2.t()

    ref_norm = lambda t, w, b: (t - t.mean(1, keepdim=True)) / torch.sqrt(t.var(1, unbiased=False, keepdim=True) + 1e-5) * w + b  # noqa: E731
    leaves = [t.double().requires_grad_(True) for t in (nw, nb, w1, w2)]
    z = forward(x.double(), *leaves, ref_norm)
    lp = torch.log_softmax(z, 1).gather(1, a[:, None])[:, 0]
    old = lp.detach() + noise
    rho = torch.exp(lp - old)
    d = old - lp
    loss = (-torch.minimum(rho * adv, rho.clamp(0.8, 1.2) * adv) + 0.05 * (torch.exp(d) - d - 1)).mean()
    want = torch.autograd.grad(loss, leaves)

    params = [torch.nn.Parameter(t.to(D)) for t in (nw, nb, w1, w2)]
    opt = optim.Muon(params, lr=0.02, momentum=0.0, nesterov=False, adam_lr=1e-3)
    old32 = old.float().to(D)
    got, logp, _ = losses.policy_loss(forward(x.to(D), *params, ops.layer_norm), a.to(D), old32, adv.to(D), old32, beta=0.05)
    got.backward()
    assert abs(float(got) - float(loss)) <= 1e-5
    for p, r in zip(params, want):
        assert float((p.grad.cpu().double() - r).abs().max()) <= 1e-4 * float(r.abs().max())
    before = [p.detach().clone() for p in params]
    opt.step()
    for p, b, r in zip(params[2:], before[2:], want[2:]):
        u = r / r.norm()
        for _ in range(5):
            s = u @ u.t()
            u = 3.4445 * u - 4.7750 * (s @ u) + 2.0315 * (s @ (s @ u))
        u = 0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * u
        assert float((b.cpu().double() - p.detach().cpu().double() - u).norm()) <= 2e-3 * float(u.norm())
    for p, b in zip(params[:2], before[:2]):
        assert float((p.detach() - b).abs().max()) <= 1.001e-3 and not torch.equal(p.detach(), b)


def test_hybrid_classifier_steps_with_all_three():
    from step_amd import losses, optim
    from step_amd.net.classifier_hybrid import Classifier
    torch.manual_seed(0)
    m = Classifier(3, 29, 4, {"strategy": "spatial"}, head_norm="layer").to(D).train()
    opt = optim.Muon([{"params": [p for p in m.parameters() if p.dim() == 4]},
                      {"params": [p for p in m.parameters() if p.dim() != 4], "matrices": False}], lr=0.01)
    xa, xg = torch.randn(8, 29, device=D), 0.3 * torch.randn(8, 3, 75, 16, 1, device=D)
    a = torch.arange(8, device=D) % 4
    old, adv = torch.full((8,), -1.4, device=D), torch.linspace(-1, 1, 8, device=D)
    mask = torch.tensor([True] * 7 + [False], device=D)
    for _ in range(3):
        loss, logp, stats = losses.policy_loss(m(xa, xg), a, old, adv, old, mask, beta=0.04)
        opt.zero_grad()
        loss.backward()
        grads = [p.grad.clone() for p in m.parameters()]
        before = copy.deepcopy(m.state_dict())
        opt.step()
        assert torch.isfinite(loss) and all(torch.isfinite(x).all() for x in grads)
        moved = [k for k, v in m.named_parameters() if not torch.equal(v, before[k])]
        assert len(moved) == len(list(m.parameters()))


@pytest.mark.parametrize("variant", ["classifier", "classifier_real_and_synth"])
def test_harness_with_muon_and_rewards(tmp_path, variant):
    import importlib
    from step_amd import harness
    mod = importlib.import_module("step_amd.net." + variant)
    torch.manual_seed(0)
    model = mod.Classifier(3, 4, {"strategy": "spatial"})
    train, test = harness.synthetic_gaits(40, 75, 4, 0, test_size=0.25)
    run = harness.EpochRunner(model, train, test, str(tmp_path), 2, batch_size=8, base_lr=0.02, optimizer="Muon")
    hist = run.train()
    assert len(hist) == 2 and all(torch.isfinite(p).all() for p in model.parameters())
    before = [p.detach().clone() for p in model.parameters()]
    loss, reward = run.per_policy(lambda data, drawn, label: drawn == label)
    assert loss == loss and 0.0 <= reward <= 1.0
    assert any(not torch.equal(p, b) for p, b in zip(model.parameters(), before))
    run.load_best_model()
