"""CPU: what the layer norm, the policy loss, newton_schulz and Muon refuse, in Python and at the C ABI, before any launch."""
import ctypes

import pytest
import torch

from step_amd import _lib, losses, ops, optim
from step_amd._lib import StepHipError

PTR = ctypes.c_void_p(4096)          # never followed: every call below is refused on the host


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3)
    with pytest.raises(StepHipError, match="no CPU path"):
        ops.layer_norm(x)
    with pytest.raises(StepHipError, match="no CPU path"):
        losses.policy_loss(x, torch.zeros(2, dtype=torch.int64), torch.zeros(2), torch.zeros(2))
    with pytest.raises(StepHipError, match="no CPU path"):
        optim.newton_schulz(x)
    p = torch.nn.Parameter(x)
    p.grad = torch.zeros(2, 3)
    with pytest.raises(StepHipError, match="no CPU path"):
        optim.Muon([p]).step()


@pytest.mark.parametrize("kw,what", [
    (dict(x=torch.zeros(2, 3, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(2, 3, dtype=torch.int32)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(())), "no last axis"),
    (dict(x=torch.zeros(2, 0)), "no last axis"),
    (dict(x=torch.zeros(2, 3), weight=torch.zeros(4)), "does not fit"),
    (dict(x=torch.zeros(2, 3), bias=torch.zeros(1, 3)), "does not fit"),
    (dict(x=torch.zeros(2, 3), weight=torch.zeros(3, dtype=torch.bfloat16)), "wanted"),
    (dict(x=torch.zeros(2, 3, dtype=torch.bfloat16), weight=torch.zeros(3), bias=torch.zeros(3, dtype=torch.bfloat16)), "weight is"),
])
def test_layer_norm_refusals(kw, what):
    with pytest.raises(StepHipError, match=what):
        ops.layer_norm(**kw)


def policy(**kw):
    args = dict(logits=torch.zeros(4, 5), actions=torch.zeros(4, dtype=torch.int64), old_logp=torch.zeros(4), advantages=torch.zeros(4))
    args.update(kw)
    return losses.policy_loss(**args)


@pytest.mark.parametrize("kw,what", [
    (dict(logits=torch.zeros(4, 5, dtype=torch.float64)), "logits wanted"),
    (dict(logits=torch.zeros(4, 0)), "classes"),
    (dict(actions=torch.zeros(4)), "actions"),
    (dict(actions=torch.zeros(5, dtype=torch.int64)), "does not fit"),
    (dict(old_logp=torch.zeros(4, dtype=torch.int64)), "old_logp"),
    (dict(advantages=torch.zeros(2, 4)), "does not fit"),
    (dict(advantages=None), "advantages"),
    (dict(ref_logp=torch.zeros(3)), "does not fit"),
    (dict(mask=torch.zeros(4)), "mask"),
    (dict(mask=torch.zeros(4, dtype=torch.uint8)), "mask"),
    (dict(clip=-0.1), "clip"),
    (dict(clip=(1.5, 0.2)), "clip"),
    (dict(clip=float("nan")), "clip"),
    (dict(logits=torch.zeros(4, 5, device="meta")), "is on"),
])
def test_policy_loss_refusals(kw, what):
    with pytest.raises(StepHipError, match=what):
        policy(**kw)


@pytest.mark.parametrize("g,kw,what", [
    (torch.zeros(3), {}, "matrices"),
    ([torch.zeros(3, 3), 4], {}, "matrices"),
    (torch.zeros(3, 3, dtype=torch.float64), {}, "float32, bfloat16 or float16"),
    ([torch.zeros(3, 3), torch.zeros(3, 3, dtype=torch.bfloat16)], {}, "one type"),
    (torch.zeros(3, 3), dict(steps=0), "steps"),
    (torch.zeros(3, 3), dict(steps=2.0), "steps"),
    (torch.zeros(3, 3), dict(eps=-1.0), "eps"),
    (torch.zeros(3, 3), dict(eps=float("nan")), "eps"),
])
def test_newton_schulz_refusals(g, kw, what):
    with pytest.raises(StepHipError, match=what):
        optim.newton_schulz(g, **kw)


def test_muon_refusals():
    p = torch.nn.Parameter(torch.zeros(2, 2))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(adam_lr=-1.0)):
        with pytest.raises(ValueError):
            optim.Muon([p], **kw)
    half = torch.nn.Parameter(torch.zeros(2, 2, dtype=torch.bfloat16))
    half.grad = torch.zeros_like(half)
    with pytest.raises(StepHipError, match="fp32"):
        optim.Muon([half]).step()
    opt = optim.Muon([p])
    assert opt.step() is None and not opt.state               # nothing to do without a gradient


def code(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.step_last_error().decode()


def test_layer_norm_abi():
    ok = (PTR, None, None, PTR, None, None, 4, 8, 0, 0, 1e-5, None)
    for i, bad in ((0, None), (3, None), (4, PTR), (6, 0), (7, 0), (8, 3), (9, -1)):
        args = list(ok)
        args[i] = bad
        rc, msg = code("step_layernorm_fwd", *args)
        assert rc == -1 and "step_layernorm_fwd" in msg, i
    nb = _lib.query("step_layernorm_bwd_ws_bytes", 4, 8)
    ok = (PTR, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 4, 8, 0, 0, PTR, nb, None)
    for i, bad, rcode in ((0, None, -1), (1, None, -1), (3, None, -1), (4, None, -1), (8, 0, -1), (9, -5, -1), (10, 7, -1), (12, None, -1),
                          (13, nb - 1, -3)):
        args = list(ok)
        args[i] = bad
        rc, msg = code("step_layernorm_bwd", *args)
        assert rc == rcode and "step_layernorm_bwd" in msg, i
    assert _lib.query("step_layernorm_bwd_ws_bytes", 0, 8) == 0
    # every launch's lines of partial sums fit, the longest rows' as well
    assert _lib.query("step_layernorm_bwd_ws_bytes", 1 << 40, 100000) >= 512 * 2 * 100000 * 4


def test_policy_loss_abi():
    nb = _lib.query("step_policy_loss_ws_bytes", 4, 8)
    ok = (PTR, PTR, PTR, PTR, None, None, 0.2, 0.2, 0.0, None, 0, PTR, PTR, PTR, PTR, 4, 8, 0, PTR, nb, None)
    for i, bad, rcode in ((0, None, -1), (1, None, -1), (2, None, -1), (3, None, -1), (11, None, -1), (12, None, -1), (13, None, -1), (15, 0, -1),
                          (16, 0, -1), (17, 9, -1), (18, None, -1), (19, nb - 1, -3), (14, ctypes.c_void_p(4098), -1), (0, ctypes.c_void_p(4098), -1)):
        args = list(ok)
        args[i] = bad
        rc, msg = code("step_policy_loss", *args)
        assert rc == rcode and "step_policy_loss" in msg, i
    args = list(ok)
    args[9], args[14] = PTR, None                             # a backward without a place for its gradient
    assert code("step_policy_loss", *args)[0] == -1


def test_newton_schulz_abi():
    def items(*shapes, **kw):
        base = dict(g=4096, out=4096, momentum=None, param=None, scale=1.0)
        base.update(kw)
        return (_lib.NsItem * len(shapes))(*[_lib.NsItem(base["g"], base["out"], base["momentum"], base["param"], *s, base["scale"]) for s in shapes])

    def call(it, n, dtype=0, steps=5, ws=PTR, nb=1 << 40):
        return code("step_newton_schulz", it, n, dtype, steps, 1e-7, 0.0, 0, 0.0, 0.0, ws, nb, None)

    good = items((1, 8, 8))
    assert call(good, 0)[0] == -1 and call(None, 1)[0] == -1
    for shape in ((0, 8, 8), (1, 0, 8), (1, 8, -1), (1, 1 << 23, 8), (1, 40000, 40000)):
        rc, msg = call(items(shape), 1)
        assert rc == -1 and "step_newton_schulz" in msg, shape
        assert _lib.query("step_newton_schulz_ws_bytes", items(shape), 1) == 0
    assert call(good, 1, dtype=5)[0] == -1 and call(good, 1, steps=0)[0] == -1 and call(good, 1, steps=101)[0] == -1
    assert call(good, 1, ws=None)[0] == -1 and call(good, 1, nb=16)[0] == -3
    assert call(items((1, 8, 8), g=None), 1)[0] == -1 and call(items((1, 8, 8), out=None), 1)[0] == -1
    assert call(items((1, 8, 8), momentum=4096), 1, dtype=1)[0] == -1      # the optimizer's form takes fp32
    # the workspace covers the largest group and the largest matrix of a list
    one, big = _lib.query("step_newton_schulz_ws_bytes", good, 1), _lib.query("step_newton_schulz_ws_bytes", items((1, 300, 5000)), 1)
    assert _lib.query("step_newton_schulz_ws_bytes", items((1, 8, 8), (1, 300, 5000)), 2) == max(one, big)


def test_harness_and_head_arguments():
    from step_amd.net.classifier_hybrid import Classifier
    with pytest.raises(ValueError, match="head_norm"):
        Classifier(3, 29, 4, {"strategy": "spatial"}, head_norm="group")
    plain, layer = (Classifier(3, 29, 4, {"strategy": "spatial"}, **kw).state_dict() for kw in ({}, {"head_norm": "layer"}))
    assert set(plain) - set(layer) == {"data_bn2.running_mean", "data_bn2.running_var", "data_bn2.num_batches_tracked"}
    assert not set(layer) - set(plain)


def test_sizes_beyond_the_library_are_refused():
    """whose counts are C ints: nothing is cut off silently"""
    huge = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="meta")  # noqa: E731
    with pytest.raises(StepHipError, match="columns"):
        ops.layer_norm(huge(1, (1 << 32) + 5))
    with pytest.raises(StepHipError, match="classes"):
        losses.policy_loss(huge(1, (1 << 32) + 5), huge(1), huge(1), huge(1))
    for shape in ((1, (1 << 32) + 5), ((1 << 32) + 5, 3), ((1 << 32) + 1, 2, 2)):
        with pytest.raises(StepHipError, match="at most"):
            optim.newton_schulz(huge(*shape))
    for name, at in (("step_layernorm_fwd", 7), ("step_policy_loss", 16)):
        args = {"step_layernorm_fwd": [PTR, None, None, PTR, None, None, 4, 8, 0, 0, 1e-5, None],
                "step_policy_loss": [PTR, PTR, PTR, PTR, None, None, 0.2, 0.2, 0.0, None, 0, PTR, PTR, PTR, PTR, 4, 8, 0, PTR, 1 << 20, None]}[name]
        args[at] = (1 << 31) - 1
        assert code(name, *args)[0] == -1


def test_policy_logits_of_a_saturated_softmax():
    """a model that answers with probabilities, one of them gone to zero: finite logits, finite gradients"""
    from step_amd.harness import EpochRunner

    class Sure:
        RETURNS_SOFTMAX = True

        def __call__(self, x):
            return torch.softmax(x, 1), None
    x = torch.tensor([[0.0, -200.0, 1.0]], requires_grad=True)
    logits = EpochRunner._logits(None, Sure(), x)
    (logits * torch.tensor([[1.0, -1.0, 0.5]])).sum().backward()
    assert bool(logits.isfinite().all()) and bool(x.grad.isfinite().all())
    assert torch.equal(logits[0, 0], torch.log(torch.softmax(x, 1))[0, 0])


def ns_bytes(*shapes):
    return _lib.query("step_newton_schulz_ws_bytes", (_lib.NsItem * len(shapes))(*[_lib.NsItem(4096, 4096, None, None, *s, 1.0) for s in shapes]), len(shapes))


@pytest.mark.parametrize("shapes", [
    [(1000000, 4, 4)], [(1 << 24, 2, 2)], [(1 << 20, 64, 64)], [(600, 64, 1 << 21)], [(1, 64, 1 << 21), (512, 8, 8)],
    [(512, 8, 8), (1, 64, 1 << 21), (5000, 30, 200)], [(300, 20, 40)] * 100, [(4095, 3, 3), (2, 3, 3), (4096, 3, 3), (4097, 3, 3)]])
def test_the_workspace_of_many_small_matrices_is_bounded(shapes):
    """they are taken in groups, at most 4096 matrices each, of 6656 fp64 numbers (a chunk's sums, P) and of 31 more chunks of 2560 where
    fewer than 1024 matrices share the card"""
    assert 0 < ns_bytes(*shapes) <= 8 * (4096 * 6656 + 1024 * 2560)
    assert ns_bytes(*shapes) >= 8 * 6656 * min(sum(s[0] for s in shapes), 500)


def test_a_captured_backward_of_copies_is_refused(monkeypatch):
    """on the host, before any launch: the copies that the eager forward made are not the caller's to keep until a replay"""
    from types import SimpleNamespace
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(_lib, "capture", lambda device: 7)
    z = torch.zeros(4, 5)
    for copied, capture, refused in ((True, None, True), (False, None, False), (True, 3, False), (True, 7, False)):
        ctx = SimpleNamespace(saved_tensors=(z,) * 6, grad=torch.zeros(4, 5), ws=torch.zeros(8, dtype=torch.uint8), capture=capture, copied=copied,
                              config=(0.2, 0.2, 0.0))
        what = "captured without its forward" if refused else "no CPU path"      # (what follows is the launch, which takes no CPU tensors)
        with pytest.raises(StepHipError, match=what):
            losses._PolicyLossFn.backward(ctx, torch.ones(()), None, None)


def test_no_capture_without_a_gpu():
    assert _lib.query("step_capture_id", None) == 0
