"""Reference log-probabilities far below the policy's, in steps that count: -inf (what compute_action_log_probs gives for an
action that the reference forbids), the type's lowest value, and large finite ones.

With e = ref - log pi the KL term is e^e - 1 - e and its slope 1 - e^e, which tends to 1: finite however low the reference is.
Bounds (u = 2^-24): as for ordinary references (test_gpu_policy_loss.py): terms and slopes 3e-6 of the sizes that they are made of."""
import math

import pytest
import torch

import rl_triton.policy as policy
from _policy_reference import UNIT, logits_grad, policy_loss, softmax_rows

pytestmark = pytest.mark.gpu
LOW, HIGH, KL = 0.2, 0.3, 0.1
LOWEST = {"-inf": -math.inf, "lowest": None, "-1e9": -1e9, "-2e7": -2e7, "-100": -100.0}


@pytest.fixture(autouse=True, params=["0", "1"], ids=["fast", "checked"])
def _path(request, monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", request.param)


def _terms(lp, dtype, value, seed):
    g = torch.Generator().manual_seed(seed)
    E, T = lp.shape
    old = (lp.float() - torch.linspace(-0.15, 0.15, E * T).view(E, T)).to(dtype)  # (inside the clipping's bounds)
    adv = torch.randn(E, T, generator=g).to(dtype)
    ref = (lp.float() + torch.randn(E, T, generator=g) * 0.5).to(dtype)
    low = torch.rand(E, T, generator=g) < 0.3
    low[0, 0] = True
    ref[low] = torch.finfo(dtype).min if value is None else value
    mask = (torch.rand(E, T, generator=g) < 0.7).to(dtype)
    mask[0, 0] = 1
    return old, adv, ref, mask


def _close(got, want, bound):
    got, want = got.detach().cpu().double(), want.double()
    same = got == want  # (infinities)
    assert bool((same | ((got - want).abs() <= bound)).all()), (got[~same][:4], want[~same][:4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kl_coef", [KL, 0.0])
@pytest.mark.parametrize("name", LOWEST)
@pytest.mark.parametrize("E,T", [(1, 1), (5, 30), (40, 300)])
def test_from_log_probs(E, T, name, kl_coef, dtype):
    lp = torch.log(torch.rand(E, T, generator=torch.Generator().manual_seed(E)).clamp_min(1e-2)).to(dtype)
    old, adv, ref, mask = _terms(lp, dtype, LOWEST[name], T)
    for m in (None, mask):
        for reduction in ("steps", "rows"):
            loss, grad, means = policy.compute_policy_loss(*(t.cuda() for t in (lp, old, adv, ref)), LOW, HIGH, kl_coef,
                                                           mask=None if m is None else m.cuda(), reduction=reduction)
            _, _, wmeans, sizes, w = policy_loss(lp, old, adv, ref, m, LOW, HIGH, None, 0.0, reduction)
            wgrad = policy_loss(lp, old, adv, ref, m, LOW, HIGH, None, kl_coef, reduction)[1]
            want = wmeans[0] + (kl_coef * wmeans[1] if kl_coef else 0)
            _close(means, wmeans, torch.where(sizes.isfinite(), 6e-6 * sizes, 0.0) + 1e-30)
            _close(loss, want, 6e-6 * float(sizes[0] + (kl_coef * sizes[1] if kl_coef else 0)) + 1e-30)
            e = ref.double() - lp.double()
            size = w * (adv.double().abs() * (lp.double() - old.double()).exp() + kl_coef * (e.exp() + 1))
            unit = 0 if dtype == torch.float32 else UNIT[dtype]
            _close(grad, wgrad, 3e-6 * size + unit * wgrad.abs())
            assert bool(grad.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kl_coef", [KL, 0.0])
@pytest.mark.parametrize("name", LOWEST)
@pytest.mark.parametrize("A", [5, 18, 70, 1000, 140001])
def test_from_logits(A, name, kl_coef, dtype):
    E, T = (6, 20) if A <= 1000 else (1, 3)
    g = torch.Generator().manual_seed(A)
    x = (torch.randn(E, T, A, generator=g) * 2).to(dtype)
    a = torch.randint(0, A, (E, T), generator=g)
    lp, ent, p, logp = softmax_rows(x, a, 0.9)
    old, adv, ref, mask = _terms(lp.float(), torch.float32, LOWEST[name], A)
    loss, grad, means = policy.compute_policy_loss_from_logits(x.cuda(), a.cuda(), *(t.cuda() for t in (old, adv, ref)), LOW, HIGH, kl_coef,
                                                               0.0, 0.9, mask=mask.cuda())
    _, _, wmeans, sizes, w = policy_loss(lp, old, adv, ref, mask, LOW, HIGH, None, 0.0, "steps")
    slope = policy_loss(lp, old, adv, ref, mask, LOW, HIGH, None, kl_coef, "steps")[1]
    want = wmeans[0] + (kl_coef * wmeans[1] if kl_coef else 0)
    more = 8e-5 * float((w * (adv.abs() + 1)).sum())  # (log pi itself is off by 4e-5)
    _close(means[:4], wmeans, torch.where(sizes.isfinite(), 8e-5 * sizes, 0.0) + more)
    _close(loss, want, 8e-5 * float(sizes[0] + (kl_coef * sizes[1] if kl_coef else 0)) + more)
    wgrad = logits_grad(p, logp, ent, a, slope, torch.zeros_like(w), 0.9)
    hot = torch.zeros_like(p).scatter_(-1, a[..., None], 1.0)
    size = (w * (adv.double().abs() * 1.3 + kl_coef * ((ref.double() - lp).exp() + 1)))[..., None] * (p + hot)
    unit = 2.0 ** -22 if dtype == torch.float32 else UNIT[dtype]
    _close(grad, wgrad, 2e-4 * size + unit * wgrad.abs() + 1e-30)
    assert bool(grad.isfinite().all())


def test_a_policy_that_forbids_the_action():
    """log pi = -inf under a finite reference: the KL term is +inf, and nothing of it enters without a coefficient."""
    lp = torch.tensor([[-1.0, -math.inf, -2.0]])
    old, adv, ref = torch.tensor([[-1.1, -3.0, -2.0]]), torch.tensor([[1.0, 1.0, -1.0]]), torch.tensor([[-1.0, -1.0, -1.0]])
    loss, grad, means = policy.compute_policy_loss(*(t.cuda() for t in (lp, old, adv, ref)))
    assert float(means[1]) == math.inf and float(means[3]) == math.inf and bool(grad.isfinite().all()) and math.isfinite(float(loss))
    loss, grad, means = policy.compute_policy_loss(*(t.cuda() for t in (lp, old, adv, ref)), kl_coef=0.5)
    assert float(loss) == math.inf and float(grad[0, 1]) == -math.inf and bool(grad[0, ::2].isfinite().all())


@pytest.mark.parametrize("tau", [1e-38, 1e-9, 1e9, 1e38])
@pytest.mark.parametrize("A", [7, 300, 70001])
def test_extreme_temperatures(A, tau):
    """At the ends of what is allowed: all on the largest logit, or even over those that are allowed.  (x / tau in float64 loses no
    digit; entropies and log-probabilities are off by a few u of log A.)"""
    g = torch.Generator().manual_seed(A)
    x = torch.randn(3, 2, A, generator=g)
    x[..., 1::3] = -math.inf
    x[..., 0] = 6.0  # (the largest, by far more than tau where tau is small)
    for act in (0, 1, 2):
        a = torch.full((3, 2), act)
        lp, ent = policy.compute_action_log_probs(x.cuda(), a.cuda(), tau)
        want, went, _, _ = softmax_rows(x, a, tau)
        _close(lp, want.float(), 1e-6 * (1 + want.abs().nan_to_num(posinf=0)))
        _close(ent, went, 1e-5 * (1 + math.log(A)))
