"""compute_policy_loss and compute_policy_loss_from_logits against the float64 definitions.

Error bounds (u = 2^-24).  A step's D = log pi - log pi_old is rounded once (u |D|); r = e^D, held or not, is off by
(|D| + 2) u, a KL term by 4 u of itself and (|d| + 2) u of r's size beyond the series; with |D| <= 4 every term and
slope is off by less than 2e-6 of the sizes that it is made of, and the weight by 2 u.  Sums of float32 terms in at most
64 steps per thread before they are added in float64: another 64 u = 4e-6 of the sum of sizes.  From logits, log pi itself
is off by 4e-5 (test_gpu_policy_log_probs.py), and r and the slope by 4e-5 of their sizes.
Ratios are kept 1e-3 and more from the corners."""
import math
import os

import pytest
import torch

import rl_triton.policy as policy
from _policy_reference import UNIT, logits_grad, policy_loss, softmax_rows

pytestmark = pytest.mark.gpu
LOW, HIGH, DUAL, KL = 0.2, 0.3, 2.5, 0.1


def _off(d):
    for c in (math.log(1 - LOW), math.log(1 + HIGH), math.log(DUAL)):
        d = torch.where((d - c).abs() < 2e-3, c + 4e-3 * torch.where(d < c, -1.0, 1.0), d)
    return d


def _make(E, T, seed, dtype=torch.float32, ref=True, mask="random", lp=None):
    g = torch.Generator().manual_seed(seed)
    if lp is None:
        lp = torch.log(torch.rand(E, T, generator=g).clamp_min(1e-3)).to(dtype)
    old = (lp.float() - _off(torch.randn(E, T, generator=g).clamp(-4, 4) * 0.4)).to(dtype)
    adv = torch.randn(E, T, generator=g).to(dtype)
    r = (lp.float() + torch.randn(E, T, generator=g) * 0.5).to(dtype) if ref else None
    m = None
    if mask is not None:
        m = (torch.rand(E, T, generator=g) < 0.6).to(dtype)
        if mask == "empty rows":
            m[::2] = 0
        if mask == "empty":
            m[:] = 0
    return lp, old, adv, r, m


def _dev(ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["steps", "rows"])
@pytest.mark.parametrize("mask", [None, "random", "empty rows", "empty"])
@pytest.mark.parametrize("E,T", [(1, 1), (1, 3), (3, 1), (5, 7), (17, 64), (33, 257), (2, 5000), (700, 3), (300, 1001)])
def test_loss_and_gradient(E, T, mask, reduction, dtype):
    for ref, dual in ((True, DUAL), (False, None)):
        lp, old, adv, r, m = _make(E, T, E * T, dtype, ref, mask)
        d = _dev((lp, old, adv, r, m))
        loss, grad, means = policy.compute_policy_loss(*d[:4], LOW, HIGH, KL, dual_clip=dual, mask=d[4], reduction=reduction)
        want, wgrad, wmeans, sizes, w = policy_loss(lp, old, adv, r, m, LOW, HIGH, dual, KL, reduction)
        assert loss.shape == () and means.shape == (4,) and grad.dtype == dtype and loss.dtype == torch.float32
        tol = 6e-6 * (sizes + 1e-30) + 2 ** -23 * wmeans.abs()
        assert bool(((means.cpu().double() - wmeans).abs() <= tol).all())
        assert abs(float(loss) - float(want)) <= float(tol[0] + KL * tol[1]) + 2 ** -23 * abs(float(want))
        slope = w * (adv.double().abs() * (lp.double() - old.double()).exp() + KL * (0 if r is None else
                     (r.double() - lp.double()).exp() + 1))
        unit = 0 if dtype == torch.float32 else UNIT[dtype]
        assert bool(((grad.cpu().double() - wgrad).abs() <= 3e-6 * slope + unit * wgrad.abs()).all())


def test_gradient_against_differences():
    lp, old, adv, r, m = _make(6, 40, 5)
    d = _dev((lp, old, adv, r, m))
    _, grad, _ = policy.compute_policy_loss(*d[:4], LOW, HIGH, KL, dual_clip=DUAL, mask=d[4], reduction="rows")
    v = torch.randn(lp.shape, generator=torch.Generator().manual_seed(6)).double()
    h = 1e-5  # (no corner within h |v|: ratios stay 2e-3 from them)
    f = [float(policy_loss(lp.double() + s * h * v, old, adv, r, m, LOW, HIGH, DUAL, KL, "rows")[0]) for s in (1, -1)]
    dot = float((grad.cpu().double() * v).sum())
    # h^2 times third derivatives below 5 each, |v|^3 below 40; float64 rounding 1e-15 / h; the gradient 3e-6 of its size
    assert abs((f[0] - f[1]) / (2 * h) - dot) < 1e-10 * 200 + 1e-9 + 1e-5 * float((grad.cpu().double() * v).abs().sum())


def test_masked_steps_may_hold_anything():
    lp, old, adv, r, m = _make(9, 50, 3, mask="empty rows")
    want = policy_loss(lp, old, adv, r, m, LOW, HIGH, DUAL, KL, "rows")
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min):
        ts = [torch.where(m != 0, t, bad) for t in (lp, old, adv, r)]
        loss, grad, _ = policy.compute_policy_loss(*_dev(ts), LOW, HIGH, KL, dual_clip=DUAL, mask=m.cuda(), reduction="rows")
        assert abs(float(loss) - float(want[0])) < 1e-5
        assert bool((grad.cpu()[m == 0] == 0).all()) and bool(grad.isfinite().all())


def test_kl_near_zero():
    """The KL term of nearly equal policies keeps its digits: for d = 1e-3 it is d^2 / 2, 5e-7."""
    lp = torch.full((1, 512), -1.0)
    r = lp + torch.linspace(-2e-3, 2e-3, 512)
    z = torch.zeros_like(lp)
    _, _, means = policy.compute_policy_loss(*_dev((lp, lp, z, r)), 0.2, 0.2, 1.0)
    e = (r.double() - lp.double())
    want = float((torch.expm1(e) - e).mean())
    assert abs(float(means[1]) - want) < 1e-5 * want


def test_strided_and_time_major_inputs():
    lp, old, adv, r, m = _make(12, 33, 8)
    want = policy.compute_policy_loss(*_dev((lp, old, adv, r)), LOW, HIGH, KL, mask=m.cuda())
    views = [t.cuda().t().contiguous().t() for t in (lp, old, adv, r, m)]
    got = policy.compute_policy_loss(*views[:4], LOW, HIGH, KL, mask=views[4])
    assert all(torch.allclose(a, b, rtol=1e-6, atol=1e-9) for a, b in zip(got, want))
    wide = torch.zeros(12, 70, device="cuda")
    wide[:, 1:34] = lp.cuda()
    got = policy.compute_policy_loss(wide[:, 1:34], *_dev((old, adv, r)), LOW, HIGH, KL, mask=m.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_steps():
    for shape in ((0, 4), (4, 0)):
        z = torch.zeros(shape, device="cuda")
        loss, grad, means = policy.compute_policy_loss(z, z, z, mask=z)
        assert float(loss) == 0 and grad.shape == shape and bool((means == 0).all())
        x = torch.zeros(*shape, 5, device="cuda")
        loss, grad, means = policy.compute_policy_loss_from_logits(x, torch.zeros(shape, dtype=torch.int64, device="cuda"), z, z)
        assert float(loss) == 0 and grad.shape == x.shape and bool((means == 0).all())


def test_runs_alike():
    """The same bits every time."""
    d = _dev(_make(300, 1001, 1))
    runs = [policy.compute_policy_loss(*d[:4], LOW, HIGH, KL, mask=d[4], reduction="rows") for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


# ---------------------------------------------------------------------------------------
# from logits
# ---------------------------------------------------------------------------------------
def _make_logits(E, T, A, seed, dtype, invalid=False, **kw):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(E, T, A, generator=g) * 2
    a = torch.randint(0, A, (E, T), generator=g)
    if invalid:
        x[torch.rand(E, T, A, generator=g) < 0.3] = -math.inf
        x.scatter_(-1, a[..., None], torch.randn(E, T, 1, generator=g))
    x = x.to(dtype)
    lp = softmax_rows(x, a, 0.9)[0]
    return x, a, _make(E, T, seed, torch.float32, lp=lp.float(), **kw)


def _logits_check(x, a, terms, xd, reduction, dual=DUAL, eta=0.02):
    _, old, adv, r, m = terms
    d = _dev((old, adv, r, m))
    loss, grad, means = policy.compute_policy_loss_from_logits(xd, a.cuda(), *d[:3], LOW, HIGH, KL, eta, 0.9, dual_clip=dual,
                                                               mask=d[3], reduction=reduction)
    lp, ent, p, logp = softmax_rows(x, a, 0.9)
    base, slope, wmeans, sizes, w = policy_loss(lp, old, adv, r, m, LOW, HIGH, dual, KL, reduction)
    went = float((w * ent).sum())
    tol = 8e-5 * (sizes + (w * (adv.abs() + 1)).sum())
    assert bool(((means[:4].cpu().double() - wmeans).abs() <= tol).all())
    assert abs(float(means[4]) - went) <= 1e-4 * (1 + went)
    assert abs(float(loss) - float(base) + eta * went) <= float(tol[0] + KL * tol[1]) + 1e-4 * eta * (1 + went)
    want = logits_grad(p, logp, ent, a, slope, -eta * w, 0.9)
    assert grad.dtype == x.dtype and grad.shape == x.shape and grad.is_contiguous()
    raw = w * (adv.double().abs() * (lp - old.double()).exp() + KL * (0 if r is None else (r.double() - lp).exp() + 1))
    hot = torch.zeros_like(p).scatter_(-1, a[..., None], 1.0)
    size = raw[..., None] * (p + hot) + eta * w[..., None] * p * torch.where(p > 0, logp.abs() + 1 + 2 * ent[..., None], 0.0)
    unit = 2.0 ** -22 if x.dtype == torch.float32 else UNIT[x.dtype]
    err = (grad.cpu().double() - want).abs()
    bound = 2e-4 * size + unit * want.abs() + 1e-30
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("A", [1, 2, 6, 18, 33, 64, 129, 1000, 1025, 5001, 20001, 40000, 70001, 140001])
def test_from_logits(A, dtype):
    E, T = (7, 45) if A <= 1025 else (2, 3)
    for i, (mask, ref, reduction) in enumerate(((None, False, "steps"), ("random", True, "rows"), ("empty rows", True, "steps"))):
        x, a, terms = _make_logits(E, T, A, A + i, dtype, invalid=i == 1, mask=mask, ref=ref)
        _logits_check(x, a, terms, x.cuda(), reduction)
    wide = torch.zeros(E, T, A + 3, dtype=dtype, device="cuda")
    wide[..., 1:A + 1] = x.cuda()
    _logits_check(x, a, terms, wide[..., 1:A + 1], "rows")
    _logits_check(x, a, terms, x.cuda().transpose(0, 1).contiguous().transpose(0, 1), "rows")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,A", [(1, 131072), (1, 16389), (3, 32771), (64, 33000), (65, 33000), (70, 140001), (13, 70003)])
def test_from_logits_few_long_rows(rows, A, dtype):
    """Rows shared by several workgroups, masked ones among them."""
    if rows > 20 and A > 100000 and dtype == torch.float32:
        rows = 5
    for mask in (None, "random"):
        x, a, terms = _make_logits(1, rows, A, A + rows, dtype, mask=mask, ref=True)
        _logits_check(x, a, terms, x.cuda(), "rows")


def test_from_logits_many_rows():
    """More rows than workgroups: every group of lanes takes several."""
    x, a, terms = _make_logits(600, 500, 6, 2, torch.float32, mask="random", ref=True)
    _logits_check(x, a, terms, x.cuda(), "rows")


def test_from_logits_masked_steps_may_hold_anything():
    x, a, terms = _make_logits(5, 20, 70, 9, torch.float32, mask="random", ref=True)
    _, old, adv, r, m = terms
    os.environ["RL_TRITON_CORRECTNESS_WARNINGS"] = "0"
    want = policy.compute_policy_loss_from_logits(x.cuda(), a.cuda(), *_dev((old, adv, r)), LOW, HIGH, KL, 0.01, mask=m.cuda())
    bad = [torch.where(m != 0, t, math.nan) for t in (old, adv, r)]
    xb = torch.where((m != 0)[..., None], x, math.nan)
    ab = torch.where(m != 0, a, 1 << 40)
    got = policy.compute_policy_loss_from_logits(xb.cuda(), ab.cuda(), *_dev(bad), LOW, HIGH, KL, 0.01, mask=m.cuda())
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    assert bool((got[1].cpu()[m == 0] == 0).all())


def test_from_logits_agrees_with_the_parts():
    """compute_action_log_probs, compute_policy_loss and their gradients chained give the same gradient."""
    x, a, terms = _make_logits(8, 30, 50, 4, torch.float32, mask="random", ref=True)
    _, old, adv, r, m = terms
    d = _dev((old, adv, r))
    loss, grad, _ = policy.compute_policy_loss_from_logits(x.cuda(), a.cuda(), *d, LOW, HIGH, KL, mask=m.cuda())
    xd = x.cuda().requires_grad_()
    lp, _ = policy.compute_action_log_probs(xd, a.cuda())
    loss2, g, _ = policy.compute_policy_loss(lp, *d, LOW, HIGH, KL, mask=m.cuda())
    lp.backward(g)
    assert abs(float(loss) - float(loss2)) < 1e-6 * (1 + abs(float(loss)))
    assert torch.allclose(xd.grad, grad, rtol=1e-4, atol=1e-7 * float(grad.abs().max()))


def test_graph():
    os.environ["RL_TRITON_CORRECTNESS_WARNINGS"] = "0"
    x, a, terms = _make_logits(40, 30, 18, 4, torch.float32, mask="random", ref=True)
    _, old, adv, r, m = _dev(terms)
    xd, ad = x.cuda(), a.cuda()

    def call():
        lp, _ = policy.compute_action_log_probs(xd, ad)
        return (*policy.compute_policy_loss(lp, old, adv, r, LOW, HIGH, KL, mask=m, reduction="rows"),
                *policy.compute_policy_loss_from_logits(xd, ad, old, adv, r, LOW, HIGH, KL, mask=m, reduction="rows"))

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in (11, 12, 13):
        x2, _, t2 = _make_logits(40, 30, 18, seed, torch.float32, mask="random", ref=True)
        xd.copy_(x2)
        m.copy_(t2[4])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, call()))
