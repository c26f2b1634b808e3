"""Offsets and counts past 32 bits in rl_triton.policy: the far ends of arrays against small calls on copies of them, which do the same
arithmetic, so the same bits; rows of logits in another order of their sums where there are fewer of them, so within twice
(actions + 16) u of 1 + |result|, and one more rounding of a bfloat16 gradient (losses against their definition)."""
import pytest
import torch

import rl_triton.policy as policy
from _policy_reference import U16, U32

pytestmark = pytest.mark.gpu

FAR = 1 << 31  # elements


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("actions", [18, 40000])
def test_logits(actions):
    """More than 2^31 logits: the last rows' log-probabilities, gradients and loss gradients."""
    rows = FAR // actions + 5
    x = torch.zeros(1, rows, actions, device="cuda", dtype=torch.bfloat16)
    x[0, -3:] = _randn(1, 3, actions).bfloat16()
    a = torch.zeros(1, rows, device="cuda", dtype=torch.int64)
    a[0, -3:] = actions - 1
    tail, ta = x[:, -300:].clone().requires_grad_(), a[:, -300:].clone()
    x.requires_grad_()
    lp, ent = policy.compute_action_log_probs(x, a)
    tlp, tent = policy.compute_action_log_probs(tail, ta)
    def same(got, want, u=U32):
        assert bool(((got - want).abs() <= 2 * (actions + 16) * U32 * (1 + want.abs()) + (2 * U16 * want.abs() if u == U16 else 0)).all())

    same(lp[:, -300:], tlp)
    same(ent[:, -300:], tent)
    up = torch.zeros_like(lp)
    up[0, -3:] = 1.0
    g, = torch.autograd.grad(lp, x, up)
    tg, = torch.autograd.grad(tlp, tail, up[:, -300:].contiguous())
    same(g[:, -300:], tg, U16)
    assert bool(tg[0, -3:].any())
    del g
    # one unmasked step, the last: the loss is its own
    mask = torch.zeros(1, rows, device="cuda")
    mask[0, -1] = 1.0
    old, adv = lp.detach() - 0.1, torch.full((1, rows), 2.0, device="cuda")
    loss, grad, _ = policy.compute_policy_loss_from_logits(x.detach(), a, old, adv, mask=mask)
    tloss, tgrad, _ = policy.compute_policy_loss_from_logits(tail.detach(), ta, old[:, -300:].contiguous(), adv[:, -300:].contiguous(),
                                                             mask=mask[:, -300:].contiguous())
    same(loss, tloss)
    same(grad[:, -300:], tgrad, U16)
    assert bool((tgrad != 0).any())
    assert not bool(grad[0, 0].any())


@pytest.mark.parametrize("reduction", ["steps", "rows"])
def test_more_steps_than_31_bits_count(reduction):
    E, T = 70001, 32768
    lp = torch.full((E, T), -1.0, device="cuda")
    adv, mask = torch.ones(E, T, device="cuda"), torch.ones(E, T, device="cuda")
    adv[-1, -1] = 3.0
    mask[0, :2] = 0.0
    loss, grad, means = policy.compute_policy_loss(lp, lp, adv, mask=mask, reduction=reduction)
    n = E * T - 2
    assert n > FAR
    # of 2.3e9 equal terms and one other: sums in float64, weights rounded to float32
    assert abs(float(loss) + 1.0 + (2.0 / n if reduction == "steps" else 2.0 / (E * T))) < 1e-6
    want = -1.0 / n if reduction == "steps" else -1.0 / E / T
    assert abs(float(grad[-1, 0]) / want - 1) < 1e-6 and abs(float(grad[-1, -1]) / (3 * want) - 1) < 1e-6 and not bool(grad[0, :2].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sequences(dtype):
    """Environments, and steps, more than 2^31 elements apart."""
    decay = torch.tensor([0.9, 0.99], device="cuda")
    for shape, strides in (((2, 150, 2, 64), (FAR + 192, 128, 64, 1)), ((1, 150, 2, 64), (0, FAR // 128 + 64, 64, 1))):
        span = sum((n - 1) * s for n, s in zip(shape, strides)) + 1
        buf = torch.empty(span, device="cuda", dtype=dtype)
        far = torch.as_strided(buf, shape, strides)
        assert span > FAR
        q, v = (_randn(s, *shape).to(dtype) for s in (2, 3))
        far.copy_(_randn(4, *shape).to(dtype))
        near = far.contiguous().clone()
        for args, small in (((far, q, v), (near, q, v)), ((q, far, v), (q, near, v)), ((q, v, far), (q, v, near)), ((far, far, far), (near, near, near))):
            got, want = policy.compute_linear_attention(*args, decay), policy.compute_linear_attention(*small, decay)
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        leaves, small = [t.detach().requires_grad_() for t in (q, far, v)], [t.detach().requires_grad_() for t in (q, near, v)]
        up = _randn(5, *shape).to(dtype)
        got = torch.autograd.grad(policy.compute_linear_attention(*leaves, decay)[0], leaves, up)
        want = torch.autograd.grad(policy.compute_linear_attention(*small, decay)[0], small, up)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        del buf, far, got, leaves


def test_step():
    """A state of more than 2^31 elements."""
    E, d = FAR // (128 * 128) + 3, 128
    q, k, v = (_randn(s, E, 1, d).bfloat16() for s in (6, 7, 8))
    state = torch.empty(E, 1, d, d, device="cuda")
    state[-5:] = _randn(9, 5, 1, d, d)
    decay = torch.tensor([0.5], device="cuda")
    out, new = policy.compute_linear_attention_step(q, k, v, decay, state)
    o, n = policy.compute_linear_attention_step(q[-5:], k[-5:], v[-5:], decay, state[-5:].clone())
    assert torch.equal(out[-5:], o) and torch.equal(new[-5:], n)
