"""compute_gated_delta_rule from states that are not finite, or leave float32's range, over sequences that are cut into segments: what such a state
does ends with its episode, as in a sequence of one piece.

Sequences of 2500 steps of two heads have segments of 512 steps.  Results behind the cut are held to the float64 recurrence from a finite state (tests/_delta_reference.py),
on which they depend as little."""
import math

import pytest
import torch

import rl_triton.policy as policy
from _delta_reference import held, held_rounded, inputs, relative, rule

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


DTYPES = [torch.float32, torch.bfloat16]
E, T, H, DK, DV = 1, 2500, 2, 40, 64
LEAVES = (0, 1, 2, 3, 4, 6)  # q, k, v, log_decays, betas, state


def _inputs(dtype, cut, seed):
    """`cut`: the first step of the second episode, or 0: nothing of the state stays at the first step."""
    x = list(inputs(E, T, H, DK, DV, dtype, seed, None))
    x[3] = x[3].clamp_min(-2.0)
    x[5] = torch.zeros(E, T)
    if cut:
        x[5][:, cut - 1] = 1.0
    else:
        x[3][:, 0] = -math.inf
    g = torch.Generator().manual_seed(seed)
    return x, torch.randn(E, T, H, DV, generator=g).to(dtype), torch.randn(E, H, DK, DV, generator=g)


def _run(x, ups):
    d = [t.cuda() for t in x]
    for i in LEAVES:
        d[i].requires_grad_()
    out, last = policy.compute_gated_delta_rule(*d, 0.7)
    with torch.no_grad():
        alone = policy.compute_gated_delta_rule(*d, 0.7)
    assert torch.equal(alone[0].nan_to_num(), out.nan_to_num()) and torch.equal(alone[1].nan_to_num(), last.nan_to_num())
    return out.detach(), last.detach(), torch.autograd.grad((out, last), [d[i] for i in LEAVES], [u.cuda() for u in ups])


def _hold_from(cut, got, want, x, dtype):
    """Outputs, the last state and gradients of what comes at `cut` and later."""
    (out, last, grads), (wout, wlast, wgrads) = got, want
    hold = held if dtype == torch.float32 else held_rounded
    hold(out[:, cut:], wout[:, cut:], relative(T, DK), "out")
    held(last, wlast, relative(T, DK), "state")
    size = float((x[0].double() * wgrads[0]).norm() + (x[1].double() * wgrads[1]).norm())
    for i, (a, b) in enumerate(zip(grads[:5], wgrads[:5])):
        if i < 3:
            hold(a[:, cut:], b[:, cut:], relative(T, DK), i)
        else:
            held(a[:, cut:], b[:, cut:], relative(T, DK), i, size if i == 3 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cut", [0, 1, 300, 512, 700, 2100])
def test_a_state_that_is_not_finite(cut, value, dtype):
    """One number of one head's state: what comes behind the cut does not depend on it, nor does the other head, nor (before the cut) another column."""
    x, *ups = _inputs(dtype, cut, 31)
    clean = _run(x, ups)
    want = rule(*x, 0.7, *ups)
    x[6] = x[6].clone()
    x[6][0, 0, 3, 5] = value
    got = _run(x, ups)
    _hold_from(cut, got, want, x, dtype)
    assert torch.equal(got[0][:, :, 1], clean[0][:, :, 1]) and torch.equal(got[1][:, 1], clean[1][:, 1])
    for a, b in zip(got[2][:5], clean[2][:5]):
        assert torch.equal(a[:, :, 1], b[:, :, 1])
    assert torch.equal(got[2][5][:, 1], clean[2][5][:, 1])
    hold = held if dtype == torch.float32 else held_rounded
    others = [c for c in range(DV) if c != 5]
    hold(got[0][:, :cut][..., others], want[0][:, :cut][..., others], relative(T, DK), "other columns")
    if cut == 0:
        assert not bool(got[2][5].any())  # nothing depends on the state
    else:
        assert not bool(torch.isfinite(got[0][0, 0, 0, 5]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cut", [300, 700, 1100])
def test_a_state_that_leaves_float32_on_its_way(cut, dtype):
    """A state of 3e38, of which one step turns a row to some -6 times that: finite when it comes, out of float32's range when the segment ends (a segment's own
    share of it is finite).  Nothing else is written and nothing is forgotten until the episode ends."""
    x, *ups = _inputs(dtype, cut, 32)
    x[3][:, :cut] = 0.0
    x[4][:, :cut] = 0.0
    x[4][:, 10] = 2.0
    x[1][:, 10] = torch.cat([torch.tensor([0.8]), torch.full((DK - 1,), 0.6 / math.sqrt(DK - 1))]).to(dtype)
    want = rule(*x, 0.7, *ups)  # (behind the cut)
    x[6] = torch.full_like(x[6], 3e38)
    got = _run(x, ups)
    assert not bool(torch.isfinite(got[0][:, 10:cut]).all())
    _hold_from(cut, got, want, x, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_state_that_leaves_float32_without_an_end(dtype):
    """No episode ends: it stays in what it has reached, and steps of the other head are as before."""
    x, *ups = _inputs(dtype, 2000, 33)
    x[5].zero_()
    clean = _run(x, ups)
    x[6] = x[6].clone()
    x[6][0, 1] = math.inf
    out, last, _ = _run(x, ups)
    assert not bool(torch.isfinite(last[:, 1]).any())
    assert torch.equal(out[:, :, 0], clean[0][:, :, 0]) and torch.equal(last[:, 0], clean[1][:, 0])


def test_a_replay_does_not_remember_the_last_state():
    """Captured once, replayed with a state that is not finite and with finite ones before and after: as the eager calls."""
    x, *_ = _inputs(torch.bfloat16, 700, 34)
    static = [t.cuda() for t in x]
    fine = static[6].clone()
    bad = fine.clone()
    bad[0, 0, 3, 5], bad[0, 1, 0, 0] = math.nan, math.inf
    policy.compute_gated_delta_rule(*static, 0.7)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, last = policy.compute_gated_delta_rule(*static, 0.7)
    for state in (fine, bad, fine, bad, bad, fine):
        static[6].copy_(state)
        graph.replay()
        want = policy.compute_gated_delta_rule(*static, 0.7)
        torch.cuda.synchronize()
        for a, b in zip((out, last), want):
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())
