"""A bfloat16 output of compute_gated_delta_rule is the float32 one rounded once.

The same numbers go through the rule as bfloat16 and as float32 arrays.  Computed to float32's accuracy both times, an output's n = dim + 64 terms
round at 2^-24 of their size s each, sqrt(n) 2^-24 s < 2^-20 s together.  Looked at are outputs above 2^-6 of the largest, s / 16 where they are
distributed as normal numbers are (the largest is some 4 s); over these s / |output| is 0.8 (log 16 + ..) on average, below 4.  So one lands on
the other side of the middle between two bfloat16 numbers, 2^-8 to 2^-7 of it apart, in at most 2 * 4 * 2^-20 / 2^-8 = 2^-9 of the cases, and
there it is the neighbour.  (Factors of two bfloat16 numbers each, 2^-16 off, do so in some 2^-7.)"""
import pytest
import torch

import rl_triton.policy as policy
from _delta_reference import inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


def _apart(got, whole):
    """The share of numbers that are not the rounded ones, none of them further off than a step."""
    large = whole.abs() > 2.0 ** -6 * whole.abs().amax()
    got, want = got[large], whole[large].bfloat16()
    other = got != want
    step = torch.maximum(got.float().abs(), want.float().abs()) * 2.0 ** -7
    assert bool(((got.float() - want.float()).abs() <= step).all())
    return float(other.float().mean())


@pytest.mark.parametrize("shape", [(8, 256, 4, 64, 64), (2, 333, 3, 40, 72), (1, 4096, 2, 128, 128), (4, 64, 8, 16, 128), (3, 200, 4, 100, 24)])
def test_outputs_of_sequences_are_rounded_once(shape):
    x = [None if t is None else t.cuda() for t in inputs(*shape, torch.bfloat16, 41)]
    out, last = policy.compute_gated_delta_rule(*x, 1.0)
    whole, whole_last = policy.compute_gated_delta_rule(*(t.float() for t in x[:3]), *x[3:], 1.0)
    assert out.dtype == torch.bfloat16 and whole.dtype == torch.float32
    assert _apart(out, whole) <= 2.0 ** -9
    assert bool(torch.allclose(last, whole_last, rtol=0, atol=2.0 ** -20 * float(whole_last.abs().max())))


@pytest.mark.parametrize("shape", [(8, 256, 4, 64, 64), (2, 333, 3, 40, 72), (1, 2200, 2, 128, 128)])
def test_gradients_are_rounded_once(shape):
    x = [None if t is None else t.cuda() for t in inputs(*shape, torch.bfloat16, 42)]
    up = torch.randn(shape[0], shape[1], shape[2], shape[4], generator=torch.Generator().manual_seed(1)).cuda().bfloat16()
    results = []
    for dtype in (torch.bfloat16, torch.float32):
        leaves = [t.detach().to(dtype).requires_grad_() for t in x[:3]]
        out, _ = policy.compute_gated_delta_rule(*leaves, *x[3:], 1.0)
        results.append(torch.autograd.grad(out, leaves, up.to(dtype)))
    for a, b in zip(*results):
        assert _apart(a, b) <= 2.0 ** -9
