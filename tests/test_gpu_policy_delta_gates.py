"""Gradients of compute_gated_delta_rule's gates, head by head: those of a head that forgets fast are small, and are held to what they are made of.

With S the state that a gate has acted on and R its gradient, a gate's gradient is the sum of the products of their numbers, so float32's rounding of the chain
(tests/_delta_reference.py: 8 sqrt(T + dim + 64) 2^-24) counts in |S| |R|, however much larger other heads' gradients are, or the head's own of queries and keys.
A product of gates is formed from their sum, rounded at 2^-24 of itself: exp turns that into as much times the sum, 100 2^-24 for the smallest that
counts, and it is in S and in R: 200 2^-24 more."""
import math

import pytest
import torch

import rl_triton.policy as policy
from _delta_reference import U32, relative, rule

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


def _sizes(q, k, v, g, beta, dones, state, scale, up):
    """|S| |R| of every step and head, by the recurrence in float64."""
    q, k, v, beta, up = (x.double() for x in (q, k, v, beta, up))
    E, T, H, dk = q.shape
    a = torch.where(g < -104, 0.0, g.double().exp())
    a[:, 1:] = torch.where(dones[:, :-1, None] != 0, 0.0, a[:, 1:])
    S, kept, size = state.double(), [], torch.zeros(E, T, H, dtype=torch.float64)
    for t in range(T):
        B = S * a[:, t, :, None, None]
        kept.append(B)
        e = v[:, t] - (k[:, t, :, :, None] * B).sum(-2)
        S = B + k[:, t, :, :, None] * (beta[:, t, :, None] * e)[..., None, :]
    R = torch.zeros_like(S)
    for t in range(T - 1, -1, -1):
        R = R + scale * q[:, t, :, :, None] * up[:, t][..., None, :]
        du = (k[:, t, :, :, None] * R).sum(-2)
        R = R - k[:, t, :, :, None] * (beta[:, t, :, None] * du)[..., None, :]
        size[:, t] = kept[t].flatten(-2).norm(dim=-1) * R.flatten(-2).norm(dim=-1)
        R = R * a[:, t, :, None, None]
    return size


RATES = (0.0, 0.01, 0.3, 1.0, 3.0, 10.0, 20.0, 50.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 200, 64, 64), (1, 333, 40, 72), (2, 65, 128, 128), (1, 130, 100, 20), (3, 64, 16, 16), (4, 7, 24, 40)])
@pytest.mark.parametrize("ends", [0.0, 0.04])
def test_each_head_by_itself(shape, dtype, ends):
    E, T, dk, dv = shape
    H = len(RATES)
    g = torch.Generator().manual_seed(T + dk)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k = ((0.99 * torch.nn.functional.normalize(n(E, T, H, dk), dim=-1)).to(dtype) for _ in range(2))
    v, up = n(E, T, H, dv).to(dtype), n(E, T, H, dv).to(dtype)
    gates = -torch.tensor(RATES) * (0.5 + torch.rand(E, T, H, generator=g))
    betas, state = torch.rand(E, T, H, generator=g), n(E, H, dk, dv)
    dones = (torch.rand(E, T, generator=g) < ends).float()
    x = (q, k, v, gates, betas, dones, state)
    want = rule(*x, 0.7, up)[2][3]
    size = _sizes(*x, 0.7, up)
    d = [t.cuda() for t in x]
    d[3].requires_grad_()
    out, _ = policy.compute_gated_delta_rule(*d, 0.7)
    got, = torch.autograd.grad(out, d[3], up.cuda())
    err = (got.cpu().double() - want).abs()
    tol = relative(T, dk) + 200 * U32
    for h, rate in enumerate(RATES):
        assert float(err[..., h].norm()) <= tol * float(size[..., h].norm()) + 1e-37, (rate, float(err[..., h].norm() / want[..., h].norm()))
        assert bool((err[..., h] <= 8 * tol * size[..., h].amax(1, keepdim=True) + 1e-37).all()), rate


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_strong_gate_among_weak_ones(dtype):
    """A gate of -30 in the middle of steps that forget next to nothing: its gradient is small by itself, that of the others as ever."""
    E, T, H, d = 2, 192, 2, 64
    g = torch.Generator().manual_seed(9)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k = ((0.99 * torch.nn.functional.normalize(n(E, T, H, d), dim=-1)).to(dtype) for _ in range(2))
    v, up = n(E, T, H, d).to(dtype), n(E, T, H, d).to(dtype)
    gates = torch.full((E, T, H), -0.01)
    strong = (5, 63, 64, 100, 127, 191)
    gates[:, strong] = -30.0
    betas, state, dones = torch.rand(E, T, H, generator=g), n(E, H, d, d), torch.zeros(E, T)
    x = (q, k, v, gates, betas, dones, state)
    want, size = rule(*x, 0.7, up)[2][3], _sizes(*x, 0.7, up)
    c = [t.cuda() for t in x]
    c[3].requires_grad_()
    got, = torch.autograd.grad(policy.compute_gated_delta_rule(*c, 0.7)[0], c[3], up.cuda())
    err = (got.cpu().double() - want).abs()
    # (element by element: 8 times what an array's norm is held to, as in tests/_delta_reference.py)
    assert bool((err <= 8 * (relative(T, d) + 200 * U32) * size + 1e-37).all()), float((err / size).max())
    assert float(want[:, strong].abs().max()) < 1e-9 < 1e-3 < float(want.abs().max())
