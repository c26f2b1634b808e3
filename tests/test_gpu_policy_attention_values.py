"""Linear attention at values and sizes where one path of it could answer otherwise than another: infinities at head dims that fill
no whole tile."""
import math

import pytest
import torch

import rl_triton.policy as policy
from _policy_reference import attention, attention_grads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", [(24, 24), (40, 72), (64, 64), (100, 33), (128, 128), (1, 1)])
def test_infinities_stay_infinities(dk, dv, dtype):
    """Where the recurrence gives inf the call does, and NaN where it gives NaN: dims that do not exist have no part in it.
    (Queries and values have no zeros, so that inf times one of them is inf.)"""
    E, T, H = 2, 90, 2
    g = torch.Generator().manual_seed(dk)
    n = lambda *s: (torch.rand(s, generator=g) + 0.5).to(dtype)  # noqa: E731
    q, k, v, go = n(E, T, H, dk), n(E, T, H, dk), n(E, T, H, dv), n(E, T, H, dv)
    decay = torch.tensor([0.9, 1.0])
    dones = torch.zeros(E, T)
    dones[:, 80] = 1
    k[0, 70, 0, 0] = math.inf
    v[0, 75, 1, dv - 1] = -math.inf
    k[1, 66, 0, dk - 1], v[1, 67, 0, 0] = math.inf, math.nan
    q[1, 72, 1, 0] = math.inf
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, last = policy.compute_linear_attention(*leaves, decay.cuda(), dones.cuda(), None, 0.5)
    got = (out, last, *torch.autograd.grad(out, leaves, go.cuda()))
    want = (*attention(q, k, v, decay, dones, None, 0.5), *attention_grads(q, k, v, decay, dones, None, 0.5, go, None)[:3])
    for i, (x, w) in enumerate(zip(got, want)):
        x = x.detach().cpu().double()
        assert torch.equal(x.isnan(), w.isnan()), i
        assert torch.equal(x == math.inf, w == math.inf) and torch.equal(x == -math.inf, w == -math.inf), i
