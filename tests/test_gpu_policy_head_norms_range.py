"""compute_query_key_norms of rows whose squares leave float32's range: a row of 1e25 is normed as one of 1 is.

Bounds as in test_gpu_policy_head_norms.py: (n / 16 + 16) 2^-24 of the larger of a pair, times 2 back and sqrt(n) for the mean that is taken off, and the storage type's
rounding.  A root below 2^-126 has fewer bits, of rows above 2^126: at 3e38 some 2^-21 of itself, which 16 * 2^-24 does not cover: 2^-20 is added for these.  Results below 2^-126
are multiples of 2^-149 in float32, and 2^-133 in bfloat16."""
import math

import pytest
import torch

import rl_triton.policy as policy
from test_gpu_policy_head_norms import U16, U32, definition

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


# (largest element, eps): rows of the like are normed to length sqrt(dim)
SIZES = [(1e14, 1e-6), (1e16, 1e-6), (2e19, 1e-6), (1e25, 0.5), (3e38, 1e-6), (1e-14, 0.0), (1e-16, 0.0), (1e-21, 0.0), (1e-30, 0.0), (1e-25, 1e-6), (1e-16, 1e-38)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [3, 40, 72, 128, 200])
@pytest.mark.parametrize("size, eps", SIZES)
def test_rows_of_any_size(size, eps, dim, dtype):
    g = torch.Generator(device="cuda").manual_seed(dim)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    # every other row is an ordinary one
    q = torch.rand(4, 6, 3, dim, generator=g, device="cuda") * 2 - 1
    q[..., 0] = 1.0
    q[:, ::2] *= size
    q = q.to(dtype).requires_grad_()
    k = n(4, 6, 2, dim).to(dtype).requires_grad_()
    w = (1 + 0.2 * n(dim)).requires_grad_()
    pos = torch.randint(0, 1000, (4, 6), generator=g, device="cuda")
    up = n(*q.shape).to(dtype)
    rotary = dim // 2 * 2
    out, _ = policy.compute_query_key_norms(q, k, w, w, pos, rotary_dim=rotary, eps=eps)
    dq, dw = torch.autograd.grad(out, (q, w), up)
    want, grad, wdw, sizes, largest = definition(q.detach(), w.detach(), pos, rotary=rotary, eps=eps, up=up)
    far = 2.0 ** -20 if size > 2.0 ** 126 else 0.0
    u = U16 if dtype == torch.bfloat16 else U32
    least = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149
    tol = (dim / 16 + 16) * U32 + far
    pair = (want / w.detach().double()).abs().amax(-1, keepdim=True) * 2
    assert bool(((out.detach().double() - want).abs() <= tol * pair + u * want.abs() + 2 * least).all())
    grad = grad.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    assert bool(((dq.double() - grad).abs() <= 2 * tol * math.sqrt(dim) * largest + u * grad.abs() + 2 * least).all())
    rows = q.numel() // dim
    assert bool(((dw.double() - wdw).abs() <= ((dim / 8 + 32 + math.sqrt(rows)) * U32 + 2 * far) * sizes.clamp_min(float(sizes.max()) / 4)).all())


def test_rows_of_zeros_and_rows_that_are_not_finite():
    q = torch.zeros(2, 3, 2, 16, device="cuda")
    q[0, 1, 0, 3], q[0, 2, 1, 5], q[1, 0, 0] = math.inf, math.nan, 1e30
    k = torch.randn(2, 3, 1, 16, device="cuda")
    out, keys = policy.compute_query_key_norms(q, k)
    want = definition(q, None, None)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and bool((out.nan_to_num() - want.nan_to_num()).abs().max() <= 32 * U32)
    assert bool(torch.isfinite(keys).all())
    assert bool(torch.isnan(policy.compute_query_key_norms(q[1:, 1:], k[1:, 1:], eps=0.0)[0]).all())  # 0 / 0
