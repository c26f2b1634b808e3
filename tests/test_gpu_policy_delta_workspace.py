"""A training call's forward pass asks for what it leaves, its results and, cut into segments, for theirs: not for its records once more."""
import pytest
import torch

import rl_triton.policy as policy
from rl_triton.policy import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("warnings", ["0", "1"])  # (the C++ path, the Python one)
@pytest.mark.parametrize("shape", [(16, 256, 8, 64, 64), (1, 4096, 2, 64, 64)])
def test_memory_of_a_forward_pass(shape, warnings, monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", warnings)
    E, T, H, dk, dv = shape
    q, k = (torch.nn.functional.normalize(torch.randn(E, T, H, dk, device="cuda"), dim=-1) for _ in range(2))
    v, gates, betas = torch.randn(E, T, H, dv, device="cuda"), -torch.rand(E, T, H, device="cuda"), torch.rand(E, T, H, device="cuda")
    leaf = q.requires_grad_()
    policy.compute_gated_delta_rule(leaf, k, v, gates, betas)
    torch.cuda.synchronize()
    lib = _native.load()
    saved, segments = lib.rlk_delta_rule_saved_bytes(*shape), lib.rlk_delta_rule_workspace_bytes(*shape, 2)
    assert (segments > 0) == (E == 1)
    results = 4 * (v.numel() + E * H * dk * dv)
    asked = lambda which: torch.cuda.memory_stats()["requested_bytes.all." + which]  # noqa: E731  (of the allocator, whose blocks may be larger)
    before = asked("current")
    torch.cuda.reset_peak_memory_stats()
    out, last = policy.compute_gated_delta_rule(leaf, k, v, gates, betas)
    checks = 2 * betas.numel() if warnings == "1" else 0  # (of values: bytes of comparisons)
    assert asked("peak") - before <= max(saved + segments + results, checks) + (1 << 14)
    up = torch.ones_like(out)
    got, = torch.autograd.grad(out, leaf, up)
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    want, = torch.autograd.grad(policy.compute_gated_delta_rule(leaf, k, v, gates, betas)[0], leaf, up)
    assert torch.equal(got, want)
