"""compute_gated_delta_rule over more environments than one set of launches takes, with everything that is read at an environment's place: gates, episode
ends, states, and back the upstream gradients and what the forward pass has left.  Environments on both sides of a set's border are, bit by bit, what they are
by themselves."""
import pytest
import torch

import rl_triton.policy as policy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


# Sets hold 1 GiB: of records (11536 bytes a chunk of 64 steps and head) forward, of states and columns back (5120 bytes at up to 16 dims, 98304 at 128).
@pytest.mark.parametrize("shape, borders, dtype", [
    ((2110, 70, 50, 2, 2), (930, 2097), torch.float32),  # forward sets of 930, back of 2097
    ((700, 65, 8, 128, 128), (682,), torch.bfloat16),  # forward one set, back of 682
])
def test_environments_beside_a_border(shape, borders, dtype):
    E, T, H, dk, dv = shape
    g = torch.Generator(device="cuda").manual_seed(3)

    def n(*s):
        return torch.randn(s, generator=g, device="cuda")

    q, k = (torch.nn.functional.normalize(n(E, T, H, dk), dim=-1).to(dtype) for _ in range(2))
    v, up = n(E, T, H, dv).to(dtype), n(E, T, H, dv).to(dtype)
    gates, betas = -torch.rand(E, T, H, generator=g, device="cuda"), torch.rand(E, T, H, generator=g, device="cuda")
    dones = (torch.rand(E, T, generator=g, device="cuda") < 0.05).float()
    state, up_last = n(E, H, dk, dv), n(E, H, dk, dv)

    def run(lo, hi):
        x = [t[lo:hi].detach().requires_grad_(i != 5) for i, t in enumerate((q, k, v, gates, betas, dones, state))]
        out, last = policy.compute_gated_delta_rule(*x, 0.7)
        return (out.detach(), last.detach(), *torch.autograd.grad((out, last), [t for i, t in enumerate(x) if i != 5], (up[lo:hi], up_last[lo:hi])))

    whole = run(0, E)
    for lo in (0, *(b - 1 for b in borders), E - 2):
        for a, b in zip(whole, run(lo, lo + 2)):
            assert torch.equal(a[lo:lo + 2], b), lo
