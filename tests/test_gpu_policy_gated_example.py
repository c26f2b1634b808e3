"""The example's policy with a gated memory: it runs, and its gradients are those of the same network in float64, played step by step."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
import recall  # noqa: E402
import rl_triton.policy as policy  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_it_runs(dtype):
    right = recall.train(updates=2, envs=32, steps=40, dtype=dtype, say=lambda _: None, memory="gated")
    assert len(right) == 2 and all(0.0 <= r <= 1.0 for r in right)


def test_gradients():
    """Against the network in float64 with the memory written out: 64-bit sums against float32's, whose errors are some sqrt(40) 2^-24 of the
    gradients' sizes; 1e-4 leaves a factor of more than a hundred for what cancels."""
    torch.manual_seed(1)
    net = recall.GatedPolicy(5, 4).cuda()
    E, T, H, d = 9, 40, net.heads, net.dim
    obs = torch.randn(E, T, 5, device="cuda")
    dones = (torch.rand(E, T, device="cuda") < 0.1).float()
    places = (recall.rl_triton.compute_episodic_prefix_sum(torch.ones(E, T, device="cuda"), dones) - 1).long()
    state = torch.randn(E, H, d, d, device="cuda") * 0.3
    up = torch.randn(E, T, 4, device="cuda")
    logits, _ = net(obs, state, dones, places)
    names = [n for n, p in net.named_parameters() if not n.startswith("value")]
    got = torch.autograd.grad(logits, [p for n, p in net.named_parameters() if n in names], up)

    wide = recall.GatedPolicy(5, 4, dtype=torch.float64).cuda().double()
    wide.load_state_dict(net.state_dict())
    x, q, k, v = recall.Policy.parts(wide, obs.double())
    angle = places.double()[..., None, None] * 10000.0 ** (-2 * torch.arange(d // 2, dtype=torch.float64, device="cuda") / d)
    heads = []
    for y, w in ((q, wide.q_norm), (k, wide.k_norm)):
        y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        a, b = y.chunk(2, -1)
        heads.append(torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1))
    q, k = heads
    forget, write = wide.gates(x).chunk(2, -1)
    decay, beta = torch.exp(-0.1 * torch.nn.functional.softplus(forget)), torch.sigmoid(write)
    S, outs = state.double(), []
    for t in range(T):
        S = S * decay[:, t, :, None, None] * ((1 - dones[:, t - 1].double()) if t else torch.ones(E, device="cuda", dtype=torch.float64))[:, None, None, None]
        u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, :, None] * S).sum(-2))
        S = S + k[:, t, :, :, None] * u[..., None, :]
        outs.append((q[:, t, :, :, None] * S).sum(-2))
    y = torch.tanh(wide.outer(torch.cat([x, torch.stack(outs, 1).flatten(-2)], -1)))
    want = torch.autograd.grad(wide.logits(y), [p for n, p in wide.named_parameters() if n in names], up.double())
    for n, a, b in zip(names, got, want):
        assert float((a.double() - b).norm()) <= 1e-4 * float(b.norm()), n


def test_playing_and_learning_agree():
    """At the policy that played, step by step and as a window are the same float32 sums in another order (40 steps: below 1e-4)."""
    torch.manual_seed(2)
    net = recall.GatedPolicy(5, 4).cuda()
    E, T = 33, 40
    obs, u = torch.randn(E, T, 5, device="cuda"), torch.rand(E, T, device="cuda")
    dones = (torch.rand(E, T, device="cuda") < 0.1).float()
    places = (recall.rl_triton.compute_episodic_prefix_sum(torch.ones(E, T, device="cuda"), dones) - 1).long()
    state = torch.zeros(E, net.heads, net.dim, net.dim, device="cuda")
    actions, log_probs = [], []
    for t in range(T):
        logits, _ = net.act(obs[:, t], state, dones[:, t - 1] if t else torch.zeros(E, device="cuda"), places[:, t].contiguous())
        a, lp = policy.compute_sampled_actions(logits, u[:, t].contiguous())
        actions.append(a), log_probs.append(lp)
    logits, _ = net(obs, torch.zeros_like(state), dones, places)
    again, _ = policy.compute_action_log_probs(logits, torch.stack(actions, 1))
    assert float((again.detach() - torch.stack(log_probs, 1)).abs().max()) < 1e-4
