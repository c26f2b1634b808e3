"""The operators together: the memory that a policy plays with is the one it is trained with, and the training works."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
import recall  # noqa: E402
import rl_triton.policy as policy  # noqa: E402

pytestmark = pytest.mark.gpu


def test_playing_and_learning_agree():
    """At the policy that played, step by step and as a window are the same float32 sums in another order: every ratio is 1, the
    divergence 0, and the loss the negative mean of the advantages, to well below 1e-4 (networks of unit scale, 40 steps)."""
    torch.manual_seed(1)
    g = torch.Generator(device="cuda").manual_seed(1)
    task = recall.Recall(33, 4, 9, torch.device("cuda"), g)
    net = recall.Policy(5, 4).cuda()
    state, done = torch.zeros(33, 2, 32, 32, device="cuda"), torch.zeros(33, device="cuda")
    for window in range(2):
        begin = torch.where(done[:, None, None, None] != 0, 0.0, state)
        played = []
        for _ in range(40):
            obs = task.observe()
            logits, value = net.act(obs, state, done)
            action = torch.multinomial(torch.softmax(logits, -1), 1, generator=g).squeeze(-1)
            log_prob, _ = policy.compute_action_log_probs(logits, action)
            _, done = task.step(action)
            played.append((obs, action, log_prob, done))
        obs, actions, old, dones = (torch.stack(x, 1) for x in zip(*played))
        logits, _ = net(obs, begin, dones)
        log_probs, _ = policy.compute_action_log_probs(logits, actions)
        assert float((log_probs - old).abs().max()) < 1e-4
        advantages = torch.randn(33, 40, generator=g, device="cuda")
        loss, grad, means = policy.compute_policy_loss_from_logits(logits, actions, old, advantages)
        assert abs(float(loss) + float(advantages.mean())) < 1e-4 and float(means[2]) == 0 and abs(float(means[3])) < 1e-6
        assert grad.shape == logits.shape


@pytest.mark.parametrize("dtype,from_log_probs", [(torch.float32, False), (torch.bfloat16, True)])
def test_it_learns(dtype, from_log_probs):
    """A policy that does not remember the symbol is right once in four."""
    right = recall.train(updates=60, dtype=dtype, from_log_probs=from_log_probs, say=lambda _: None)
    assert sum(right[:3]) / 3 < 0.4 and sum(right[-5:]) / 5 > 0.6
