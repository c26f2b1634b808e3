"""A policy with a linear-attention memory, trained with the clipped policy loss on a task it cannot do without the memory.

Every episode shows one of `cues` symbols at its first step and blanks after it; at its last step, which a flag announces, the
action named by the symbol earns 1.  Episodes last from 2 to `longest` steps, so windows of a rollout begin and end inside them.

    python examples/recall.py [--updates 150] [--dtype bfloat16] [--from-log-probs]

The operators as a learner uses them:
  acting    compute_linear_attention_step, with the state written in place; compute_action_log_probs
  targets   rl_triton.compute_gae
  learning  compute_linear_attention over the window, from the state that it began with; compute_policy_loss_from_logits
            and `logits.backward(grad)`, or, with --from-log-probs, compute_action_log_probs and compute_policy_loss
"""
import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "rl-triton_amd"))
import rl_triton  # noqa: E402
import rl_triton.policy as policy  # noqa: E402


class Recall:
    """The task, for all environments at once on the GPU."""

    def __init__(self, envs, cues, longest, device, generator):
        self.cues, self.longest, self.generator = cues, longest, generator
        self.left = torch.zeros(envs, dtype=torch.int64, device=device)  # steps after this one
        self.cue = torch.zeros(envs, dtype=torch.int64, device=device)
        self.fresh = torch.ones(envs, dtype=torch.bool, device=device)
        self._begin()

    def _draw(self, low, high):
        return torch.randint(low, high, self.cue.shape, generator=self.generator, device=self.cue.device)

    def _begin(self):
        self.left = torch.where(self.fresh, self._draw(1, self.longest), self.left)
        self.cue = torch.where(self.fresh, self._draw(0, self.cues), self.cue)

    def observe(self):
        """[envs, cues + 1]: the symbol at the first step, then blanks; the last entry announces the last step."""
        seen = nn.functional.one_hot(self.cue, self.cues) * self.fresh[:, None]
        return torch.cat([seen, (self.left == 0)[:, None]], -1).float()

    def step(self, action):
        """(reward, done), float32."""
        done = self.left == 0
        reward = (done & (action == self.cue)).float()
        self.left = self.left - 1
        self.fresh = done
        self._begin()
        return reward, done.float()


class Policy(nn.Module):
    def __init__(self, inputs, actions, heads=2, dim=32, width=64, dtype=torch.float32):
        super().__init__()
        self.heads, self.dim, self.dtype = heads, dim, dtype
        self.inner = nn.Linear(inputs, width)
        self.qkv = nn.Linear(width, 3 * heads * dim)
        self.outer = nn.Linear(width + heads * dim, width)
        self.logits = nn.Linear(width, actions)
        self.value = nn.Linear(width, 1)
        self.register_buffer("decay", torch.tensor([1.0, 0.95]).repeat(heads)[:heads].contiguous())

    def parts(self, obs):
        x = torch.tanh(self.inner(obs))
        q, k, v = self.qkv(x).to(self.dtype).unflatten(-1, (3 * self.heads, self.dim)).chunk(3, -2)  # (views of the joint product)
        return x, q, k, v

    def heads_of(self, x, memory):
        y = torch.tanh(self.outer(torch.cat([x, memory.float().flatten(-2)], -1)))
        return self.logits(y), self.value(y).squeeze(-1)

    @torch.no_grad()
    def act(self, obs, state, done):
        """One step of every environment; `state` goes on in place."""
        x, q, k, v = self.parts(obs)
        memory, _ = policy.compute_linear_attention_step(q, k, v, self.decay, state, done, out_state=state)
        return self.heads_of(x, memory)

    def forward(self, obs, state, dones):
        """A window [envs, steps, ...] from `state`, as it was played."""
        x, q, k, v = self.parts(obs)
        memory, _ = policy.compute_linear_attention(q, k, v, self.decay, dones, state)
        return self.heads_of(x, memory)


def train(updates=150, envs=256, steps=64, cues=4, longest=12, epochs=4, dtype=torch.float32, from_log_probs=False, seed=0, say=print):
    """Trains a policy; returns the share of episodes that ended with the right action, one number an update."""
    device = torch.device("cuda")
    torch.manual_seed(seed)
    generator = torch.Generator(device=device).manual_seed(seed)
    task = Recall(envs, cues, longest, device, generator)
    net = Policy(cues + 1, cues, dtype=dtype).to(device)
    adam = torch.optim.Adam(net.parameters(), lr=3e-3)
    state = torch.zeros(envs, net.heads, net.dim, net.dim, device=device)
    done = torch.zeros(envs, device=device)
    right = []
    for update in range(updates):
        begin = torch.where(done[:, None, None, None] != 0, 0.0, state)  # (the step takes the flag with it, a window the state alone)
        played = []
        for _ in range(steps):
            obs = task.observe()
            logits, value = net.act(obs, state, done)
            action = torch.multinomial(torch.softmax(logits, -1), 1, generator=generator).squeeze(-1)
            log_prob, _ = policy.compute_action_log_probs(logits, action)
            reward, done = task.step(action)
            played.append((obs, action, log_prob, value, reward, done))
        obs, actions, old, values, rewards, dones = (torch.stack(x, 1) for x in zip(*played))
        with torch.no_grad():
            last_value = net.act(task.observe(), state.clone(), done)[1]
        advantages = rl_triton.compute_gae(rewards, values, dones, gamma=0.95, lambda_=0.95, last_value=last_value)
        returns = advantages + values
        advantages = (advantages - advantages.mean()) / (advantages.std() + 1e-6)

        for _ in range(epochs):
            logits, value = net(obs, begin, dones)
            if from_log_probs:
                log_probs, entropies = policy.compute_action_log_probs(logits, actions)
                loss, grad, means = policy.compute_policy_loss(log_probs, old, advantages)
                outs, grads = (log_probs, entropies), (grad, torch.full_like(entropies, -0.01 / entropies.numel()))
            else:
                loss, grad, means = policy.compute_policy_loss_from_logits(logits, actions, old, advantages, entropy_coef=0.01)
                outs, grads = (logits,), (grad,)
            value_loss = 0.5 * (value - returns).square().mean()
            adam.zero_grad()
            torch.autograd.backward((*outs, value_loss), (*grads, None))
            adam.step()
        right.append(float(rewards.sum() / dones.sum().clamp(min=1)))
        if update % 10 == 0 or update == updates - 1:
            say(f"update {update:4d}  right {right[-1]:.3f}  loss {float(loss):+.4f}  clipped {float(means[2]):.3f}  moved {float(means[3]):.5f}")
    return right


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--updates", type=int, default=150)
    parser.add_argument("--dtype", choices=("float32", "bfloat16"), default="float32")
    parser.add_argument("--from-log-probs", action="store_true")
    args = parser.parse_args()
    train(args.updates, dtype=getattr(torch, args.dtype), from_log_probs=args.from_log_probs)
