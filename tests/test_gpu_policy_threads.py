"""Calls from several Python threads while backward passes run on torch's: each has scratch memory of its own stream, and answers as
it does alone."""
import threading

import pytest
import torch

import rl_triton.policy as policy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("checked", ["0", "1"], ids=["fast", "checked"])
def test_losses_beside_backward_passes_over_segments(checked, monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", checked)
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v, go = (n(1, 700, 2, 32) for _ in range(4))
    decay = torch.tensor([0.99, 0.9], device="cuda")
    lp, old, adv = n(20, 150) - 3, n(20, 150) * 0.1 - 3, n(20, 150)
    mask = (n(20, 150) > 0).float()
    logits, acts = n(3, 1, 65536), torch.tensor([[5], [60000], [0]], device="cuda")

    def backward():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out, _ = policy.compute_linear_attention(*leaves, decay)
        return torch.autograd.grad(out, leaves, go)

    def losses():
        return (*policy.compute_policy_loss(lp, old, adv, mask=mask, reduction="rows"), *policy.compute_action_log_probs(logits, acts),
                *policy.compute_linear_attention(q, k, v, decay))

    want = {backward: backward(), losses: losses()}
    torch.cuda.synchronize()
    # streams are made beforehand, and each thread goes from one to the next: the scratch memory of every one is new to the process
    streams = [[torch.cuda.Stream() for _ in range(8)] for _ in range(4)]
    errors = []

    def work(fn, mine):
        try:
            for stream in mine:
                with torch.cuda.stream(stream):
                    got = fn()
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[fn])):
                    errors.append(f"{fn.__name__} differs")
        except Exception as e:  # (an exception of a thread would pass unseen)
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(fn, mine), daemon=True) for fn, mine in zip((backward, losses, backward, losses), streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
