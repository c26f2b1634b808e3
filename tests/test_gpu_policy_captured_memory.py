"""Scratch memory of captured calls belongs to the graph and goes with it."""
import gc

import pytest
import torch

import rl_triton.policy as policy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["0"], ids=["fast"])
def _path(request, monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", request.param)  # (the checks of values read the device: not in a capture)


def _inputs():
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return n(1, 2048, 2, 64).bfloat16(), n(1, 2048, 2, 64).bfloat16(), n(1, 2048, 2, 64).bfloat16(), n(8, 1, 131072), n(64, 100), n(64, 100)


def _calls(q, k, v, logits, lp, adv):
    """Segments forward (with and without a graph of torch's) and backward, shared rows, and the losses' sums."""
    decay = torch.full((2,), 0.99, device="cuda")
    acts = torch.zeros(8, 1, dtype=torch.int64, device="cuda")
    ones = torch.ones_like(lp)

    def call():
        plain = policy.compute_linear_attention(q, k, v, decay)
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out, _ = policy.compute_linear_attention(*leaves, decay)
        grads = torch.autograd.grad(out, leaves, v)
        flags = policy.compute_linear_attention.__wrapped__(q, k, v, decay)  # (the Python path's scratch memory)
        a, b = policy.compute_action_log_probs(logits, acts)
        return (*plain, *grads, *flags, a, b, *policy.compute_policy_loss(lp, lp, adv, mask=ones, reduction="rows"))
    return call


def test_it_goes_with_the_graph():
    xs = _inputs()
    call = _calls(*xs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    call()
    torch.cuda.synchronize()
    levels = []
    for _ in range(4):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        graph.replay()
        torch.cuda.synchronize()
        del graph, got
        gc.collect()
        levels.append(torch.cuda.memory_stats()["requested_bytes.all.current"])
    assert levels == [levels[0]] * 4, levels


def test_replays_agree_with_calls_between_them():
    """The graph's scratch memory is its own: eager calls, other allocations and replays on new values in turn."""
    xs = _inputs()
    call = _calls(*xs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (1, 2, 3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in xs:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        noise = [torch.full((1 << 22,), 3.0, device="cuda") for _ in range(4)]
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del noise
