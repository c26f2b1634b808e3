"""Which calls of compute_query_key_norms launch: all that have something to compute, whichever of queries and keys has no heads."""
import pytest
import torch

from rl_triton.policy import _native, head_norms

SETTINGS = (10000.0, 0, 1e-6, False)


@pytest.mark.parametrize("lead", [(5,), (5, 2)])
@pytest.mark.parametrize("heads", [(0, 3), (3, 0), (2, 1)])
def test_either_side_may_have_no_heads(lead, heads, monkeypatch):
    launched = []
    monkeypatch.setattr(_native, "query_key_norms", lambda *a: launched.append("forward"))
    monkeypatch.setattr(_native, "query_key_norms_backward", lambda *a: launched.append("backward"))
    q, k = (torch.ones(*lead, h, 8, requires_grad=True) for h in heads)
    w = torch.ones(8, requires_grad=True)
    outs = head_norms._QueryKeyNorms.apply(q, k, w, w, None, SETTINGS)
    assert launched == ["forward"]
    torch.autograd.grad(outs, (q, k, w), [torch.ones_like(x) for x in outs])
    assert launched == ["forward", "backward"]


@pytest.mark.parametrize("shape", [(0, 3, 8), (5, 0, 8), (0, 2, 3, 8), (5, 0, 3, 8), (5, 2, 0, 8)])
def test_nothing_to_compute(shape, monkeypatch):
    """No launch, and gradients of weights that are zero."""
    monkeypatch.setattr(_native, "query_key_norms", None)
    monkeypatch.setattr(_native, "query_key_norms_backward", None)
    q, k = (torch.ones(shape, requires_grad=True) for _ in range(2))
    w = torch.ones(8, requires_grad=True)
    outs = head_norms._QueryKeyNorms.apply(q, k, w, w, None, SETTINGS)
    grads = torch.autograd.grad(outs, (q, k, w), [torch.ones_like(x) for x in outs])
    assert grads[0].shape == q.shape and grads[1].shape == k.shape and not bool(grads[2].any())
