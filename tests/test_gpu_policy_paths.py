"""The two ways into rl_triton.policy: the C++ fast path and the Python one, which reaches the same entry points through
ctypes.  Well-formed calls take the fast path, and both give the same bits."""
import pytest
import torch

import rl_triton.policy as policy
from rl_triton import _native

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


def _calls(dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, a = n(6, 50, 18).to(dtype), torch.randint(0, 18, (6, 50), generator=g, device="cuda")
    lp, old, adv, ref = -n(6, 50).abs(), -n(6, 50).abs(), n(6, 50), -n(6, 50).abs()
    mask = (n(6, 50) > 0).float()
    low = [t.to(dtype) for t in (lp, old, adv, ref, mask)]
    q, k, v = n(3, 80, 2, 24).to(dtype), n(3, 80, 2, 24).to(dtype), n(3, 80, 2, 40).to(dtype)
    decay, dones, state = torch.tensor([0.9, 0.99], device="cuda"), (n(3, 80) > 1).float(), n(3, 2, 24, 40)
    return [
        (policy.compute_action_log_probs, (x, a), {}),
        (policy.compute_action_log_probs, (x, a, 2), {}),
        (policy.compute_policy_loss, tuple(low[:3]), {}),
        (policy.compute_policy_loss, tuple(low[:4]), dict(kl_coef=0.1, dual_clip=3.0, mask=low[4], reduction="rows")),
        (policy.compute_policy_loss_from_logits, (x, a, old, adv), {}),
        (policy.compute_policy_loss_from_logits, (x, a, old, adv, ref, 0.1, 0.3, 0.1, 0.01, 0.7), dict(mask=mask, reduction="rows")),
        (policy.compute_linear_attention, (q, k, v, decay), {}),
        (policy.compute_linear_attention, (q, k, v, decay, dones, state, 0.5), {}),
        (policy.compute_linear_attention_step, (q[:, 0], k[:, 0], v[:, 0], decay, state), {}),
        (policy.compute_linear_attention_step, (q[:, 0], k[:, 0], v[:, 0], decay, state, dones[:, 3], 0.5), {}),
    ]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_both_paths_give_the_same_bits(dtype):
    for fn, args, kw in _calls(dtype):
        before = _native.fast.launched()
        fast = fn(*args, **kw)
        assert _native.fast.launched() == before + 1, fn.__name__
        slow = fn.__wrapped__(*args, **kw)
        assert _native.fast.launched() == before + 1, fn.__name__
        assert len(fast) == len(slow)
        for f, s in zip(fast, slow):
            assert f.dtype == s.dtype and f.shape == s.shape and torch.equal(f, s), fn.__name__


def test_calls_the_fast_path_leaves(monkeypatch):
    """Gradients wanted, copies needed, malformed, correctness warnings on: the Python path serves or refuses them."""
    x, a = torch.randn(4, 5, 7, device="cuda"), torch.zeros(4, 5, dtype=torch.int64, device="cuda")
    z = torch.zeros(4, 5, device="cuda")
    before = _native.fast.launched()
    lp, _ = policy.compute_action_log_probs(x.clone().requires_grad_(), a)
    assert lp.requires_grad
    policy.compute_action_log_probs(x.transpose(1, 2).contiguous().transpose(1, 2), a)
    policy.compute_policy_loss(z.t().contiguous().t(), z, z)
    with pytest.raises(AssertionError, match="temperature"):
        policy.compute_action_log_probs(x, a, 0.0)
    with pytest.raises(AssertionError, match="reduction"):
        policy.compute_policy_loss(z, z, z, reduction="none")
    with pytest.raises(AssertionError, match="dual_clip"):
        policy.compute_policy_loss(z, z, z, dual_clip=0.9)
    with pytest.raises(AssertionError, match="advantages shape"):
        policy.compute_policy_loss(z, z, z[:, :4])
    q = torch.zeros(2, 3, 1, 8, device="cuda")
    decay = torch.ones(1, device="cuda")
    with pytest.raises(AssertionError, match="scale"):
        policy.compute_linear_attention(q, q, q, decay, None, None, 0.0)
    with pytest.raises(AssertionError, match="constant"):
        policy.compute_linear_attention(q, q, q, decay.clone().requires_grad_())
    with pytest.raises(TypeError):
        policy.compute_linear_attention(q, q, q)
    state = torch.zeros(2, 1, 8, 8, device="cuda")
    with pytest.raises(AssertionError, match="overlaps"):
        both = torch.zeros(3, 1, 8, 8, device="cuda")
        policy.compute_linear_attention_step(q[:, 0], q[:, 0], q[:, 0], decay, both[:2], out_state=both[1:])
    policy.compute_linear_attention_step(q[:, 0], q[:, 0], q[:, 0], decay, state, out_state=state)
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "1")
    policy.compute_policy_loss(z, z, z)
    with pytest.raises(AssertionError, match="actions must lie"):
        policy.compute_action_log_probs(x, a - 1)
    with pytest.raises(AssertionError, match="decay must lie"):
        policy.compute_linear_attention(q, q, q, decay + 1)
    assert _native.fast.launched() == before
