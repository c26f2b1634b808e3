"""What torch's automatic differentiation has to know of rl_triton.policy's calls: which tensors they write, and which derivatives
they cannot give."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import rl_triton.policy as policy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["0", "1"], ids=["fast", "checked"])
def _path(request, monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", request.param)


def _step_args(grad=False):
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v = (n(3, 2, 16).requires_grad_(grad) for _ in range(3))
    return q, k, v, torch.tensor([0.9, 0.5], device="cuda"), n(3, 2, 16, 16)


def test_a_state_written_in_place_is_a_new_version():
    """A sequence's backward pass needs the state that it began with: once a step has written over it, torch has to refuse."""
    q, k, v, decay, state = _step_args()
    leaf = torch.randn(3, 5, 2, 16, device="cuda", requires_grad=True)
    out, _ = policy.compute_linear_attention(leaf, leaf, leaf, decay, None, state)
    before = state._version
    policy.compute_linear_attention_step(q, k, v, decay, state, out_state=state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    # written elsewhere, or into a view: the version is the storage's
    other = torch.empty(2, *state.shape, device="cuda")
    out, _ = policy.compute_linear_attention(leaf, leaf, leaf, decay, None, other[1].copy_(state))
    policy.compute_linear_attention_step(q, k, v, decay, state, out_state=other[1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    version = state._version
    policy.compute_linear_attention_step(q, k, v, decay, state)  # (a new tensor: `state` stays as it is)
    assert state._version == version


def test_a_tensor_with_a_gradient_is_not_written_over():
    q, k, v, decay, state = _step_args()
    leaf = state.clone().requires_grad_()
    for out_state in (leaf, leaf * 1):
        keep = out_state.detach().clone()
        with pytest.raises(RuntimeError, match="requires a gradient"):
            policy.compute_linear_attention_step(q, k, v, decay, state, out_state=out_state)
        assert torch.equal(out_state, keep)
    with torch.no_grad():  # as for torch's own in-place operations
        policy.compute_linear_attention_step(q, k, v, decay, state, out_state=leaf)
    want = policy.compute_linear_attention_step(q, k, v, decay, state)[1]
    assert torch.equal(leaf.detach(), want)
    with torch.inference_mode():
        frozen = state.clone()
        policy.compute_linear_attention_step(q, k, v, decay, frozen, out_state=frozen)
    assert torch.equal(frozen, want)


def test_forward_derivatives_are_refused():
    """A dual tensor need not require a gradient: its tangent must not be dropped in silence."""
    q, k, v, decay, state = _step_args()
    x, a = torch.randn(4, 7, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    seq = torch.randn(3, 5, 2, 16, device="cuda")
    for mode in (torch.enable_grad, torch.no_grad):
        for wants in (False, True):
            with mode(), fwAD.dual_level():
                dual = lambda t: fwAD.make_dual(t.detach().clone().requires_grad_(wants), torch.ones_like(t))  # noqa: E731
                calls = [lambda: policy.compute_action_log_probs(dual(x), a),
                         lambda: policy.compute_linear_attention(dual(seq), seq, seq, decay),
                         lambda: policy.compute_linear_attention(seq, dual(seq), seq, decay),
                         lambda: policy.compute_linear_attention(seq, seq, dual(seq), decay),
                         lambda: policy.compute_linear_attention(seq, seq, seq, decay, None, dual(state)),
                         lambda: policy.compute_linear_attention(seq, seq, seq, fwAD.make_dual(decay, torch.ones_like(decay))),
                         lambda: policy.compute_linear_attention_step(dual(q), k, v, decay, state),
                         lambda: policy.compute_linear_attention_step(q, k, v, decay, dual(state))]
                for call in calls:
                    with pytest.raises((NotImplementedError, RuntimeError), match="[Ff]orward"):
                        call()
                policy.compute_linear_attention(seq, seq, seq, decay)  # (no dual among them: as ever)
                policy.compute_action_log_probs(x, a)
