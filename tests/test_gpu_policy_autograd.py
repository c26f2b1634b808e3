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


def _requested(which):
    """Bytes asked of the allocator (what it hands out depends on the blocks that it has from before)."""
    return torch.cuda.memory_stats()[f"requested_bytes.all.{which}"]


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


def test_a_step_says_that_it_has_no_gradient():
    """Steps that are unrolled into a loss: the error comes when the gradient is asked for, not a gradient without a part of it."""
    q, k, v, decay, state = _step_args(True)
    plain = policy.compute_linear_attention_step(q.detach(), k.detach(), v.detach(), decay, state)
    for wrt in (q, k, v, state.clone().requires_grad_()):
        args = [q.detach(), k.detach(), v.detach(), decay, state]
        if wrt is q or wrt is k or wrt is v:
            args[0 if wrt is q else 1 if wrt is k else 2] = wrt
        else:
            args[4] = wrt
        out, new = policy.compute_linear_attention_step(*args)
        assert torch.equal(out, plain[0]) and torch.equal(new, plain[1])
        assert not new.requires_grad
        weight = torch.ones((), device="cuda", requires_grad=True)
        with pytest.raises(RuntimeError, match="compute_linear_attention_step"):
            (weight * out).sum().backward()
        out, new = policy.compute_linear_attention_step(*args, out_state=torch.empty_like(state))
        assert torch.equal(out, plain[0]) and not new.requires_grad
        with pytest.raises(RuntimeError, match="compute_linear_attention_step"):
            out.sum().backward()
        with torch.no_grad():
            assert not any(t.requires_grad for t in policy.compute_linear_attention_step(*args))
    assert not any(t.requires_grad for t in plain)


def test_unrolled_steps_hold_nothing_back():
    """What a step's results hold on to does not grow with the steps before them."""
    q, k, v, decay, state = _step_args(True)
    sizes = []
    for _ in range(6):
        out, state = policy.compute_linear_attention_step(q * 1, k * 1, v * 1, decay, state)
        sizes.append(_requested("current"))
    assert sizes[-1] == sizes[1] and out.requires_grad


@pytest.mark.parametrize("seq_len", [40, 700])  # (one segment and several)
def test_only_the_gradients_that_are_asked_for_are_computed(seq_len):
    """With some of the inputs frozen: the same gradients of the others, and no memory taken for those of the frozen ones."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    E = 64 if seq_len == 40 else 1
    inputs = n(E, seq_len, 2, 64), n(E, seq_len, 2, 64), n(E, seq_len, 2, 64), n(E, 2, 64, 64)
    decay, up, us = torch.tensor([0.99, 0.9], device="cuda"), n(E, seq_len, 2, 64), n(E, 2, 64, 64)

    def run(wanted):
        leaves = [t.clone().requires_grad_(w) for t, w in zip(inputs, wanted)]
        outs = policy.compute_linear_attention(*leaves[:3], decay, None, leaves[3])
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = _requested("current")
        grads = torch.autograd.grad(outs, [t for t in leaves if t.requires_grad], (up, us))
        return grads, _requested("peak") - before

    run((True,) * 4)  # (the scratch memory is there)
    full, _ = run((True,) * 4)
    for wanted in ((True, False, False, False), (False, True, False, False), (False, False, True, False), (False, False, False, True),
                   (True, False, True, False), (False, True, False, True), (False, True, True, True)):
        grads, peak = run(wanted)
        assert all(torch.equal(a, b) for a, b in zip(grads, [x for x, w in zip(full, wanted) if w]))
        # the state's gradient comes with v's: room for both
        room = sum(x.numel() * 4 for x, w in zip(inputs, (*wanted[:2], wanted[2] or wanted[3], wanted[3])) if w)
        assert peak <= room, (wanted, peak, room)
