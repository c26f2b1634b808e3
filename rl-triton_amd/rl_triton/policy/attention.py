"""Linear attention with a decay for each head and episode ends (csrc/rlk_attention.hip, csrc/rlk_attention_step.hip)."""
import math

import torch

from rl_triton.ops._scan import _CORRECTNESS_WARNINGS
from rl_triton.policy import _native

MAX_HEAD_DIM = 128


def check_heads(q, k, v, dones, state, steps):
    """Checks of queries, keys, values, episode ends and states; `steps`: the tensors have a seq_len axis."""
    names = "[num_envs, seq_len, heads, dim]" if steps else "[num_envs, heads, dim]"
    assert q.is_cuda, "q must be on CUDA"
    assert q.dtype in (torch.float32, torch.bfloat16), f"q: expected float32 or bfloat16, got {q.dtype}"
    assert q.dim() == (4 if steps else 3), f"q must be {names}, got shape {tuple(q.shape)}"
    for name, t in (("k", k), ("v", v)):
        assert t.get_device() == q.get_device(), f"{name} must be on the device of q"
        assert t.dtype == q.dtype, f"{name}: expected {q.dtype} as q, got {t.dtype}"
    assert k.shape == q.shape, f"k shape {k.shape} != q shape {q.shape}"
    assert v.dim() == q.dim() and v.shape[:-1] == q.shape[:-1], f"v shape {v.shape} != q shape {q.shape} but for the last axis"
    for name, t in (("q", q), ("v", v)):
        assert 1 <= t.shape[-1] <= MAX_HEAD_DIM, f"{name}: head dimensions of 1 to {MAX_HEAD_DIM}, got {t.shape[-1]}"
    if dones is not None:
        assert dones.get_device() == q.get_device(), "dones must be on the device of q"
        assert dones.dtype in (torch.float32, torch.bfloat16, torch.bool), f"dones: expected float32, bfloat16 or bool, got {dones.dtype}"
        want = q.shape[:2] if steps else q.shape[:1]
        assert dones.shape == want, f"dones shape {dones.shape} != {want}"
    if state is not None:
        assert state.get_device() == q.get_device() and state.dtype == torch.float32, "state must be float32 on the device of q"
        want = (q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1])
        assert state.shape == want, f"state must have shape {list(want)}, got {list(state.shape)}"


def _check_attention(q, k, v, decay, dones, state, scale, steps):
    """Checks of both forms.  Returns the scale."""
    check_heads(q, k, v, dones, state, steps)
    heads = q.shape[-2]
    assert decay.get_device() == q.get_device() and decay.dtype == torch.float32, "decay must be float32 on the device of q"
    assert decay.shape == (heads,), f"decay must have shape [{heads}], got {tuple(decay.shape)}"
    assert not decay.requires_grad, "decay is a constant of the layer: no gradient is computed for it"
    if scale is None:
        scale = q.shape[-1] ** -0.5
    assert isinstance(scale, (int, float)) and math.isfinite(scale) and scale != 0, f"scale must be a number other than 0, got {scale!r}"
    _native.refuse_forward_derivatives(q, k, v, decay, state)
    if _CORRECTNESS_WARNINGS():
        assert bool(((decay >= 0) & (decay <= 1)).all()), "decay must lie in [0, 1]"
    return float(scale)


def check_out_state(state, out_state):
    """Where a step writes its state: a new tensor, or `out_state` once it is known to be fit for it."""
    assert state.is_contiguous(), "state must be contiguous"
    if out_state is None:
        return torch.empty(state.shape, dtype=state.dtype, device=state.device)
    assert out_state.get_device() == state.get_device() and out_state.dtype == torch.float32 and \
        out_state.shape == state.shape and out_state.is_contiguous(), "out_state must be a contiguous float32 tensor like state"
    apart = abs(out_state.data_ptr() - state.data_ptr())
    assert apart == 0 or apart >= 4 * state.numel(), "out_state overlaps state without being it"
    if torch.is_grad_enabled() and out_state.requires_grad:
        raise RuntimeError("out_state requires a gradient and cannot be written over")
    torch.autograd.graph.increment_version(out_state)  # (a graph that saved what it held has to know)
    return out_state


def _dones(dones):
    return None if dones is None else dones.to(torch.float32).contiguous()


def _inner(x):
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _forward(q, k, v, decay, dones, state, scale):
    e, t, h, dk = q.shape
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    last = torch.empty((e, h, dk, v.shape[-1]), dtype=torch.float32, device=q.device)
    if t == 0:
        return out, last.zero_() if state is None else last.copy_(state)
    if e and h:
        _native.linear_attention(decay, dones, [_native.Pass(q, k, v, out, state, last, scale)])
    return out, last


class _LinearAttention(torch.autograd.Function):
    """The gradients are the same recurrence over other arrays: for an upstream gradient g of the outputs,
    dq_t = scale S_t g_t with S run forward over (v, k), and with R_t = decay (1 - done_t) R_{t+1} + q_t g_t^T
    run from the end, dk_t = scale R_t v_t and dv_t = scale R_t^T k_t."""

    @staticmethod
    def forward(ctx, q, k, v, decay, dones, state, scale):
        ctx.save_for_backward(q, k, v, decay, dones, state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return _forward(q, k, v, decay, dones, state, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_last):
        q, k, v, decay, dones, state = ctx.saved_tensors
        scale = ctx.scale
        wants_q, wants_k, wants_v, _, _, wants_state, _ = ctx.needs_input_grad
        if (grad_out is None and grad_last is None) or not (wants_q or wants_k or wants_v or wants_state):
            return (None,) * 7
        e, t, h, _ = q.shape
        # (the state's gradient comes with that of v)
        grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) if wanted else None
                 for x, wanted in ((q, wants_q), (k, wants_k), (v, wants_v or wants_state))]
        grad_state = torch.empty(q.shape[0], h, q.shape[-1], v.shape[-1], dtype=torch.float32, device=q.device) if wants_state else None
        if t == 0:
            if grad_state is not None:
                grad_state.zero_() if grad_last is None else grad_state.copy_(grad_last)
        elif e and h:
            g = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if grad_out is None else _inner(grad_out)
            last = None if grad_last is None else grad_last.contiguous()
            back = dict(reverse=True, state_scale=1.0 / scale, out_scale=scale)
            passes = []
            if grads[0] is not None:
                passes.append(_native.Pass(g, v, k, grads[0], state, None, scale, transposed=True))
            if grads[1] is not None:
                passes.append(_native.Pass(v, g, q, grads[1], last, None, scale, transposed=True, **back))
            if grads[2] is not None:
                passes.append(_native.Pass(k, q, g, grads[2], last, grad_state, scale, **back))
            _native.linear_attention(decay, dones, passes)
        return (*grads, None, None, grad_state, None)


class _StepOutput(torch.autograd.Function):
    """A step's output where a gradient is wanted of it: it has none, and says so when it is asked for.  `asked` is a tensor of its
    own, so that nothing of the steps before is held."""

    @staticmethod
    def forward(ctx, asked, out):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, grad_out):
        raise RuntimeError("compute_linear_attention_step computes no gradient: a learner runs compute_linear_attention over the steps")


def compute_linear_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    decay: torch.Tensor,
    dones: torch.Tensor | None = None,
    state: torch.Tensor | None = None,
    scale: float | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """
    Linear attention with a decay for each head, over whole sequences of episodes.

    - S[t] = decay[h] * (1 - done[t-1]) * S[t-1] + k[t] v[t]^T,  S[-1] = state, done[-1] = 0
    - out[t] = scale * S[t]^T q[t]

    the recurrence of compute_eligibility_traces with a matrix in place of the trace: no step reads from an episode
    that ended before it.  Computed in chunks of steps with matrix instructions, float32 sums throughout; in
    bfloat16 calls the products of queries and keys, and the state where outputs are read from it, are factors of two bfloat16
    numbers each (2^-15 off), and an output is rounded once.
    Differentiable in q, k, v and state.

    What is not finite, in padded steps for one, reaches no step before it and none past its episode's end; a chunk that
    holds such values is computed step by step, in some twenty times the time.

    Args:
        q, k:  [num_envs, seq_len, heads, dim_k], float32 or bfloat16, GPU; any strides with a contiguous last axis
               (time-major views and slices of a joint projection are read in place, and heads that share keys or
               values may be expanded ones).  Dimensions of 1 to 128.
        v:     [num_envs, seq_len, heads, dim_v], the dtype of q.
        decay: [heads], float32, in [0, 1].  (0 leaves nothing of a state, NaN included.)
        dones: nonzero where the episode ended with that step, [num_envs, seq_len], float32, bfloat16 or bool, or None.
        state: what the sequences go on from, [num_envs, heads, dim_k, dim_v], float32, or None (zeros).
        scale: default dim_k ** -0.5.

    Returns:
        out:   [num_envs, seq_len, heads, dim_v], contiguous, the dtype of q.
        state: after the last step, [num_envs, heads, dim_k, dim_v], float32; zero where that step was done.
    """
    scale = _check_attention(q, k, v, decay, dones, state, scale, True)
    q, k, v = _inner(q), _inner(k), _inner(v)
    decay, dones = decay.contiguous(), _dones(dones)
    state = None if state is None else state.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    (state is not None and state.requires_grad)):
        return _LinearAttention.apply(q, k, v, decay, dones, state, scale)
    return _forward(q, k, v, decay, dones, state, scale)


def compute_linear_attention_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    decay: torch.Tensor,
    state: torch.Tensor,
    dones: torch.Tensor | None = None,
    scale: float | None = None,
    *,
    out_state: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """
    One step of compute_linear_attention for every environment: what an actor calls while it plays.

    - S' = decay[h] * (1 - done) * state + k v^T,  out = scale * S'^T q

    No gradient is computed (a learner runs whole sequences): where one of the inputs requires one, a backward pass through
    the output raises.  The state comes without a graph.

    Args:
        q, k:      [num_envs, heads, dim_k], float32 or bfloat16, GPU.
        v:         [num_envs, heads, dim_v], the dtype of q.
        decay:     [heads], float32, in [0, 1].
        state:     [num_envs, heads, dim_k, dim_v], float32, contiguous.
        dones:     nonzero where the step before ended its episode, [num_envs], float32, bfloat16 or bool, or None.
        scale:     default dim_k ** -0.5.
        out_state: where to write the new state (`state` itself: in place), float32, contiguous; default a new tensor.  As for
                   torch's in-place operations, a backward pass that needs what it held raises, and where gradients are
                   enabled it must not require one.

    Returns:
        out:   [num_envs, heads, dim_v], the dtype of q.
        state: [num_envs, heads, dim_k, dim_v], float32.
    """
    assert state is not None, "state is required"
    scale = _check_attention(q, k, v, decay, dones, state, scale, False)
    out_state = check_out_state(state, out_state)
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if q.shape[0] and q.shape[1]:
        _native.linear_attention_step(decay.contiguous(), _dones(dones),
                                      _native.Pass(_inner(q.detach()), _inner(k.detach()), _inner(v.detach()), out, state.detach(),
                                                   out_state, scale))
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state)):
        out = _StepOutput.apply(torch.empty(0, dtype=out.dtype, device=out.device, requires_grad=True), out)
    return out, out_state
