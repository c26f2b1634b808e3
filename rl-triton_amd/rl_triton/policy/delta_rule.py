"""The gated delta rule (csrc/rlk_delta.hip, csrc/rlk_delta_records.hip, csrc/rlk_delta_walk.hip, csrc/rlk_delta_gradients.hip)."""
import math

import torch

from rl_triton.ops._scan import _CORRECTNESS_WARNINGS
from rl_triton.policy import _native
from rl_triton.policy.attention import _dones, _inner, check_heads, check_out_state

MAX_CHUNKS = 1 << 22  # heads times chunks of 64 steps: what one environment's launches hold


def _check(q, k, v, log_decays, betas, dones, state, scale, steps):
    """Checks of both forms; `steps`: the tensors have a seq_len axis.  Returns the scale."""
    check_heads(q, k, v, dones, state, steps)
    lead = q.shape[:-1]
    for name, t in (("log_decays", log_decays), ("betas", betas)):
        if t is None and name == "log_decays":
            continue
        assert t.get_device() == q.get_device() and t.dtype == torch.float32, f"{name} must be float32 on the device of q"
        assert t.shape == lead, f"{name} shape {t.shape} != {lead}"
    if steps:
        assert q.shape[2] * -(-q.shape[1] // 64) <= MAX_CHUNKS and q.shape[1] <= 1 << 30, \
            f"heads times chunks of 64 steps: at most {MAX_CHUNKS}, got {q.shape[2]} heads of {q.shape[1]} steps"
    if scale is None:
        scale = q.shape[-1] ** -0.5
    assert isinstance(scale, (int, float)) and math.isfinite(scale) and abs(scale) <= 3.4e38, f"scale must be a number, got {scale!r}"
    _native.refuse_forward_derivatives(q, k, v, log_decays, betas, state)
    if _CORRECTNESS_WARNINGS():
        assert log_decays is None or bool((log_decays <= 0).all()), "log_decays must not be above 0"
        assert bool(((betas >= 0) & (betas <= 2)).all()), "betas must lie in [0, 2]"
    return float(scale)


def _flat(t):
    return None if t is None else t.contiguous()


def _forward(q, k, v, log_decays, betas, dones, state, scale, keep=False):
    e, t, h, dk = q.shape
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    last = torch.empty((e, h, dk, v.shape[-1]), dtype=torch.float32, device=q.device)
    saved = None
    if t == 0:
        last.zero_() if state is None else last.copy_(state)
    elif e and h:
        saved = _native.gated_delta_rule(q, k, v, out, log_decays, betas, dones, state, last, scale, keep)
    return out, last, saved


class _GatedDeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decays, betas, dones, state, scale):
        out, last, saved = _forward(q, k, v, log_decays, betas, dones, state, scale, True)
        ctx.save_for_backward(q, k, v, log_decays, betas, dones, state, saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_last):
        q, k, v, log_decays, betas, dones, state, saved = ctx.saved_tensors
        wants = ctx.needs_input_grad
        if grad_out is None and grad_last is None:
            return (None,) * 8
        grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) if wanted else None
                 for x, wanted in zip((q, k, v, log_decays, betas), wants)]
        grad_state = torch.empty(state.shape, dtype=state.dtype, device=state.device) if wants[6] else None
        e, t, h, _ = q.shape
        if t == 0:
            if grad_state is not None:
                grad_state.zero_() if grad_last is None else grad_state.copy_(grad_last)
        elif e and h:
            g = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if grad_out is None else _inner(grad_out)
            _native.gated_delta_rule_backward(q, k, v, log_decays, betas, dones, state, ctx.scale, saved, g, _flat(grad_last), grads, grad_state)
        return (*grads, None, grad_state, None)


def compute_gated_delta_rule(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decays: torch.Tensor | None,
    betas: torch.Tensor,
    dones: torch.Tensor | None = None,
    state: torch.Tensor | None = None,
    scale: float | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """
    The gated delta rule over whole sequences of episodes: a memory that writes what it does not already read.

    - S~[t] = exp(log_decays[t]) * (1 - done[t-1]) * S[t-1],  S[-1] = state, done[-1] = 0
    - S[t] = S~[t] + k[t] u[t]^T,  u[t] = betas[t] * (v[t] - S~[t]^T k[t])
    - out[t] = scale * S[t]^T q[t]

    compute_linear_attention with gates that the policy sets at every step, and with the value that a key already reads
    taken off what is written under it.  Keys are expected to have length 1 (compute_query_key_norms), so that betas
    up to 1 (2 with sign changes) keep the state bounded.  Computed in chunks of 64 steps with matrix instructions; states, gates and their
    gradients to float32's accuracy, that of a gate however little it leaves of the state; an output rounded once.  A chunk's
    rounding counts in the state that it begins with: where its steps erase it, up to some 2^-18 of it is left, and where betas near 2 turn it back and forth along
    keys that are nearly alike, results are off by up to 2^-12 of it (float32 step by step: 2^-20).
    Differentiable in q, k, v, log_decays, betas and state.  For the backward pass a call keeps the state before every chunk
    and the corrections of every step in float32.

    What is not finite, in padded steps for one, reaches no step before it and none past its episode's end; a chunk that
    holds such values is computed step by step, more slowly.

    Args:
        q, k:       [num_envs, seq_len, heads, dim_k], float32 or bfloat16, GPU; any strides with a contiguous last axis
                    (as in compute_linear_attention).  Dimensions of 1 to 128.
        v:          [num_envs, seq_len, heads, dim_v], the dtype of q.
        log_decays: [num_envs, seq_len, heads], float32, at most 0, or None (nothing is forgotten).  Below -104 (-inf) nothing
                    of the state stays, NaN included, as at an episode's end, and the gradient is 0.
        betas:      [num_envs, seq_len, heads], float32.
        dones:      nonzero where the episode ended with that step, [num_envs, seq_len], float32, bfloat16 or bool, or None.
        state:      what the sequences go on from, [num_envs, heads, dim_k, dim_v], float32, or None (zeros).
        scale:      default dim_k ** -0.5.

    Returns:
        out:   [num_envs, seq_len, heads, dim_v], contiguous, the dtype of q.
        state: after the last step, [num_envs, heads, dim_k, dim_v], float32; zero where that step was done.
    """
    scale = _check(q, k, v, log_decays, betas, dones, state, scale, True)
    q, k, v = _inner(q), _inner(k), _inner(v)
    log_decays, betas, dones, state = _flat(log_decays), _flat(betas), _dones(dones), _flat(state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decays, betas, state)):
        return _GatedDeltaRule.apply(q, k, v, log_decays, betas, dones, state, scale)
    return _forward(q, k, v, log_decays, betas, dones, state, scale)[:2]


class _StepOutput(torch.autograd.Function):
    """A step's output where a gradient is wanted of it (as compute_linear_attention_step's)."""

    @staticmethod
    def forward(ctx, asked, out):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, grad_out):
        raise RuntimeError("compute_gated_delta_rule_step computes no gradient: a learner runs compute_gated_delta_rule over the steps")


def compute_gated_delta_rule_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decays: torch.Tensor | None,
    betas: torch.Tensor,
    state: torch.Tensor,
    dones: torch.Tensor | None = None,
    scale: float | None = None,
    *,
    out_state: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """
    One step of compute_gated_delta_rule for every environment: what an actor calls while it plays.

    - S~ = exp(log_decays) * (1 - done) * state,  S' = S~ + k (betas * (v - S~^T k))^T,  out = scale * S'^T q

    No gradient is computed (a learner runs whole sequences): where one of the inputs requires one, a backward pass through
    the output raises.  The state comes without a graph.

    Args:
        q, k:       [num_envs, heads, dim_k], float32 or bfloat16, GPU.
        v:          [num_envs, heads, dim_v], the dtype of q.
        log_decays: [num_envs, heads], float32, at most 0, or None.
        betas:      [num_envs, heads], float32.
        state:      [num_envs, heads, dim_k, dim_v], float32, contiguous.
        dones:      nonzero where the step before ended its episode, [num_envs], float32, bfloat16 or bool, or None.
        scale:      default dim_k ** -0.5.
        out_state:  where to write the new state, as for compute_linear_attention_step; default a new tensor.

    Returns:
        out:   [num_envs, heads, dim_v], the dtype of q.
        state: [num_envs, heads, dim_k, dim_v], float32.
    """
    assert state is not None, "state is required"
    scale = _check(q, k, v, log_decays, betas, dones, state, scale, False)
    out_state = check_out_state(state, out_state)
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if q.shape[0] and q.shape[1]:
        _native.gated_delta_rule_step(*(None if t is None else t.detach() for t in (_inner(q), _inner(k), _inner(v))), out,
                                      *(None if t is None else t.detach() for t in (_flat(log_decays), _flat(betas))), _dones(dones),
                                      state.detach(), out_state, scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decays, betas, state)):
        out = _StepOutput.apply(torch.empty(0, dtype=out.dtype, device=out.device, requires_grad=True), out)
    return out, out_state
