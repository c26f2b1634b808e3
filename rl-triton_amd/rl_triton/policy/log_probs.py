"""Log-probabilities and entropies of taken actions, from logits (csrc/rlk_action_log_probs.hip)."""
import math

import torch

from rl_triton.ops._scan import _CORRECTNESS_WARNINGS
from rl_triton.policy import _native


def _check_rows(logits, actions, temperature):
    """The checks of every call on logits; they raise before anything is launched."""
    assert logits.is_cuda, "logits must be on CUDA"
    assert logits.dtype in (torch.float32, torch.bfloat16), f"logits: expected float32 or bfloat16, got {logits.dtype}"
    assert logits.dim() >= 1 and logits.shape[-1] >= 1, f"logits must have an action axis, got shape {tuple(logits.shape)}"
    assert actions.get_device() == logits.get_device(), "actions must be on the device of logits"
    assert actions.dtype == torch.int64, f"actions: expected int64, got {actions.dtype}"
    assert actions.shape == logits.shape[:-1], f"actions shape {actions.shape} != logits shape {logits.shape} without its last axis"
    assert isinstance(temperature, (int, float)) and 1e-38 <= temperature <= 1e38, \
        f"temperature must be a number from 1e-38 to 1e38 (float32 holds its reciprocal), got {temperature!r}"
    if _CORRECTNESS_WARNINGS():
        assert actions.numel() == 0 or bool(((actions >= 0) & (actions < logits.shape[-1])).all()), \
            "actions must lie in [0, num_actions)"


def _as_rows(logits):
    """`logits` as [envs, steps, actions] with contiguous actions, without a copy where its strides allow."""
    if logits.dim() != 3:
        lead = logits.shape[:-1]
        logits = logits.reshape(1, math.prod(lead), logits.shape[-1])
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    return logits


def _forward(logits, actions, temperature, norms):
    shape = actions.shape
    log_probs = torch.empty(shape, dtype=torch.float32, device=logits.device)
    entropies = torch.empty_like(log_probs)
    if actions.numel():
        _native.action_log_probs(_as_rows(logits), actions.contiguous(), temperature, log_probs, entropies, norms)
    return log_probs, entropies


class _ActionLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, temperature):
        norms = torch.empty((*actions.shape, 2), dtype=torch.float32, device=logits.device)
        log_probs, entropies = _forward(logits, actions, temperature, norms)
        ctx.save_for_backward(logits, actions, entropies, norms)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return log_probs, entropies

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_log_probs, grad_entropies):
        logits, actions, entropies, norms = ctx.saved_tensors
        if grad_log_probs is None and grad_entropies is None:
            return None, None, None
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if actions.numel():
            gl, ge = (None if g is None else g.contiguous() for g in (grad_log_probs, grad_entropies))
            _native.action_log_probs_backward(_as_rows(logits), actions.contiguous(), ctx.temperature, entropies, norms,
                                              gl, ge, grad)
        return grad, None, None


def compute_action_log_probs(
    logits: torch.Tensor,
    actions: torch.Tensor,
    temperature: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """
    Log-probabilities of the taken actions and entropies of their distributions.

    With x = logits / temperature and p = softmax(x):

    - log_probs = x[a] - log sum_j exp x[j]
    - entropies = -sum_j p[j] log p[j]

    One pass over the logits; differentiable in them.  An action that is not allowed has a logit of -inf and no
    part in either (a row of nothing else has log-probability -inf, entropy 0 and a zero gradient).  An action
    outside [0, num_actions) gives NaN.

    Args:
        logits:      [..., num_actions], float32 or bfloat16, GPU; usually [num_envs, seq_len, num_actions], of any
                     strides as long as the actions of a row are contiguous (others are copied).
        actions:     the taken actions, [...], int64.
        temperature: what the logits are divided by (default 1), from 1e-38 to 1e38.

    Returns:
        log_probs, entropies: [...], float32 whatever the logits' type (ratios of probabilities are taken of them).
    """
    _check_rows(logits, actions, temperature)
    _native.refuse_forward_derivatives(logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _ActionLogProbs.apply(logits, actions, float(temperature))
    return _forward(logits, actions, float(temperature), None)
