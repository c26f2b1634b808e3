"""The clipped policy loss with a KL term and its gradient (csrc/rlk_policy_loss.hip, csrc/rlk_logits_loss.hip)."""
import math

import torch

from rl_triton.ops._scan import _CORRECTNESS_WARNINGS, _float_io
from rl_triton.policy import _native
from rl_triton.policy.log_probs import _as_rows, _check_rows


def _number(x, name, low=-math.inf):
    assert isinstance(x, (int, float)) and math.isfinite(x) and x >= low, \
        f"{name} must be a number" + (f" of at least {low}" if low > -math.inf else "") + f", got {x!r}"
    return float(x)


def _check_terms(lead, shape, dtype, old_log_probs, advantages, ref_log_probs, mask, clip_low, clip_high, kl_coef, dual_clip,
                 reduction):
    """Checks of what both losses read; the clipping as numbers (0: no dual clip)."""
    for name, t in (("old_log_probs", old_log_probs), ("advantages", advantages), ("ref_log_probs", ref_log_probs), ("mask", mask)):
        if t is None and name in ("ref_log_probs", "mask"):
            continue
        assert t.get_device() == lead.get_device() and t.is_cuda, f"{name} must be on the device of the policy's outputs"
        assert t.dtype == dtype, f"{name}: expected {dtype}, got {t.dtype}"
        assert t.shape == shape, f"{name} shape {t.shape} != {shape}"
    assert reduction in ("steps", "rows"), f'reduction must be "steps" or "rows", got {reduction!r}'
    _number(kl_coef, "kl_coef")
    assert dual_clip is None or _number(dual_clip, "dual_clip") > 1, f"dual_clip must be above 1, got {dual_clip!r}"
    return _number(clip_low, "clip_low", 0), _number(clip_high, "clip_high", 0), 0.0 if dual_clip is None else float(dual_clip)


def compute_policy_loss(
    log_probs: torch.Tensor,
    old_log_probs: torch.Tensor,
    advantages: torch.Tensor,
    ref_log_probs: torch.Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    kl_coef: float = 0.0,
    *,
    dual_clip: float | None = None,
    mask: torch.Tensor | None = None,
    reduction: str = "steps",
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    The clipped policy loss with a KL term, and its gradient.

    Step by step, with D = log_probs - old_log_probs, r = exp D and d = ref_log_probs - log_probs:

    - policy = max(-A r, -A clip(r, 1 - clip_low, 1 + clip_high)), at most -A dual_clip where A < 0
    - kl     = exp d - 1 - d  (0 without ref_log_probs)
    - loss   = mean(policy) + kl_coef mean(kl)

    The mean is over the steps with mask != 0 (reduction "steps"), or over rows of the means of their steps, rows
    without any left out ("rows").  What a masked step holds has no part in anything, NaN included.  With no step
    at all the loss is 0.

    The loss comes with its gradient, not with a graph: `log_probs.backward(grad)` goes on from it into the policy.

    Args:
        log_probs:     log-probabilities of the taken actions under the policy, [num_envs, seq_len], float32 or
                       bfloat16 (every tensor of the call alike), GPU.
        old_log_probs: the same under the policy that took them.
        advantages:    [num_envs, seq_len] (compute_gae, compute_gae_normalized, compute_vtrace).
        ref_log_probs: the same under a reference policy, or None.
        clip_low, clip_high: how far the ratio may leave 1 (default 0.2 each).
        kl_coef:       what the KL term counts for (0: it is measured, and has no part in the loss or the gradient).
        dual_clip:     bound of the ratio for negative advantages, above 1, or None.
        mask:          nonzero for the steps that take part, or None for all.
        reduction:     "steps" or "rows".

    Returns:
        loss:  float32, no dimensions.
        grad:  d loss / d log_probs, [num_envs, seq_len], the inputs' dtype.
        means: float32 [4]: mean(policy), mean(kl), the share of steps whose gradient the clipping took away, and
               mean(r - 1 - D), an estimate of the KL divergence from the old policy.
    """
    assert log_probs.is_cuda, "log_probs must be on CUDA"
    assert _float_io(log_probs, log_probs), f"log_probs: expected float32 (or bfloat16 throughout), got {log_probs.dtype}"
    assert log_probs.dim() == 2, f"log_probs must be [num_envs, seq_len], got shape {tuple(log_probs.shape)}"
    clip = _check_terms(log_probs, log_probs.shape, log_probs.dtype, old_log_probs, advantages, ref_log_probs, mask, clip_low,
                        clip_high, kl_coef, dual_clip, reduction)
    out = torch.empty(5, dtype=torch.float32, device=log_probs.device)
    grad = torch.empty(log_probs.shape, dtype=log_probs.dtype, device=log_probs.device)
    loss, means = out[0], out[1:]
    _native.policy_loss(log_probs.detach().contiguous(), old_log_probs.contiguous(), advantages.contiguous(),
                        None if ref_log_probs is None else ref_log_probs.contiguous(),
                        None if mask is None else mask.contiguous(), clip, float(kl_coef), reduction == "rows", loss, means, grad)
    return loss, grad, means


def compute_policy_loss_from_logits(
    logits: torch.Tensor,
    actions: torch.Tensor,
    old_log_probs: torch.Tensor,
    advantages: torch.Tensor,
    ref_log_probs: torch.Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    kl_coef: float = 0.0,
    entropy_coef: float = 0.0,
    temperature: float = 1.0,
    *,
    dual_clip: float | None = None,
    mask: torch.Tensor | None = None,
    reduction: str = "steps",
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    compute_policy_loss from the policy's logits, minus entropy_coef times the mean entropy, with the gradient
    of the logits.

    The log-probabilities are those of compute_action_log_probs.  A row of logits is read once, held while its
    loss is found, and its gradient written from there (rows of up to 256 KB; longer ones are read twice, and so are up to 64 rows
    of 64 KB and more, which several workgroups share).  Masked steps have zero gradients whatever their logits hold.
    `logits.backward(grad)` goes on into the policy.

    Args:
        logits:       [num_envs, seq_len, num_actions], float32 or bfloat16, GPU.
        actions:      the taken actions, [num_envs, seq_len], int64, in [0, num_actions).
        old_log_probs, advantages, ref_log_probs, mask: as for compute_policy_loss, float32.
        entropy_coef: what the entropies count for.
        temperature:  what the logits are divided by.
        The others as for compute_policy_loss.

    Returns:
        loss:  float32, no dimensions.
        grad:  d loss / d logits, contiguous, the logits' dtype.
        means: float32 [5]: those of compute_policy_loss, and the mean entropy.
    """
    assert logits.dim() == 3, f"logits must be [num_envs, seq_len, num_actions], got shape {tuple(logits.shape)}"
    if mask is not None and _CORRECTNESS_WARNINGS():
        _check_rows(logits, torch.where(mask.ne(0), actions, 0) if mask.shape == actions.shape else actions, temperature)
    else:
        _check_rows(logits, actions, temperature)
    _number(entropy_coef, "entropy_coef")
    clip = _check_terms(logits, actions.shape, torch.float32, old_log_probs, advantages, ref_log_probs, mask, clip_low, clip_high,
                        kl_coef, dual_clip, reduction)
    out = torch.empty(6, dtype=torch.float32, device=logits.device)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    loss, means = out[0], out[1:]
    _native.policy_loss_from_logits(_as_rows(logits.detach()), actions.contiguous(), float(temperature),
                                    old_log_probs.contiguous(), advantages.contiguous(),
                                    None if ref_log_probs is None else ref_log_probs.contiguous(),
                                    None if mask is None else mask.contiguous(), clip, float(kl_coef), float(entropy_coef),
                                    reduction == "rows", loss, means, grad)
    return loss, grad, means
