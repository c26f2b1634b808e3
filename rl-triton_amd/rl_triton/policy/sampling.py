"""Actions sampled from logits with truncation, by given uniform numbers (csrc/rlk_sample.hip)."""
import torch

from rl_triton.ops._scan import _CORRECTNESS_WARNINGS
from rl_triton.policy import _native
from rl_triton.policy.log_probs import _as_rows

MAX_ACTIONS = 1 << 20


def compute_sampled_actions(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    temperature: float = 1.0,
    *,
    top_k: int | None = None,
    top_p: float | None = None,
    min_p: float | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """
    Actions sampled from softmax(logits / temperature), truncated to the likeliest, by given uniform numbers.

    Of the actions in the order of their logits, the largest first and of equal ones the first, are kept

    - the first `top_k`;
    - of these the shortest beginning that holds at least `top_p` of their probability;
    - of these the ones at least `min_p` times as likely as the first.

    With p the probabilities of the kept ones, made to sum to 1, the action is the first, in the order of their numbers, with
    p[0] + .. + p[action] > uniform.

    Probabilities are summed as whole numbers of 2^-43 of the largest, formed in float64, so an action depends neither on the order of
    the sums nor on the storage of the rows, and is the definition's unless a uniform number lies as near to a border as the roundings add up to:
    some 1e-13 for a few actions, 1e-11 for a vocabulary, never above num_actions * 2^-44.  An action that is
    not allowed has a logit of -inf and is never taken; of a row of nothing else the action is -1 and the log-probability -inf, of a row with
    a NaN -1 and NaN.  A largest logit of +inf shares everything among its equals.  No gradient is computed.

    Args:
        logits:      [..., num_actions], float32 or bfloat16, GPU, as for compute_action_log_probs; up to 2^20 actions.
        uniforms:    [...], float32, in [0, 1): one number per row.  Others are taken as the nearest that is (NaN as 0).
        temperature: what the logits are divided by (default 1), from 1e-38 to 1e38.
        top_k:       at least 1, or None (all).
        top_p:       above 0 and up to 1, or None (all).
        min_p:       0 to 1, or None (none).

    Returns:
        actions:   [...], int64.
        log_probs: [...], float32: log p[action], of the distribution that it was sampled from.
    """
    assert logits.is_cuda, "logits must be on CUDA"
    assert logits.dtype in (torch.float32, torch.bfloat16), f"logits: expected float32 or bfloat16, got {logits.dtype}"
    assert logits.dim() >= 1 and 1 <= logits.shape[-1] <= MAX_ACTIONS, \
        f"logits must have an action axis of 1 to {MAX_ACTIONS}, got shape {tuple(logits.shape)}"
    assert uniforms.get_device() == logits.get_device(), "uniforms must be on the device of logits"
    assert uniforms.dtype == torch.float32, f"uniforms: expected float32, got {uniforms.dtype}"
    assert uniforms.shape == logits.shape[:-1], f"uniforms shape {uniforms.shape} != logits shape {logits.shape} without its last axis"
    assert isinstance(temperature, (int, float)) and 1e-38 <= temperature <= 1e38, \
        f"temperature must be a number from 1e-38 to 1e38, got {temperature!r}"
    assert top_k is None or (isinstance(top_k, int) and not isinstance(top_k, bool) and top_k >= 1), \
        f"top_k must be a whole number of at least 1 or None, got {top_k!r}"
    assert top_p is None or (isinstance(top_p, (int, float)) and 0 < top_p <= 1), f"top_p must be a number above 0 and up to 1 or None, got {top_p!r}"
    assert min_p is None or (isinstance(min_p, (int, float)) and 0 <= min_p <= 1), f"min_p must be a number from 0 to 1 or None, got {min_p!r}"
    _native.refuse_forward_derivatives(logits)
    if _CORRECTNESS_WARNINGS():
        assert uniforms.numel() == 0 or bool(((uniforms >= 0) & (uniforms < 1)).all()), "uniforms must lie in [0, 1)"
    actions = torch.empty(uniforms.shape, dtype=torch.int64, device=logits.device)
    log_probs = torch.empty(uniforms.shape, dtype=torch.float32, device=logits.device)
    if actions.numel():
        _native.sample_actions(_as_rows(logits.detach()), uniforms.contiguous(), float(temperature), min(top_k or 0, MAX_ACTIONS),
                               1.0 if top_p is None else float(top_p), float(min_p or 0.0), actions, log_probs)
    return actions, log_probs
