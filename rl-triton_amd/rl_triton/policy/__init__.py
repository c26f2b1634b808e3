"""What a learner computes around the return estimators, on the same hand-written HIP kernels.

Not in the reference's API, whose surface rl_triton itself keeps:
  * compute_action_log_probs: log-probabilities and entropies of the taken actions, from logits --
    what V-trace, the policy loss and a KL term read;
  * compute_policy_loss: the clipped policy loss with a KL term and its gradient, from log-probabilities;
  * compute_policy_loss_from_logits: the same from logits, with the gradient of the logits, in one pass over them;
  * compute_linear_attention, compute_linear_attention_step: a memory over the steps of an episode, the done-masked
    recurrence of the estimators with a matrix for its state, over whole sequences and one step at a time.
"""
from rl_triton._native import public_entry as _public_entry
from rl_triton.policy import attention as _attention
from rl_triton.policy import log_probs as _log_probs
from rl_triton.policy import loss as _loss

# The Python implementations, each behind the C++ fast path (rl_triton._native.public_entry).
compute_action_log_probs = _public_entry(_log_probs.compute_action_log_probs, "action_log_probs")
compute_linear_attention = _public_entry(_attention.compute_linear_attention, "linear_attention")
compute_linear_attention_step = _public_entry(_attention.compute_linear_attention_step, "linear_attention_step")
compute_policy_loss = _public_entry(_loss.compute_policy_loss, "policy_loss")
compute_policy_loss_from_logits = _public_entry(_loss.compute_policy_loss_from_logits, "policy_loss_from_logits")

__all__ = [
    "compute_action_log_probs",
    "compute_linear_attention",
    "compute_linear_attention_step",
    "compute_policy_loss",
    "compute_policy_loss_from_logits",
]
