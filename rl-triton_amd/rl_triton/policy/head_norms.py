"""Queries and keys normed head by head and rotated by their positions (csrc/rlk_head_norms.hip)."""
import math

import torch

from rl_triton.ops._scan import _CORRECTNESS_WARNINGS
from rl_triton.policy import _native
from rl_triton.policy.attention import _inner

MAX_DIM, MAX_HEADS = 256, 65536


def _check(q, k, q_weight, k_weight, positions, base, rotary_dim, eps):
    assert q.is_cuda, "q must be on CUDA"
    assert q.dtype in (torch.float32, torch.bfloat16), f"q: expected float32 or bfloat16, got {q.dtype}"
    assert q.dim() in (3, 4), f"q must be [num_envs, seq_len, heads, dim] or [num_envs, heads, dim], got shape {tuple(q.shape)}"
    assert k.get_device() == q.get_device(), "k must be on the device of q"
    assert k.dtype == q.dtype, f"k: expected {q.dtype} as q, got {k.dtype}"
    assert k.dim() == q.dim() and k.shape[:-2] == q.shape[:-2] and k.shape[-1] == q.shape[-1], \
        f"k shape {k.shape} != q shape {q.shape} but for the heads"
    dim = q.shape[-1]
    assert 1 <= dim <= MAX_DIM, f"q: head dimensions of 1 to {MAX_DIM}, got {dim}"
    assert q.shape[-2] <= MAX_HEADS and k.shape[-2] <= MAX_HEADS, f"at most {MAX_HEADS} heads"
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None:
            assert t.get_device() == q.get_device() and t.dtype == torch.float32, f"{name} must be float32 on the device of q"
            assert t.shape == (dim,), f"{name} must have shape [{dim}], got {tuple(t.shape)}"
    if rotary_dim is None:
        rotary_dim = dim if positions is not None else 0
    assert isinstance(rotary_dim, int) and 0 <= rotary_dim <= dim and rotary_dim % 2 == 0, \
        f"rotary_dim must be an even number from 0 to {dim}, got {rotary_dim!r}"
    if positions is not None:
        assert positions.get_device() == q.get_device(), "positions must be on the device of q"
        assert positions.dtype == torch.int64, f"positions: expected int64, got {positions.dtype}"
        assert positions.shape == q.shape[:-2], f"positions shape {positions.shape} != {q.shape[:-2]}"
    assert isinstance(base, (int, float)) and math.isfinite(base) and base > 0, f"base must be a positive number, got {base!r}"
    assert isinstance(eps, (int, float)) and 0 <= eps <= 3.4e38, f"eps must be a number of at least 0, got {eps!r}"
    _native.refuse_forward_derivatives(q, k, q_weight, k_weight)
    if _CORRECTNESS_WARNINGS():
        assert positions is None or positions.numel() == 0 or bool((positions >= 0).all()), "positions must not be negative"
    return rotary_dim


def _forward(q, k, q_weight, k_weight, positions, settings):
    outs = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k)]
    if q.numel() or k.numel():
        _native.query_key_norms(q, k, *outs, q_weight, k_weight, positions, *settings)
    return tuple(outs)


class _QueryKeyNorms(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, settings):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.settings = settings
        ctx.set_materialize_grads(False)
        return _forward(q, k, q_weight, k_weight, positions, settings)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, q_weight, k_weight, positions = ctx.saved_tensors
        wants = ctx.needs_input_grad
        ups = [None if g is None else _inner(g) for g in (grad_q, grad_k)]
        to = [torch.empty(x.shape, dtype=x.dtype, device=x.device) if wanted and g is not None else None
              for x, wanted, g in ((q, wants[0], ups[0]), (k, wants[1], ups[1]), (q_weight, wants[2], ups[0]), (k_weight, wants[3], ups[1]))]
        if any(t is not None for t in to):
            if q.numel() or k.numel():
                _native.query_key_norms_backward(q, k, *ups, *to, q_weight, k_weight, positions, *ctx.settings)
            else:
                for t in to[2:]:
                    if t is not None:
                        t.zero_()
        return (*to, None, None)


def compute_query_key_norms(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    *,
    base: float = 10000.0,
    rotary_dim: int | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """
    Queries and keys normed head by head and rotated by their positions, in one pass.

    - y = x / sqrt(mean(x^2) + eps) * weight, the mean over a head's elements
    - each pair (y[a], y[b]) of the first `rotary_dim` elements is turned by the angle position * base^(-2 i / rotary_dim):
      (y[a] cos - y[b] sin, y[b] cos + y[a] sin), with (a, b) = (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if `interleaved`

    Keys of length 1, as compute_gated_delta_rule expects them, have a weight of dim ** -0.5 in all places.  The angles are formed in
    float64, so positions of a million are turned as exactly as near ones (from some 10^9 on 2^-53 of an angle's turns is more than float32's
    rounding); the rest in float32, rounded once.
    Differentiable in q, k, q_weight and k_weight.

    Args:
        q:          [num_envs, seq_len, heads, dim] (or [num_envs, heads, dim]: one step), float32 or bfloat16, GPU; any strides
                    with a contiguous last axis (time-major views and slices of a joint projection are read in place).
        k:          the same with a number of heads of its own.  Dimensions of 1 to 256.
        q_weight, k_weight: [dim], float32, or None (ones).
        positions:  [num_envs, seq_len] (or [num_envs]), int64, for instance the steps since the episode began; None: nothing is rotated.
        base:       of the angles' frequencies.
        rotary_dim: how many elements are rotated, an even number (default: all; dim must then be even).
        eps:        added to the mean square.
        interleaved: which elements are pairs.

    Returns:
        q, k: contiguous, the dtype of q.
    """
    rotary_dim = _check(q, k, q_weight, k_weight, positions, base, rotary_dim, eps)
    q, k = _inner(q), _inner(k)
    q_weight, k_weight, positions = (None if t is None else t.contiguous() for t in (q_weight, k_weight, positions))
    settings = (float(base), rotary_dim, float(eps), bool(interleaved))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QueryKeyNorms.apply(q, k, q_weight, k_weight, positions, settings)
    return _forward(q, k, q_weight, k_weight, positions, settings)
