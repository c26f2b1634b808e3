"""Temperatures whose reciprocal float32 does not hold are refused: x / 1e-40 came out as 0 inf = NaN at the largest logit, and
x / 1e46 as -inf 0 = NaN at a logit of -inf."""
import ctypes

import pytest
import torch

import rl_triton.policy as policy
from rl_triton.policy import _native
from test_policy_api_cpu import _Gpu


@pytest.mark.parametrize("tau", [1e-40, 5e-324, 9e-39, 1.1e38, 1e46, 1e300])
def test_refused(tau, monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    rows = _native.ActionRows(4096, 4096, 2, 3, 5, 15, 5, tau, 0)  # (never dereferenced)
    assert _native.load().rlk_action_log_probs(ctypes.byref(rows), 4096, 4096, None, None) == -1
    x, a, t = _Gpu(2, 3, 4), _Gpu(2, 3, dtype=torch.int64), _Gpu(2, 3)
    with pytest.raises(AssertionError, match="temperature"):
        policy.compute_action_log_probs(x, a, tau)
    with pytest.raises(AssertionError, match="temperature"):
        policy.compute_policy_loss_from_logits(x, a, t, t, temperature=tau)
