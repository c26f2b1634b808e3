"""The scratch memory that the gated delta rule's C entries ask for: a forward pass that keeps its records for the one back has them once."""
import ctypes

import pytest

from rl_triton.policy import _native

FORWARD, BACKWARD, SAVED = 0, 1, 2
P = 4096  # never dereferenced


@pytest.mark.parametrize("shape", [(64, 1024, 8, 64, 64), (2100, 70, 50, 2, 2), (3, 1, 1, 128, 7)])
def test_records_are_kept_once(shape):
    lib = _native.load()
    assert lib.rlk_delta_rule_workspace_bytes(*shape, SAVED) == 0 < lib.rlk_delta_rule_workspace_bytes(*shape, FORWARD)
    assert lib.rlk_delta_rule_workspace_bytes(*shape, BACKWARD) > 0


def test_segments_have_theirs():
    """What segments need depends on the number of CUs, which a machine without a GPU does not say: none is less than 0."""
    lib = _native.load()
    shape = (1, 16384, 16, 128, 128)
    records = 16 * 256 * 11536
    assert lib.rlk_delta_rule_workspace_bytes(*shape, FORWARD) - lib.rlk_delta_rule_workspace_bytes(*shape, SAVED) == records


def test_a_workspace_that_is_too_small():
    lib = _native.load()
    seq = _native.Sequence(P, 0, 0, 0)
    call = _native.DeltaRule(q=seq, k=seq, v=seq, out=seq, num_envs=2, seq_len=100, heads=3, dim_k=8, dim_v=8, betas=P, scale=1.0)
    assert lib.rlk_gated_delta_rule(ctypes.byref(call), None, 0, None) == -2  # (no records)
    need = lib.rlk_delta_rule_saved_bytes(2, 100, 3, 8, 8)
    for p, n in ((P, need - 1), (P + 8, need)):
        assert lib.rlk_gated_delta_rule(ctypes.byref(call), p, n, None) == -2
