"""The C entry of the head norms' backward pass on empty inputs: RLK_OK, as of the other entries, and no launch where no sum is asked for."""
import ctypes

import pytest

from rl_triton.policy import _native

P = 4096  # never dereferenced
SEQ, NONE = _native.Sequence(P, 0, 0, 0), _native.Sequence(None, 0, 0, 0)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("empty", [dict(seq_len=0), dict(num_envs=0), dict(num_envs=0, seq_len=0), dict(q_heads=0, k_heads=0), dict(seq_len=0, q_heads=0)])
def test_backward_of_nothing(empty, bf16):
    lib = _native.load()
    call = _native.HeadNorms(**{**dict(q=SEQ, k=SEQ, q_out=SEQ, k_out=SEQ, num_envs=2, seq_len=3, q_heads=4, k_heads=2, dim=8, rotary_dim=8, positions=P,
                                       base=1e4, eps=1e-6, bf16=bf16), **empty})
    assert lib.rlk_query_key_norms(ctypes.byref(call), None) == 0
    for grads in ((SEQ, SEQ), (SEQ, NONE), (NONE, NONE)):
        assert lib.rlk_query_key_norms_backward(ctypes.byref(call), *grads, None, None, None, 0, None) == 0
    # weights' gradients are sums over the rows: they are written, and their workspace is asked for
    assert lib.rlk_query_key_norms_backward(ctypes.byref(call), SEQ, SEQ, P, P, None, 0, None) == -2
