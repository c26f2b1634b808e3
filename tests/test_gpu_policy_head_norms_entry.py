"""The C entry of the head norms' backward pass where there are no rows: gradients of weights that are zero."""
import ctypes

import pytest
import torch

from rl_triton.policy import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("empty", [dict(seq_len=0), dict(num_envs=0), dict(q_heads=0, k_heads=0)])
def test_weights_of_no_rows(empty, bf16):
    lib = _native.load()
    x = torch.ones(64, device="cuda")
    seq = _native.Sequence(x.data_ptr(), 0, 0, 0)
    call = _native.HeadNorms(**{**dict(q=seq, k=seq, q_out=seq, k_out=seq, num_envs=2, seq_len=3, q_heads=4, k_heads=2, dim=8, rotary_dim=8, base=1e4,
                                       eps=1e-6, bf16=bf16), **empty})
    grads = torch.full((2, 8), float("nan"), device="cuda")
    need = lib.rlk_head_norms_workspace_bytes(ctypes.byref(call))
    ws = torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.rlk_query_key_norms_backward(ctypes.byref(call), seq, seq, grads[0].data_ptr(), grads[1].data_ptr(), ws.data_ptr(), need, stream) == 0
    assert not bool(grads.any())
    grads.fill_(1.0)
    assert lib.rlk_query_key_norms_backward(ctypes.byref(call), seq, seq, None, grads[1].data_ptr(), ws.data_ptr(), need, stream) == 0
    assert bool((grads[0] == 1.0).all()) and not bool(grads[1].any()) and bool((x == 1.0).all())
