"""compute_query_key_norms where queries or keys have no heads: the other side is what it is with both (bit by bit), in steps and in sequences."""
import pytest
import torch

import rl_triton.policy as policy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead", [(5,), (700,), (5, 9)])
@pytest.mark.parametrize("side", [0, 1])
def test_one_side_has_no_heads(side, lead, dtype):
    g = torch.Generator(device="cuda").manual_seed(7)
    both = [torch.randn(*lead, h, 24, generator=g, device="cuda").to(dtype).requires_grad_() for h in (2, 3)]
    weights = [(1 + torch.randn(24, generator=g, device="cuda")).requires_grad_() for _ in range(2)]
    ups = [torch.randn(x.shape, generator=g, device="cuda").to(dtype) for x in both]
    pos = torch.randint(0, 1000, lead, generator=g, device="cuda")
    outs = policy.compute_query_key_norms(*both, *weights, pos)
    grads = torch.autograd.grad(outs, (*both, *weights), ups)

    alone = [t.detach().requires_grad_() if i == side else t.detach()[..., :0, :].requires_grad_() for i, t in enumerate(both)]
    got = policy.compute_query_key_norms(*alone, *weights, pos)
    assert torch.equal(got[side], outs[side]) and got[1 - side].shape == (*lead, 0, 24)
    with torch.no_grad():
        assert torch.equal(policy.compute_query_key_norms(*alone, *weights, pos)[side], outs[side])
    back = torch.autograd.grad(got, (*alone, *weights), [u if i == side else u[..., :0, :] for i, u in enumerate(ups)])
    assert torch.equal(back[side], grads[side]) and back[1 - side].shape == alone[1 - side].shape
    # (the weights' sums are over other numbers of workgroups: float32's rounding of sums over the rows)
    rows = both[side].numel() // 24
    size = float(rows) * float(ups[side].float().abs().max()) * 24 ** 0.5
    assert float((back[2 + side] - grads[2 + side]).abs().max()) <= rows ** 0.5 * 2.0 ** -24 * size
    assert not bool(back[3 - side].any())
