"""Gradients through rl_triton.policy's C++ nodes of torch's graph, which well-formed calls get, against those of the Python
functions, which serve every other: the same kernels on the same arrays, so the same bits."""
import pytest
import torch

import rl_triton.policy as policy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


def _sequences(dtype, seq_len=80, envs=3):
    g = torch.Generator(device="cuda").manual_seed(2)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v = n(envs, seq_len, 2, 24).to(dtype), n(envs, seq_len, 2, 24).to(dtype), n(envs, seq_len, 2, 40).to(dtype)
    return q, k, v, torch.tensor([0.9, 0.99], device="cuda"), (n(envs, seq_len) > 1).float(), n(envs, 2, 24, 40)


def _is_native(t):
    return "PythonFunction" not in type(t.grad_fn).__mro__[1].__name__ and "BackwardCFunction" not in [c.__name__ for c in type(t.grad_fn).__mro__]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("seq_len", [80, 700])  # (one segment and several)
def test_linear_attention(dtype, seq_len):
    q, k, v, decay, dones, state = _sequences(dtype, seq_len)
    for d, s, scale in ((None, None, None), (dones, state, 0.3), (dones[:, ::1].bool(), state, None),
                        (dones.t().contiguous().t(), None, 2)):
        for wanted in ((True, True, True, True), (False, True, False, False), (False, False, False, True)):
            if s is None and not any(wanted[:3]):
                continue
            results = []
            for fn in (policy.compute_linear_attention, policy.compute_linear_attention.__wrapped__):
                leaves = [t.clone().requires_grad_(w) if t is not None else None for t, w in zip((q, k, v, s), wanted)]
                out, last = fn(*leaves[:3], decay, d, leaves[3], scale)
                if fn is policy.compute_linear_attention:
                    assert _is_native(out) == (d is None or d.dtype is torch.float32)
                up, us = torch.randn_like(out, generator=None) * 0 + 0.7, torch.full_like(last, -0.3)
                ask = [t for t in leaves if t is not None and t.requires_grad]
                for outs, ups in (((out, last), (up, us)), ((out,), (up.transpose(2, 3).contiguous().transpose(2, 3),)), ((last,), (us,)),
                                  ((out,), (torch.ones((), device="cuda", dtype=dtype).expand_as(out),))):
                    results.append((fn, torch.autograd.grad(outs, ask, ups, retain_graph=True)))
                results.append((fn, (out.detach(), last.detach())))
            half = len(results) // 2
            for (_, a), (_, b) in zip(results[:half], results[half:]):
                assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_action_log_probs(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(6, 50, 19, generator=g, device="cuda").to(dtype)
    a = torch.randint(0, 19, (6, 50), generator=g, device="cuda")
    for logits, acts in ((x, a), (x.transpose(0, 1).contiguous().transpose(0, 1), a), (x[:, 3], a[:, 3].contiguous()), (x.reshape(300, 19), a.reshape(300))):
        gl, ge = torch.randn(acts.shape, generator=g, device="cuda"), torch.randn(acts.shape, generator=g, device="cuda")
        results = []
        for fn in (policy.compute_action_log_probs, policy.compute_action_log_probs.__wrapped__):
            leaf = logits.detach().requires_grad_()
            lp, ent = fn(leaf, acts, 0.7)
            for outs, ups in (((lp, ent), (gl, ge)), ((lp,), (gl,)), ((ent,), (ge,)), ((lp,), (gl[..., :1].expand_as(gl),))):
                results.append(torch.autograd.grad(outs, leaf, ups, retain_graph=True)[0])
            results += [lp.detach(), ent.detach()]
        half = len(results) // 2
        assert all(torch.equal(p, q) for p, q in zip(results[:half], results[half:]))


def test_what_graphs_ask_of_a_node():
    """Second derivatives are refused, changed inputs are seen, a freed graph says so, checkpoints run the call again."""
    q, k, v, decay, dones, state = _sequences(torch.float32)
    x, a = torch.randn(4, 5, 7, device="cuda", requires_grad=True), torch.zeros(4, 5, dtype=torch.int64, device="cuda")
    q.requires_grad_()
    for y, leaf in ((policy.compute_linear_attention(q, k, v, decay, dones, state)[0], q), (policy.compute_action_log_probs(x, a)[0], x)):
        grad, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
        assert grad.requires_grad
        with pytest.raises(RuntimeError, match="twice"):
            grad.sum().backward()
    out, _ = policy.compute_linear_attention(q, k, v, decay, dones, state)
    v.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    out, _ = policy.compute_linear_attention(q, k, v, decay, dones, state)
    out.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        out.sum().backward()
    from torch.utils.checkpoint import checkpoint
    want, = torch.autograd.grad(policy.compute_linear_attention(q, k, v, decay, dones, state)[0].square().sum(), q)
    y = checkpoint(lambda t: policy.compute_linear_attention(t, k, v, decay, dones, state)[0], q, use_reentrant=False)
    got, = torch.autograd.grad(y.square().sum(), q)
    assert torch.equal(got, want)
    with torch.no_grad():
        assert not policy.compute_linear_attention(q, k, v, decay)[0].requires_grad
    with torch.inference_mode():
        frozen = k.clone()
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        policy.compute_linear_attention(q, frozen, v, decay)


def test_another_stream():
    """A backward pass runs on the stream of its forward one."""
    q, k, v, decay, dones, state = _sequences(torch.bfloat16, 700)
    g = torch.randn(v.shape, device="cuda").to(v.dtype)
    want = None
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            leaves = [t.clone().requires_grad_() for t in (q, k, v, state)]
            out, last = policy.compute_linear_attention(*leaves[:3], decay, dones, leaves[3])
        torch.cuda.current_stream().wait_stream(stream)
        got = torch.autograd.grad((out, last), leaves, (g, torch.ones_like(last)))
        torch.cuda.synchronize()
        if want is not None:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        want = got


def test_in_a_captured_graph():
    """Forward and backward passes in a graph, replayed on new values between other work, against eager calls."""
    q, k, v, decay, dones, state = _sequences(torch.float32, 700, 1)
    leaves = [t.requires_grad_() for t in (q, k, v, state)]
    x, a = torch.randn(4, 50, 7, device="cuda", requires_grad=True), torch.zeros(4, 50, dtype=torch.int64, device="cuda")

    def call():
        out, last = policy.compute_linear_attention(*leaves[:3], decay, dones, leaves[3])
        lp, _ = policy.compute_action_log_probs(x, a)
        return torch.autograd.grad((out, last, lp), (*leaves, x), (torch.ones_like(out), torch.ones_like(last), torch.ones_like(lp)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (1, 2, 3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            for t in (*leaves, x):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(got, call()))
