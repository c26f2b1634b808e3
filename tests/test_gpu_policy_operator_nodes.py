"""The head norms, the gated delta rule and the sampling of actions through C++ (which well-formed calls get) and through the Python functions
(which serve every other): the same kernels on the same arrays, so the same bits.  And a run of them together, as a policy uses them."""
import pytest
import torch

import rl_triton.policy as policy
from _delta_reference import inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


def _is_native(t):
    return "BackwardCFunction" not in [c.__name__ for c in type(t.grad_fn).__mro__]


def _both(fn, args, kwargs, wanted):
    """Results and gradients of both paths, for the arguments `wanted`."""
    results = []
    for f in (fn, fn.__wrapped__):
        xs = [t.detach().clone().requires_grad_(i in wanted) if isinstance(t, torch.Tensor) and t.is_floating_point() else t for i, t in enumerate(args)]
        outs = f(*xs, **kwargs)
        got = [o.detach() for o in outs]
        if wanted:
            assert _is_native(outs[0]) == (f is fn)
            ups = [torch.full_like(o, 0.5 + i) for i, o in enumerate(outs)]
            for use in ((0, 1), (0,), (1,)):
                got += [g for g in torch.autograd.grad([outs[i] for i in use], [xs[i] for i in wanted], [ups[i] for i in use], retain_graph=True, allow_unused=True)
                        if g is not None]
            strided = torch.full(outs[0].transpose(0, 1).shape, 0.25, device="cuda", dtype=outs[0].dtype).transpose(0, 1)
            got += [g for g in torch.autograd.grad(outs[0], [xs[i] for i in wanted], strided, allow_unused=True) if g is not None]
        results.append(got)
    a, b = results
    assert len(a) == len(b) and all(p.dtype == q.dtype and torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_delta_rule(dtype):
    for T in (70, 2100):
        q, k, v, g, beta, dones, state = (t.cuda() for t in inputs(2, T, 2, 24, 40, dtype, T))
        for args in ((q, k, v, g, beta, dones, state, 0.3), (q, k, v, None, beta), (q, k, v, g, beta, None, None, None)):
            both = [i for i in (0, 1, 2, 3, 4, 6) if i < len(args) and args[i] is not None]
            for wanted in ([], both, [2], [4], [0, 1]):
                _both(policy.compute_gated_delta_rule, args, {}, wanted)
    step = [t[:, 0] for t in (q, k, v, g, beta)]
    _both(policy.compute_gated_delta_rule_step, (*step, state, dones[:, 0], 0.5), {}, [])
    out, _ = policy.compute_gated_delta_rule_step(step[0].detach().requires_grad_(), *step[1:], state)
    with pytest.raises(RuntimeError, match="no gradient"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_norms(dtype):
    q, k = torch.randn(3, 40, 4, 24, device="cuda").to(dtype), torch.randn(3, 40, 2, 24, device="cuda").to(dtype)
    w = torch.rand(24, device="cuda")
    pos = torch.arange(120, device="cuda").view(3, 40)
    for args, kw in (((q, k, w, w + 1, pos), {}), ((q, k, None, w, pos), dict(rotary_dim=12, interleaved=True)), ((q, k, w), dict(eps=0.1)),
                     ((q[:, 0], k[:, 0], None, None, pos[:, 0].contiguous()), dict(base=100))):
        floats = [i for i, t in enumerate(args) if t is not None and t.is_floating_point()]
        for wanted in ([], floats, [0], [1], [floats[-1]]):
            _both(policy.compute_query_key_norms, args, kw, wanted)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampling(dtype):
    for shape in ((6, 5, 18), (7, 300), (2, 5000)):
        x, u = torch.randn(shape, device="cuda").to(dtype), torch.rand(shape[:-1], device="cuda")
        for kw in ({}, dict(top_k=5), dict(top_p=0.5, min_p=0.01), dict(temperature=2, top_k=10 ** 30), dict(top_p=1, min_p=0)):
            _both(policy.compute_sampled_actions, (x, u), kw, [])


def test_bad_calls_are_refused_by_both():
    x, u = torch.randn(4, 9, device="cuda"), torch.rand(4, device="cuda")
    for kw in (dict(top_k=0), dict(top_k=-(10 ** 30)), dict(top_p=0.0), dict(top_p=float("nan")), dict(min_p=1.1), dict(temperature=0), dict(top_k=True)):
        with pytest.raises(AssertionError):
            policy.compute_sampled_actions(x, u, **kw)
    q = torch.randn(2, 3, 2, 8, device="cuda")
    for kw in (dict(rotary_dim=3, positions=torch.zeros(2, 3, dtype=torch.int64, device="cuda")), dict(eps=-1.0), dict(base=0.0), dict(rotary_dim=10 ** 30)):
        with pytest.raises(AssertionError):
            policy.compute_query_key_norms(q, q, **kw)
    with pytest.raises(AssertionError):
        policy.compute_gated_delta_rule(q, q, q, None, torch.ones(2, 3, device="cuda"))
    with pytest.raises(AssertionError):
        policy.compute_gated_delta_rule(q, q, q, None, torch.ones(2, 3, 2, device="cuda"), scale=float("inf"))


def test_what_graphs_ask_of_a_node():
    """Second derivatives are refused, changed inputs are seen, a freed graph says so, checkpoints run the call again."""
    q, k, v, g, beta, dones, state = (t.cuda() for t in inputs(2, 40, 2, 16, 8, torch.float32, 3))
    q.requires_grad_()
    w = torch.ones(16, device="cuda", requires_grad=True)
    for call, leaf in ((lambda: policy.compute_gated_delta_rule(q, k, v, g, beta, dones, state)[0], q), (lambda: policy.compute_query_key_norms(q, k, w)[0], w)):
        grad, = torch.autograd.grad(call().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            grad.sum().backward()
        y = call()
        y.sum().backward()
        with pytest.raises(RuntimeError, match="second time"):
            y.sum().backward()
        y = call()
        k.add_(0.0)
        if leaf is q:
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                y.sum().backward()
        want, = torch.autograd.grad(call().sum(), leaf)
        got, = torch.autograd.grad(torch.utils.checkpoint.checkpoint(lambda x: call(), leaf, use_reentrant=False).sum(), leaf)
        assert torch.equal(got, want)


def test_a_policy_step_by_step_and_over_the_window():
    """Projections, normed and rotated heads, the memory, logits, a sampled action: played step by step it is what the learner computes over
    the window, and its loss's gradient reaches every weight."""
    E, T, H, d, A = 6, 90, 3, 32, 11
    torch.manual_seed(4)
    qkv, gates, head = torch.nn.Linear(20, 3 * H * d).cuda(), torch.nn.Linear(20, 2 * H).cuda(), torch.nn.Linear(H * d, A).cuda()
    w_q, w_k = (torch.full((d,), d ** -0.5, device="cuda", requires_grad=True) for _ in range(2))
    obs = torch.randn(E, T, 20, device="cuda")
    dones = (torch.rand(E, T, device="cuda") < 0.05).float()
    u = torch.rand(E, T, device="cuda")
    # steps since the episode began: an inclusive count of steps, which episode ends set back
    positions = (rlt().compute_episodic_prefix_sum(torch.ones(E, T, device="cuda"), dones) - 1).long()

    def parts(x, pos):
        q, k, v = qkv(x).unflatten(-1, (3 * H, d)).chunk(3, -2)
        q, k = policy.compute_query_key_norms(q, k, w_q, w_k, pos)
        a, b = gates(x).chunk(2, -1)
        return q, k, v, -torch.nn.functional.softplus(a).contiguous() * 0.1, b.sigmoid().contiguous()

    with torch.no_grad():
        state, acts, lps = torch.zeros(E, H, d, d, device="cuda"), [], []
        for t in range(T):
            q, k, v, g, b = parts(obs[:, t], positions[:, t].contiguous())
            cut = dones[:, t - 1] if t else None
            o, state = policy.compute_gated_delta_rule_step(q, k, v, g, b, state, cut, 1.0)
            a, lp = policy.compute_sampled_actions(head(o.flatten(1)), u[:, t].contiguous(), 0.9, top_k=8, top_p=0.95)
            acts.append(a), lps.append(lp)
        acts = torch.stack(acts, 1)
    out, last = policy.compute_gated_delta_rule(*parts(obs, positions), dones, None, 1.0)
    logits = head(out.flatten(2))
    again, again_lp = policy.compute_sampled_actions(logits, u, 0.9, top_k=8, top_p=0.95)
    # (logits of both ways differ by some 1e-6: a uniform number lies that near to one of its row's borders once in some ten thousand rows)
    assert float((again == acts).float().mean()) > 0.995
    assert torch.allclose(last, state * (dones[:, -1] == 0)[:, None, None, None], rtol=0, atol=1e-5 * float(state.abs().max()))
    same = again == acts
    assert torch.allclose(again_lp[same], torch.stack(lps, 1)[same], rtol=0, atol=1e-4)
    old, _ = policy.compute_action_log_probs(logits.detach(), acts, 0.9)
    loss, grad, _ = policy.compute_policy_loss_from_logits(logits, acts, old, torch.randn(E, T, device="cuda"), temperature=0.9)
    logits.backward(grad)
    for p in (*qkv.parameters(), *gates.parameters(), *head.parameters(), w_q, w_k):
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and bool(p.grad.any())


def rlt():
    import rl_triton
    return rl_triton


def test_two_threads_at_once():
    """Calls of two threads on streams of their own, forward and back: the results of calls one after the other."""
    import threading
    sets = [tuple(t.cuda() for t in inputs(2, 300, 2, 32, 32, torch.bfloat16, seed)) for seed in (1, 2)]

    def run(x):
        leaves = [t.detach().requires_grad_(i != 5) for i, t in enumerate(x)]
        q, k = policy.compute_query_key_norms(leaves[0], leaves[1])
        out, last = policy.compute_gated_delta_rule(q, k * 0.1, *leaves[2:])
        a, lp = policy.compute_sampled_actions(out.detach().flatten(2), torch.full(out.shape[:2], 0.5, device="cuda"), top_p=0.9)
        return (out.detach(), last.detach(), a, lp, *torch.autograd.grad((out, last), [t for i, t in enumerate(leaves) if i != 5],
                                                                          (torch.ones_like(out), torch.ones_like(last))))

    want = [run(x) for x in sets]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = run(sets[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_calls_keep_nothing():
    """What a call allocates and does not return is free when it is over, and so is what it returns when the caller lets go; calls without a
    gradient are C++'s to the end."""
    import gc
    from rl_triton._native import fast
    q, k, v, g, beta, dones, state = (t.cuda() for t in inputs(2, 300, 2, 24, 40, torch.float32, 1))
    w = torch.ones(24, device="cuda")
    leaf = q.clone().requires_grad_()
    step = [t[:, 0].contiguous() for t in (q, k, v, g, beta)]
    x, u = torch.randn(9, 700, device="cuda"), torch.rand(9, device="cuda")
    calls = [(4, lambda: policy.compute_gated_delta_rule(q, k, v, g, beta, dones, state)),
             (0, lambda: policy.compute_gated_delta_rule(leaf, k, v, g, beta)),
             (0, lambda: torch.autograd.grad(policy.compute_gated_delta_rule(leaf, k, v, g, beta)[0].sum(), leaf)),
             (4, lambda: policy.compute_gated_delta_rule_step(*step, state)), (4, lambda: policy.compute_query_key_norms(q, k, w, w)),
             (0, lambda: torch.autograd.grad(policy.compute_query_key_norms(leaf, k, w, w)[0].sum(), leaf)),
             (4, lambda: policy.compute_sampled_actions(x, u, top_k=5, top_p=0.9))]
    for launches, call in calls:
        call()
        torch.cuda.synchronize()
        gc.collect()
        before, taken = torch.cuda.memory_allocated(), fast.launched()
        gc.disable()
        for _ in range(4):
            call()
        torch.cuda.synchronize()
        gc.enable()
        assert torch.cuda.memory_allocated() == before
        assert fast.launched() - taken == launches


def test_offsets_past_32_bits():
    """Views whose environments or steps lie 2^31 elements and more apart: the bits of contiguous copies."""
    big = torch.empty((1 << 33) + (1 << 16), dtype=torch.bfloat16, device="cuda")  # 17 GB, of which a few rows are written
    q, k, v, g, beta, dones, state = (t.cuda() for t in inputs(3, 5, 2, 16, 16, torch.bfloat16, 5))

    def spread(x, env, step):
        y = big.as_strided(x.shape, (env, step, 16, 1))
        return y.copy_(x)

    for env, step in ((1 << 32, 64), (128, 1 << 31)):
        for slot in range(3):  # (one array at a time lies in the buffer)
            xs = [t.clone() for t in (q, k, v)]
            near = [t.clone().requires_grad_() for t in (q, k, v)]
            xs[slot] = spread(xs[slot], env, step)
            far = [t.detach().requires_grad_() for t in xs]
            outs = []
            for x in (far, near):
                y, last = policy.compute_gated_delta_rule(*x, g, beta, dones, state)
                outs.append((y, last, *torch.autograd.grad(y, x, torch.ones_like(y))))
            assert all(torch.equal(a, b) for a, b in zip(*outs))
        up = spread(torch.randn(q.shape, device="cuda").bfloat16(), env, step)
        y, _ = policy.compute_gated_delta_rule(*near, g, beta, dones, state)
        y2, _ = policy.compute_gated_delta_rule(*near, g, beta, dones, state)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, near, up), torch.autograd.grad(y2, near, up.clone())))
    for actions in (20, 5000):
        x = big.as_strided((2, 2, actions), ((1 << 32) - 8, 1 << 31, 1))
        x.copy_(torch.randn(x.shape, device="cuda"))
        u = torch.rand(2, 2, device="cuda")
        for kw in ({}, dict(top_k=9), dict(top_p=0.7)):
            assert all(torch.equal(a, b) for a, b in zip(policy.compute_sampled_actions(x, u, **kw), policy.compute_sampled_actions(x.clone(), u, **kw)))
