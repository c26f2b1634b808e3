"""compute_gated_delta_rule and compute_gated_delta_rule_step against the float64 recurrence (tests/_delta_reference.py)."""
import math

import pytest
import torch

import rl_triton.policy as policy
from _delta_reference import U16, held, held_rounded, inputs, relative, rule

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")

DTYPES = [torch.float32, torch.bfloat16]


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _hold(got, want, dtype, T, dim, what):
    (held if dtype == torch.float32 else held_rounded)(got, want, relative(T, dim), what)


SHAPES = [(1, 1, 1, 1, 1), (2, 2, 2, 3, 5), (3, 63, 2, 16, 16), (2, 64, 3, 16, 40), (2, 65, 5, 64, 64), (3, 127, 2, 72, 24), (1, 130, 2, 128, 128),
          (2, 333, 4, 40, 72), (1, 700, 1, 100, 100), (1, 1025, 1, 128, 128), (300, 5, 1, 33, 1), (2, 129, 1, 7, 120)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_sequences(shape, dtype):
    E, T, H, dk, dv = shape
    for ends, state, gates, scale in ((None, False, False, None), (0.03, True, True, 0.3), (0.5, True, True, -1.0)):
        x = inputs(*shape, dtype, T + dk, ends, state, gates)
        out, last = policy.compute_gated_delta_rule(*_cuda(*x), scale)
        want, wlast = rule(*x, dk ** -0.5 if scale is None else scale)
        assert out.dtype == dtype and last.dtype == torch.float32 and out.is_contiguous()
        _hold(out, want, dtype, T, dk, "out")
        held(last, wlast, relative(T, dk), "state")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(shape, dtype):
    E, T, H, dk, dv = shape
    names = ("q", "k", "v", "log_decays", "betas", "state")
    for ends, state, gates in ((0.03, True, True), (None, False, False), (None, False, True)):
        x = inputs(*shape, dtype, 2 * T + dk, ends, state, gates)
        g = torch.Generator().manual_seed(T)
        go, gs = torch.randn(E, T, H, dv, generator=g).to(dtype), torch.randn(E, H, dk, dv, generator=g)
        d = _cuda(*x)
        for i in (0, 1, 2, 3, 4, 6):
            if d[i] is not None:
                d[i].requires_grad_()
        out, last = policy.compute_gated_delta_rule(*d, 0.7)
        leaves = {n: t for n, t in zip(names, (*d[:5], d[6])) if t is not None}
        for use_out, use_last in ((True, True), (True, False), (False, True)):
            outs, ups = zip(*([(out, go)] * use_out + [(last, gs)] * use_last))
            got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), _cuda(*ups), retain_graph=True)))
            want = dict(zip(names, rule(*x, 0.7, go if use_out else None, gs if use_last else None)[2]))
            # the terms that a gate's gradient is the difference of
            size = float((x[0].double() * want["q"]).norm() + (x[1].double() * want["k"]).norm())
            for n in leaves:
                assert got[n].dtype == leaves[n].dtype
                if n in "qkv":
                    _hold(got[n], want[n], dtype, T, dk, n)
                else:
                    held(got[n], want[n], relative(T, dk), n, size if n == "log_decays" else 0.0)


def test_gradients_against_differences():
    """Directional differences of the float64 recurrence, h = 1e-4: the third derivative leaves h^2 of a size of some units."""
    x = inputs(2, 150, 2, 20, 12, torch.float32, 5)
    x = [t if i != 3 else t.clamp_min(-3.0) for i, t in enumerate(x)]
    g = torch.Generator().manual_seed(6)
    go, gs = torch.randn(2, 150, 2, 12, generator=g), torch.randn(2, 2, 20, 12, generator=g)
    d = _cuda(*x)
    at = (0, 1, 2, 3, 4, 6)
    for i in at:
        d[i].requires_grad_()
    grads = torch.autograd.grad(policy.compute_gated_delta_rule(*d, 0.7), [d[i] for i in at], _cuda(go, gs))
    for i, grad in zip(at, grads):
        step = torch.randn(x[i].shape, generator=g).double()
        values = []
        for sign in (1, -1):
            y = [t.double() if j in at else t for j, t in enumerate(x)]
            y[i] = y[i] + sign * 1e-4 * step
            out, last = rule(*y, 0.7)
            values.append(float((out * go).sum() + (last * gs).sum()))
        prod = grad.cpu().double() * step
        assert abs((values[0] - values[1]) / 2e-4 - float(prod.sum())) < 1e-4 * float(prod.abs().sum())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 2500, 2, 40, 64), (2, 2049, 1, 128, 100), (1, 4100, 3, 16, 24)])
def test_long_sequences_of_few_heads(shape, dtype):
    """Sequences that are cut into segments, with and without episode ends in them, and the same with gradients."""
    E, T, H, dk, dv = shape
    for ends, state in ((None, True), (0.002, True), (0.02, False)):
        x = inputs(*shape, dtype, T + dv, ends, state)
        d = _cuda(*x)
        out, last = policy.compute_gated_delta_rule(*d, 0.7)
        g = torch.Generator().manual_seed(T)
        go, gs = torch.randn(E, T, H, dv, generator=g).to(dtype), torch.randn(E, H, dk, dv, generator=g)
        want, wlast, grads = rule(*x, 0.7, go, gs)
        _hold(out, want, dtype, T, dk, "out")
        held(last, wlast, relative(T, dk), "state")
        leaves = [d[i].requires_grad_() for i in (0, 1, 2, 3, 4, 6) if d[i] is not None]
        again, again_last = policy.compute_gated_delta_rule(*d, 0.7)
        assert torch.equal(again, out) and torch.equal(again_last, last)
        got = torch.autograd.grad((again, again_last), leaves, _cuda(go, gs))
        size = float((x[0].double() * grads[0]).norm() + (x[1].double() * grads[1]).norm())
        for i, (a, b) in enumerate(zip(got, grads)):
            if i < 3:
                _hold(a, b, dtype, T, dk, i)
            else:
                held(a, b, relative(T, dk), i, size if i == 3 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_numbers_in_long_sequences(dtype):
    """A head with a NaN, and one whose state grows out of float32 though none is there at first, are walked without segments; the others as before."""
    shape = (1, 2600, 4, 24, 32)
    x = list(inputs(*shape, dtype, 21, None, False, gates=False))
    x[5] = torch.zeros(1, 2600)
    x[5][:, 1400] = x[5][:, 2000] = 1.0
    clean = policy.compute_gated_delta_rule(*_cuda(*x), 1.0)
    x[2][0, 1700, 1, 3] = math.nan
    x[1][0, 1401:2001, 2] *= 20.0
    x[2][0, :2001, 2] = 0.0  # (nothing is written before)
    out, last = policy.compute_gated_delta_rule(*_cuda(*x), 1.0)
    want, wlast = rule(*x, 1.0)
    for h in (0, 3):
        assert torch.equal(out[:, :, h], clean[0][:, :, h]) and torch.equal(last[:, h], clean[1][:, h])
    _hold(out[:, :1700, 1], want[:, :1700, 1], dtype, 2600, 24, "before")
    _hold(out[:, 2001:, 1], want[:, 2001:, 1], dtype, 2600, 24, "after")
    _hold(out[:, :, 2], want[:, :, 2], dtype, 2600, 24, "a state of zeros stays one")
    held(last, wlast, relative(2600, 24))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Time-major views, slices of a joint projection, misaligned and element-strided tensors, shared heads: the same bits."""
    x = inputs(3, 90, 4, 32, 32, dtype, 3)
    dev = _cuda(*x)
    want = policy.compute_gated_delta_rule(*dev)
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in dev[:5]]
    joint = torch.cat(dev[:3], -1)
    slices = [joint[..., 32 * i:32 * i + 32] for i in range(3)] + dev[3:5]
    strided = [torch.stack([t, t], -1)[..., 0] for t in dev[:5]]
    odd = []
    for t in dev[:3]:
        buf = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        odd.append(buf[1:].view(t.shape))
    for views in (major, slices, strided, odd + dev[3:5]):
        got = policy.compute_gated_delta_rule(*views, *dev[5:])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for flags in (dev[5].bool(), dev[5].bfloat16(), dev[5].t().contiguous().t()):
        got = policy.compute_gated_delta_rule(*dev[:5], flags, dev[6])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    k1, v1 = (t[:, :, :1].contiguous().requires_grad_() for t in dev[1:3])
    kf, vf = (t.detach().expand(-1, -1, 4, -1).contiguous().requires_grad_() for t in (k1, v1))
    shared = policy.compute_gated_delta_rule(dev[0], k1.expand(-1, -1, 4, -1), v1.expand(-1, -1, 4, -1), *dev[3:])
    full = policy.compute_gated_delta_rule(dev[0], kf, vf, *dev[3:])
    assert torch.equal(shared[0], full[0])
    up = torch.randn(full[0].shape, device="cuda").to(dtype)
    for a, b in zip(torch.autograd.grad(shared[0], (k1, v1), up), torch.autograd.grad(full[0], (kf, vf), up)):
        assert torch.allclose(a.float(), b.float().sum(2, keepdim=True), rtol=4 * U16, atol=1e-3 if dtype == torch.float32 else 0.1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_upstream_layouts(dtype):
    """Gradients that come expanded, transposed or for one of the outputs only are those of contiguous ones."""
    x = _cuda(*inputs(2, 70, 2, 24, 16, dtype, 4))
    leaves = [x[i].requires_grad_() for i in (0, 1, 2, 3, 4, 6)]
    out, last = policy.compute_gated_delta_rule(*x)
    one = torch.full((), 0.5, dtype=dtype, device="cuda").expand_as(out)
    for up in (one, torch.randn(2, 2, 70, 16, device="cuda").to(dtype).transpose(1, 2)):
        a = torch.autograd.grad(out, leaves, up, retain_graph=True)
        b = torch.autograd.grad(out, leaves, up.contiguous(), retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    for i in range(len(leaves)):  # one at a time
        a, = torch.autograd.grad(out, leaves[i], one, retain_graph=True)
        assert torch.equal(a, torch.autograd.grad(out, leaves, one, retain_graph=True)[i])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dims", [(1, 1), (16, 24), (64, 64), (33, 128), (128, 40), (100, 7), (128, 128)])
def test_steps(dims, dtype):
    """Step by step is the sequence; the state goes on in place as in a new tensor."""
    E, T, H = 5, 6, 3
    x = inputs(E, T, H, *dims, dtype, dims[0], 0.3)
    q, k, v, g, beta, dones, state = _cuda(*x)
    want, wlast = rule(*x[:5], x[5], x[6], 0.7)
    place, new = state.clone(), state
    for t in range(T):
        cut = dones[:, t - 1].contiguous() if t else None
        o, new = policy.compute_gated_delta_rule_step(q[:, t], k[:, t], v[:, t], g[:, t].contiguous(), beta[:, t], new, cut, 0.7)
        p, back = policy.compute_gated_delta_rule_step(q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t], place, cut, 0.7, out_state=place)
        assert back is place and torch.equal(o, p) and torch.equal(new, place)
        _hold(o, want[:, t], dtype, T, dims[0], t)
    held(new * (dones[:, -1] == 0)[:, None, None, None], wlast, relative(T, dims[0]))
    o, s = policy.compute_gated_delta_rule_step(q[:, 0], k[:, 0], v[:, 0], None, beta[:, 0], state)
    p, r = policy.compute_gated_delta_rule_step(q[:, 0], k[:, 0], v[:, 0], torch.zeros_like(g[:, 0]), beta[:, 0], state, torch.zeros(E, device="cuda"))
    assert torch.equal(o, p) and torch.equal(s, r)


def test_step_refuses_a_backward_pass():
    x = _cuda(*inputs(2, 1, 2, 8, 8, torch.float32, 1, None))
    q, k, v, g, beta = (t[:, 0] for t in x[:5])
    out, state = policy.compute_gated_delta_rule_step(q.requires_grad_(), k, v, g, beta, x[6])
    assert out.requires_grad and not state.requires_grad
    with pytest.raises(RuntimeError, match="no gradient"):
        out.sum().backward()
    with pytest.raises(RuntimeError, match="requires a gradient"):
        policy.compute_gated_delta_rule_step(q, k, v, g, beta, x[6], out_state=x[6].clone().requires_grad_())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v", "log_decays", "betas"])
@pytest.mark.parametrize("value", [math.nan, math.inf, 3e38])
def test_what_is_not_finite_stays_in_its_episode(which, value, dtype):
    """A bad number in one step: steps before it and other episodes are what they are without it, forward and back."""
    E, T, H, d = 2, 200, 2, 40
    x = list(inputs(E, T, H, d, d, dtype, 9, None))
    x[3] = x[3].clamp_min(-5.0)
    dones = torch.zeros(E, T)
    dones[:, 70] = dones[:, 131] = 1.0  # (in chunks of 64: 71 .. 131 is one episode)
    x[5] = dones
    up = torch.randn(E, T, H, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    bad = [None if t is None else t.clone() for t in x]
    i = ("q", "k", "v", "log_decays", "betas").index(which)
    for at in (100, 127, 128):
        bad[i][:, at] = value
        results = []
        for y in (x, bad):
            dev = _cuda(*y)
            leaves = [dev[j].requires_grad_() for j in (0, 1, 2, 3, 4, 6)]
            out, last = policy.compute_gated_delta_rule(*dev, 0.7)
            results.append((out.detach(), last.detach(), torch.autograd.grad(out, leaves, up.cuda())))
        (a, la, ga), (b, lb, gb) = results
        tol = dict(rtol=4 * U16 if dtype == torch.bfloat16 else 0, atol=relative(T, d) * 8)
        for lo, hi in ((0, at), (132, T)):
            assert torch.allclose(a[:, lo:hi].float(), b[:, lo:hi].float(), **tol)
        assert torch.allclose(la, lb, rtol=0, atol=relative(T, d) * 8 * float(la.abs().max()))
        for p, q in zip(ga[:5], gb[:5]):
            for lo, hi in ((0, 71), (132, T)):
                assert torch.allclose(p[:, lo:hi].float(), q[:, lo:hi].float(), rtol=tol["rtol"], atol=tol["atol"] * 8 * float(p.abs().max()))
        assert torch.allclose(ga[5], gb[5], rtol=0, atol=tol["atol"] * 8 * float(ga[5].abs().max()))
        bad[i][:, at] = x[i][:, at]


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_state_that_is_not_finite_ends_with_its_episode(dtype):
    x = list(inputs(2, 140, 2, 24, 24, dtype, 11, None))
    x[5] = torch.zeros(2, 140)
    x[5][:, 80] = 1.0
    x[3] = x[3].clamp_min(-5.0)
    want, wlast = rule(*x, 24 ** -0.5)
    x[6][0, 0, 3, 5] = math.nan
    x[6][1, 1, 2, 7] = math.inf
    out, last = policy.compute_gated_delta_rule(*_cuda(*x))
    # (its chunk went step by step, which rounds otherwise: held to the definition as any result)
    held(last, wlast, relative(140, 24))
    _hold(out[:, 81:], want[:, 81:], dtype, 140, 24, "the episode after")
    assert bool(torch.isnan(out[0, 0, 0, 5]))
    _hold(out[0, :, 0, :5], want[0, :, 0, :5], dtype, 140, 24, "other columns")
    x[3][:, 0] = -math.inf  # nothing of it stays
    x[6] = torch.full_like(x[6], math.nan)
    out, last = policy.compute_gated_delta_rule(*_cuda(*x))
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(last).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [4.0, 40.0])
def test_growing_states(length, dtype):
    """Keys that are too long make a state grow, at 40 times out of float32 within some steps: of that episode alone."""
    x = list(inputs(1, 128, 1, 16, 16, dtype, 12, None, length=length))
    x[4][:] = 1.0
    x[3] = None
    x[5] = torch.zeros(1, 128)
    x[5][:, [50, 100]] = 1.0
    x[1][:, 51:101] /= length
    out, _ = policy.compute_gated_delta_rule(*_cuda(*x), 1.0)
    want, _ = rule(*x, 1.0)
    if length == 40.0:
        assert not bool(torch.isfinite(out[:, 101:]).all())
    assert bool(torch.isfinite(out[:, 51:101]).all())
    _hold(out[:, 51:101], want[:, 51:101], dtype, 50, 16, "the episode between")


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_keys(dtype):
    """Every step has the same key: each write replaces the last one, and the triangular systems are full of ones."""
    x = list(inputs(1, 150, 1, 32, 32, dtype, 13, None, gates=False))
    x[1] = x[1][:, :1].expand_as(x[1]).contiguous()
    x[4][:] = 1.0
    out, last = policy.compute_gated_delta_rule(*_cuda(*x), 1.0)
    want, wlast = rule(*x, 1.0)
    _hold(out, want, dtype, 150, 32, "out")
    held(last, wlast, relative(150, 32))


def test_no_steps_and_no_environments():
    for shape in ((3, 0, 2, 8, 4), (0, 5, 2, 8, 4), (2, 5, 0, 8, 4)):
        q, k, v, g, beta, dones, state = (None if t is None else t.cuda().requires_grad_(i in (0, 6)) for i, t in enumerate((
            torch.zeros(shape[0], shape[1], shape[2], 8), torch.zeros(shape[0], shape[1], shape[2], 8), torch.zeros(shape[0], shape[1], shape[2], 4),
            torch.zeros(shape[:3]), torch.zeros(shape[:3]), torch.zeros(shape[:2]), torch.ones(shape[0], shape[2], 8, 4))))
        out, last = policy.compute_gated_delta_rule(q, k, v, g, beta, dones, state)
        assert out.shape == (*shape[:3], 4) and torch.equal(last, state)
        a, b = torch.autograd.grad((out, last), (q, state), (torch.ones_like(out), torch.full_like(last, 2.0)))
        assert a.shape == q.shape and bool((b == 2.0).all())


def test_repeats_are_bitwise_equal():
    x = _cuda(*inputs(3, 300, 2, 64, 64, torch.bfloat16, 15))
    leaves = [x[i].requires_grad_() for i in (0, 1, 2, 3, 4, 6)]
    runs = []
    for _ in range(3):
        out, last = policy.compute_gated_delta_rule(*x)
        runs.append((out.detach(), last.detach(), *torch.autograd.grad((out, last), leaves, (torch.ones_like(out), torch.ones_like(last)))))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_other_streams_and_graphs():
    """On another stream; captured with its backward pass and replayed on new inputs, with eager calls between."""
    x = [t.detach() for t in _cuda(*inputs(2, 200, 2, 64, 48, torch.bfloat16, 16))]
    up = torch.randn(2, 200, 2, 48, device="cuda").bfloat16()

    def run(xs):
        leaves = [t.detach().requires_grad_(i != 5) for i, t in enumerate(xs)]
        out, last = policy.compute_gated_delta_rule(*leaves)
        return (out.detach(), last.detach(), *torch.autograd.grad(out, [t for i, t in enumerate(leaves) if i != 5], up))

    want = run(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = [t.clone() for t in x]
    with torch.cuda.stream(side):
        run(static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(static)
    for seed in (16, 17, 18):
        fresh = [t.detach() for t in _cuda(*inputs(2, 200, 2, 64, 48, torch.bfloat16, seed))]
        for a, b in zip(static, fresh):
            a.copy_(b)
        graph.replay()
        want = run(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), seed


def test_differentiable_once_and_no_dual_tensors():
    x = _cuda(*inputs(1, 10, 1, 8, 8, torch.float32, 19))
    q = x[0].requires_grad_()
    out, _ = policy.compute_gated_delta_rule(q, *x[1:])
    grad, = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            policy.compute_gated_delta_rule(fwd.make_dual(x[0].detach(), x[0].detach()), *x[1:])


def test_many_environments_go_in_several_launches():
    """More pairs than one set of launches takes: the first and last environments as on their own."""
    E, T, H, d = 2100, 70, 50, 2  # 105000 pairs of two chunks: records of 2.4 GB
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(E, T, H, d, generator=g, device="cuda") * 0.5 for _ in range(3))
    beta = torch.rand(E, T, H, generator=g, device="cuda")
    out, last = policy.compute_gated_delta_rule(q, k, v, None, beta)
    for lo in (0, 1020, E - 2):
        few = policy.compute_gated_delta_rule(*(t[lo:lo + 2] for t in (q, k, v)), None, beta[lo:lo + 2])
        assert torch.equal(out[lo:lo + 2], few[0]) and torch.equal(last[lo:lo + 2], few[1])


def test_values_are_checked_where_that_is_asked_for(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "1")
    x, g = torch.zeros(2, 5, 1, 4, device="cuda"), torch.zeros(2, 5, 1, device="cuda")
    policy.compute_gated_delta_rule(x, x, x, g, g)
    with pytest.raises(AssertionError, match="log_decays must not"):
        policy.compute_gated_delta_rule(x, x, x, g + 0.1, g)
    with pytest.raises(AssertionError, match="betas must lie"):
        policy.compute_gated_delta_rule(x, x, x, None, g - 0.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padded_batches(dtype):
    """Steps whose betas and log_decays are 0 write nothing: sequences of several lengths, padded, end with the states of the short ones, and
    what is behind a sequence's end has no part in its gradients.  (The same sums, some of them with zeros: float32's rounding of the state, 64 steps of
    2^-24 of its size at most, and of an output its own.)"""
    q, k, v, g, beta, _, state = _cuda(*inputs(3, 150, 2, 24, 40, dtype, 23))
    lengths = (150, 70, 1)
    for e, n in enumerate(lengths):
        g[e, n:] = 0.0
        beta[e, n:] = 0.0
    xs = [t.detach().clone().requires_grad_() for t in (q, k, v, g, beta, state)]
    out, last = policy.compute_gated_delta_rule(*xs[:5], None, xs[5])
    valid = torch.zeros(3, 150, 1, 1, device="cuda", dtype=dtype)
    for e, n in enumerate(lengths):
        valid[e, :n] = 1.0
    grads = torch.autograd.grad((out, last), xs, (valid.expand_as(out).contiguous(), torch.ones_like(last)))
    for e, n in enumerate(lengths):
        ys = [t[e:e + 1, :n].detach().clone().requires_grad_() for t in (q, k, v, g, beta)] + [state[e:e + 1].detach().clone().requires_grad_()]
        alone, end = policy.compute_gated_delta_rule(*ys[:5], None, ys[5])
        step = torch.finfo(dtype).eps
        assert torch.allclose(out[e:e + 1, :n].float(), alone.float(), rtol=step, atol=64 * 2.0 ** -24 * float(alone.detach().abs().max()))
        assert torch.allclose(last[e:e + 1], end, rtol=0, atol=64 * 2.0 ** -24 * float(end.detach().abs().max()))
        want = torch.autograd.grad((alone, end), ys, (torch.ones_like(alone), torch.ones_like(end)))
        for a, b in zip((*(t[e:e + 1, :n] for t in grads[:5]), grads[5][e:e + 1]), want):
            # (a gradient sums over up to 150 steps and 40 columns)
            assert torch.allclose(a.float(), b.float(), rtol=torch.finfo(a.dtype).eps, atol=256 * 2.0 ** -24 * max(1.0, float(b.abs().max())))
