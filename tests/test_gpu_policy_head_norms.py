"""compute_query_key_norms against its definition in float64.

Roundings (u = 2^-24): the mean of n squares is within (n / 8 + 8) u of itself (a lane's 8 and more elements and then halves), its root within half of
that and 2 u; three products and a rotation (sine and cosine within 4 u of 1, two products and a sum) add 10 u of the pair's size: (n / 16 + 16) u
of the larger of a pair, and the storage type's rounding of the result.  Back, two such sums: twice that of the row's largest term, times
sqrt(n) for the mean that is taken off.  Weights' gradients are sums over the rows, in float32 over a part of them and in float64 over the parts:
each row's term within those bounds, and sqrt(rows) u for the sum, of the sum of sizes."""
import math

import pytest
import torch

import rl_triton.policy as policy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")

U32, U16 = 2.0 ** -24, 2.0 ** -8
DTYPES = [torch.float32, torch.bfloat16]


def turned(x, positions, base, rotary, interleaved, sign=1):
    if positions is None or rotary == 0:
        return x
    i = torch.arange(rotary // 2, dtype=torch.float64, device=x.device)
    angle = sign * (positions.double()[..., None, None] * base ** (-2 * i / rotary))
    cos, sin = angle.cos(), angle.sin()
    a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    y = x.clone()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def definition(x, weight, positions, base=10000.0, rotary=None, eps=1e-6, interleaved=False, up=None):
    rotary = x.shape[-1] if rotary is None else rotary
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if weight is None else weight.double()
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    out = turned(x * r * w, positions, base, rotary, interleaved)
    if up is None:
        return out
    g = turned(up.double(), positions, base, rotary, interleaved, -1)
    unit = x * r
    wg = g * w
    grad = r * (wg - unit * (wg * unit).mean(-1, keepdim=True))
    return out, grad, (g * unit).flatten(0, -2).sum(0), (g * unit).abs().flatten(0, -2).sum(0), r * wg.abs().amax(-1, keepdim=True)


def _inputs(shape, heads, dim, dtype, seed, far=1000000):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k = (n(*shape, h, dim).to(dtype) * 2 for h in heads)
    return q, k, 1 + 0.2 * n(dim), 1 + 0.2 * n(dim), torch.randint(0, far + 1, shape, generator=g, device="cuda")


def _hold_rows(got, want, dtype, dim, sizes=None, times=1.0):
    """`sizes`: what an element's error is counted in."""
    assert got.dtype == dtype and got.is_contiguous()
    sizes = want.abs().amax(-1, keepdim=True) if sizes is None else sizes
    tol = times * (dim / 16 + 16) * U32 * sizes + (U16 if dtype == torch.bfloat16 else U32) * want.abs() + 1e-37
    err = (got.detach().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


SHAPES = [((1, 1), (1, 1), 1, 0), ((2, 3), (2, 1), 2, None), ((3, 5), (4, 2), 7, 4), ((2, 9), (3, 3), 24, None), ((2, 9), (5, 1), 40, 20), ((4, 33), (9, 2), 64, None),
          ((37, 5), (4, 2), 72, 40), ((3, 70), (16, 4), 128, None), ((2, 7), (2, 2), 128, 64), ((2, 5), (2, 3), 200, 20), ((2, 5), (1, 2), 201, 20), ((3, 5), (2, 2), 256, None),
          ((5,), (3, 2), 64, None), ((700,), (1, 1), 96, 48), ((2, 3), (4, 0), 64, None), ((2, 3), (0, 4), 36, 18)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SHAPES)
def test_rows(case, dtype, interleaved):
    shape, heads, dim, rotary = case
    q, k, qw, kw, pos = _inputs(shape, heads, dim, dtype, dim)
    for weights, positions, eps in (((qw, kw), pos, 1e-6), ((None, kw), None, 0.5), ((None, None), pos, 0.0)):
        r = rotary if positions is not None else None
        got = policy.compute_query_key_norms(q, k, *weights, positions, rotary_dim=r, eps=eps, interleaved=interleaved, base=500.0)
        for x, y, w in zip((q, k), got, weights):
            if x.numel():
                want = definition(x, w, positions, 500.0, r if positions is not None else 0, eps, interleaved)
                _hold_rows(y, want, dtype, dim, (want / (1 if w is None else w.double())).abs().amax(-1, keepdim=True) * 2)
            assert y.shape == x.shape


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SHAPES)
def test_gradients(case, dtype, interleaved):
    shape, heads, dim, rotary = case
    q, k, qw, kw, pos = _inputs(shape, heads, dim, dtype, dim + 1)
    up = [torch.randn(x.shape, device="cuda").to(dtype) for x in (q, k)]
    for t in (q, k, qw, kw):
        t.requires_grad_()
    outs = policy.compute_query_key_norms(q, k, qw, kw, pos, rotary_dim=rotary, interleaved=interleaved)
    got = torch.autograd.grad(outs, (q, k, qw, kw), up, retain_graph=True)
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        _, grad, dw, size, largest = definition(x.detach(), w.detach(), pos, rotary=rotary, interleaved=interleaved, up=up[i])
        if x.numel() == 0:
            assert bool((got[2 + i] == 0).all())
            continue
        _hold_rows(got[i], grad, dtype, dim, largest * math.sqrt(dim), 2.0)
        rows = x.numel() // dim
        assert bool(((got[2 + i].double() - dw).abs() <= (dim / 8 + 32 + math.sqrt(rows)) * U32 * size.clamp_min(float(size.max()) / 4)).all())
    # one output, one gradient at a time: the same bits
    for i in range(2):
        if outs[i].numel() == 0:
            continue
        for j in (i, 2 + i):
            a, = torch.autograd.grad(outs[i], (q, k, qw, kw)[j], up[i], retain_graph=True)
            assert torch.equal(a, got[j])
        unused = torch.autograd.grad(outs[i], ((q, k)[1 - i], (qw, kw)[1 - i]), up[i], retain_graph=True, allow_unused=True)
        assert all(t is None or not bool(t.any()) for t in unused)


def test_gradients_against_differences():
    q, k, qw, kw, pos = _inputs((2, 30), (3, 2), 20, torch.float32, 4)
    up = [torch.randn(x.shape, device="cuda") for x in (q, k)]
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    grads = torch.autograd.grad(policy.compute_query_key_norms(*leaves, pos, rotary_dim=12), leaves, up)
    for i, grad in enumerate(grads):
        step = torch.randn(leaves[i].shape, device="cuda").double()
        values = []
        for sign in (1, -1):
            x = [t.detach().double() for t in leaves]
            x[i] = x[i] + sign * 1e-4 * step
            values.append(sum(float((definition(x[j], x[2 + j], pos, rotary=12) * up[j]).sum()) for j in range(2)))
        prod = grad.double() * step
        assert abs((values[0] - values[1]) / 2e-4 - float(prod.sum())) < 1e-4 * float(prod.abs().sum())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [48, 50])
def test_layouts(dtype, dim):
    """Slices of a joint projection, time-major views, misaligned and element-strided rows, shared keys, weights of a table."""
    q, k, qw, kw, pos = _inputs((4, 30), (4, 4), dim, dtype, 5)
    up = [torch.randn(x.shape, device="cuda").to(dtype) for x in (q, k)]

    def run(q, k, qw, kw, pos, up):
        leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
        outs = policy.compute_query_key_norms(*leaves, pos, rotary_dim=16)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, up))

    want = run(q, k, qw, kw, pos, up)
    joint = torch.cat([q, k], -2)
    wide = torch.zeros(4, 30, 4, dim + 1, dtype=dtype, device="cuda")
    wide[..., 1:] = q
    views = [(joint[..., :4, :], joint[..., 4:, :]), (wide[..., 1:], k)]
    views += [tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k)), tuple(torch.stack([t, t], -1)[..., 1] for t in (q, k))]
    table = torch.stack([qw, kw], -1)
    for a, b in views:
        got = run(a, b, table[:, 0], table[:, 1], pos.t().contiguous().t(), [t.transpose(1, 2).contiguous().transpose(1, 2) for t in up])
        for x, y in zip(got, want):  # (4 pairs at a time or one: sums in another order)
            assert torch.allclose(x.float(), y.float(), rtol=(dim / 16 + 16) * U32 if dtype == torch.float32 else 2 * U16, atol=3e-5 if dtype == torch.float32 else 2e-2)
    same = run(k[:, :, :1].expand(-1, -1, 4, -1), k, qw, kw, pos, up)
    assert torch.equal(same[0][:, :, 0], same[0][:, :, 3])


def test_far_positions():
    """Positions up to 2^40 are turned as exactly as near ones (float64 holds the angle's turns to 2^-13 of a float32's last bit there)."""
    q, k, _, _, _ = _inputs((4, 9), (2, 2), 32, torch.float32, 6)
    for far in (0, 1 << 20, 1 << 31, (1 << 33) + 7, 1 << 40):
        pos = far + torch.arange(36, device="cuda").view(4, 9)
        got = policy.compute_query_key_norms(q, k, None, None, pos)[0]
        want = definition(q, None, pos)
        _hold_rows(got, want, torch.float32, 32, want.abs().amax(-1, keepdim=True) * (1 if far < 1 << 32 else 1 + far * 2.0 ** -53 * 2 / U32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_rows_stay_alone(dtype):
    """A NaN or an infinity reaches its own row and the weights' gradients only; rows of zeros have finite gradients."""
    q, k, qw, kw, pos = _inputs((3, 40), (4, 2), 64, dtype, 7)
    up = [torch.randn(x.shape, device="cuda").to(dtype) for x in (q, k)]

    def run(q):
        leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
        outs = policy.compute_query_key_norms(*leaves, pos)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, up))

    clean = run(q)
    bad = q.clone()
    bad[1, 7, 2, 3], bad[2, 30, 1, 60] = math.nan, math.inf
    keep = torch.ones(3, 40, 4, dtype=torch.bool, device="cuda")
    keep[1, 7, 2] = keep[2, 30, 1] = False
    got = run(bad)
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[2][keep], clean[2][keep])
    assert torch.equal(got[1], clean[1]) and torch.equal(got[3], clean[3]) and torch.equal(got[5], clean[5])
    zero = q.clone()
    zero[1, 7] = 0.0
    got = run(zero)
    assert all(bool(torch.isfinite(t.float()).all()) for t in got) and not bool(got[0][1, 7].any())


def test_many_rows_and_empty_calls():
    """More rows than one trip of the workgroups; offsets past 32 bits; none at all."""
    q, k, qw, kw, pos = _inputs((70000, 3), (2, 1), 16, torch.bfloat16, 8)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    up = [torch.randn(x.shape, device="cuda").bfloat16() for x in (q, k)]
    outs = policy.compute_query_key_norms(*leaves, pos)
    got = torch.autograd.grad(outs, leaves, up)
    for i in range(2):
        _, grad, dw, size, largest = definition(leaves[i].detach(), leaves[2 + i].detach(), pos, up=up[i])
        _hold_rows(got[i], grad, torch.bfloat16, 16, largest * 4, 2.0)
        assert bool(((got[2 + i].double() - dw).abs() <= (34 + math.sqrt(420000)) * U32 * size).all())
    far = torch.empty(2, (1 << 32) // 64 + 1, 1, 64, dtype=torch.bfloat16, device="cuda")[:, ::1 << 20]  # (a view of a few rows, 2^31 elements and more apart)
    far.normal_()
    p = torch.zeros(far.shape[:2], dtype=torch.int64, device="cuda") + 3
    a = policy.compute_query_key_norms(far, far, None, None, p)
    b = policy.compute_query_key_norms(far.contiguous(), far.contiguous(), None, None, p)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for shape in ((0, 4), (4, 0)):
        x = torch.zeros(*shape, 2, 8, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        o = policy.compute_query_key_norms(x, x, w, None, torch.zeros(shape, dtype=torch.int64, device="cuda"))
        gx, gw = torch.autograd.grad(o, (x, w), (torch.ones_like(x), torch.ones_like(x)))
        assert gx.shape == x.shape and not bool(gw.any())


def test_streams_graphs_and_repeats():
    q, k, qw, kw, pos = _inputs((8, 200), (8, 2), 64, torch.bfloat16, 9)
    up = [torch.randn(x.shape, device="cuda").bfloat16() for x in (q, k)]

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
        outs = policy.compute_query_key_norms(*leaves, pos)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, up))

    want = run()
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for _ in range(3):
        q.normal_()
        pos.random_(0, 1000)
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_values_are_checked_where_that_is_asked_for(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "1")
    x = torch.zeros(2, 5, 1, 4, device="cuda")
    policy.compute_query_key_norms(x, x, positions=torch.zeros(2, 5, dtype=torch.int64, device="cuda"))
    with pytest.raises(AssertionError, match="positions must not be negative"):
        policy.compute_query_key_norms(x, x, positions=torch.full((2, 5), -1, device="cuda"))
