"""compute_action_log_probs against the float64 softmax, forward and backward.

Error bounds, derived for rows of A logits with spread R = max |x - m| / tau <= 60: y = (x - m) c carries three
roundings, 3 u |y| (u = 2^-24), so each exponential is off by 3 u R + 2 u; a sum of A positive terms in at most
128 steps a lane and 12 joining steps adds 140 u.  So log s is off by E = (3 R + 142) u < 2e-5, log p by E + 3 u R, the
entropy by E + (E + 3 u R) H, and p by a relative 2 E."""
import math

import pytest
import torch

import rl_triton.policy as policy
from _policy_reference import U16, logits_grad, softmax_rows

pytestmark = pytest.mark.gpu
E = 2e-5


def _make(rows, A, seed, dtype, kind="plain"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*rows, A, generator=g) * 3
    a = torch.randint(0, A, rows, generator=g)
    if kind == "invalid":
        x[torch.rand(*rows, A, generator=g) < 0.3] = -math.inf
        x.scatter_(-1, a[..., None], torch.randn(*rows, 1, generator=g))
    return x.to(dtype), a


def _check(x, a, tau, xd=None, ad=None):
    xd = x.cuda() if xd is None else xd
    lp, ent = policy.compute_action_log_probs(xd, a.cuda() if ad is None else ad, tau)
    rlp, rent, *_ = softmax_rows(x, a, tau)
    assert lp.dtype == ent.dtype == torch.float32 and lp.shape == ent.shape == a.shape
    assert torch.allclose(lp.cpu().double(), rlp, rtol=1e-6, atol=E, equal_nan=True)
    assert torch.allclose(ent.cpu().double(), rent, rtol=2 * E, atol=E, equal_nan=True)


SIZES = [1, 2, 3, 7, 18, 31, 32, 33, 63, 64, 65, 100, 255, 257, 1000, 1024, 1025, 4097, 8192, 16385, 20001, 65536, 65537, 131072,
         140001]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("A", SIZES)
def test_rows_of_every_length(A, dtype):
    rows = (3, 67) if A <= 1025 else (2, 3)
    for kind in ("plain", "invalid"):
        _check(*_make(rows, A, A, dtype, kind), 0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("A", [1, 18, 64, 1000, 5001])
def test_layouts(A, dtype):
    """Offsets into larger buffers, slices of wider rows, time-major views, rows with a strided action axis, other ranks."""
    x, a = _make((5, 9), A, 7 * A, dtype)
    for off in (1, 2, 3):
        buf = torch.zeros(x.numel() + off, dtype=dtype, device="cuda")
        buf[off:] = x.reshape(-1).cuda()
        _check(x, a, 1.0, buf[off:].view(x.shape))
    wide = torch.zeros(5, 9, A + 3, dtype=dtype, device="cuda")
    wide[..., 1:A + 1] = x.cuda()
    _check(x, a, 1.0, wide[..., 1:A + 1])
    _check(x, a, 1.0, x.cuda().transpose(0, 1).contiguous().transpose(0, 1), a.cuda().t().contiguous().t())
    _check(x, a, 1.0, x.cuda().transpose(-1, -2).contiguous().transpose(-1, -2))
    _check(x.view(-1, A), a.view(-1), 1.0)
    _check(x[0, 0], a[0, 0], 1.0)
    _check(x.view(5, 3, 3, A), a.view(5, 3, 3), 1.0)


@pytest.mark.parametrize("A", [1, 5, 40, 700, 3000, 140001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_that_masks_leave(A, dtype):
    """Rows of -inf alone, of the type's lowest value alone, one finite logit, NaN, +inf, actions out of range."""
    low = torch.finfo(dtype).min
    x, _ = _make((1, 7), A, A, dtype)
    x[0, 0] = -math.inf
    x[0, 1] = low
    x[0, 2, :] = -math.inf
    x[0, 2, A // 2] = 1.5
    x[0, 3, A - 1] = math.nan
    x[0, 4, 0] = math.inf
    a = torch.tensor([[0, A - 1, A // 2, 0, 0, -1, A]])
    import os
    os.environ["RL_TRITON_CORRECTNESS_WARNINGS"] = "0"  # (out-of-range actions are refused with it)
    lp, ent = policy.compute_action_log_probs(x.cuda(), a.cuda())
    lp, ent = lp.cpu()[0], ent.cpu()[0]
    assert lp[0] == -math.inf and ent[0] == 0
    assert abs(lp[1] + math.log(A)) < E and abs(ent[1] - math.log(A)) < E * (1 + math.log(A))
    assert lp[2] == 0 and ent[2] == 0
    assert lp[3].isnan() and ent[3].isnan() and lp[4].isnan() and ent[4].isnan()
    assert lp[5].isnan() and lp[6].isnan() and ent[5].isfinite() and ent[6].isfinite()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("A", [5, 18, 60, 300, 3000, 9000, 50001, 140001])
@pytest.mark.parametrize("rows", [(1, 3), (2, 700)])
def test_masks_of_the_lowest_value(A, rows, dtype):
    """Logits of the type's lowest value count as nothing beside others, wherever they lie: first, last, most of the row."""
    if rows[1] > 3 and A > 9000:
        rows = (2, 300)
    x, a = _make(rows, A, A + 1, dtype)
    g = torch.Generator().manual_seed(A)
    low = torch.rand(x.shape, generator=g) < torch.tensor([0.1, 0.9, 0.99])[torch.randint(0, 3, rows, generator=g)][..., None]
    low[..., :A // 3] = True
    low.scatter_(-1, a[..., None], False)
    _check(torch.where(low, torch.finfo(dtype).min, x.float()).to(dtype), a, 0.6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 2, 7, 33, 130, 256, 257])
def test_few_long_rows(rows, dtype):
    """Rows shared by several workgroups, of every alignment, with parts that hold nothing but -inf."""
    for A in (8192, 20011, 33333, 49153, 98307):
        x, a = _make((1, rows), A, A + rows, dtype, "invalid")
        x[0, 0, A // 4:3 * A // 4] = -math.inf
        a[0, 0] = A - 1
        x[0, 0, A - 1] = 1.0
        if rows > 2:
            x[0, 1] = -math.inf
            x[0, 2, A // 2] = math.nan
        if A > 33333 and rows > 100:
            continue
        _check(x, a, 0.9)


def _grad_check(x, a, tau, xd, seed=3):
    g = torch.Generator().manual_seed(seed)
    gl, ge = torch.randn(a.shape, generator=g), torch.randn(a.shape, generator=g)
    xd = xd.detach().requires_grad_()
    lp, ent = policy.compute_action_log_probs(xd, a.cuda(), tau)
    _, rent, p, logp = softmax_rows(x, a, tau)
    for use_l, use_e in ((1, 1), (1, 0), (0, 1)):
        outs, ups = zip(*[(o, u.cuda()) for o, u, use in ((lp, gl, use_l), (ent, ge, use_e)) if use])
        got, = torch.autograd.grad(outs, xd, ups, retain_graph=True)
        assert got.dtype == x.dtype and got.shape == x.shape
        want = logits_grad(p, logp, rent, a, gl.double() * use_l, ge.double() * use_e, tau)
        # p carries 2 E, the bracket E (1 + H); the stored type its own rounding
        size = (use_l * gl.abs()[..., None] * p + use_e * ge.abs()[..., None] * p *
                torch.where(p > 0, logp.abs() + 1 + 2 * rent[..., None], 0.0)) / tau
        unit = U16 if x.dtype == torch.bfloat16 else 2.0 ** -22
        bound = 4 * E * size + unit * want.abs() + 1e-30
        err = (got.cpu().double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("A", [1, 2, 18, 33, 257, 1025, 20001, 70001])
def test_gradient(A, dtype):
    x, a = _make((3, 21) if A < 2000 else (2, 2), A, A + 1, dtype, "invalid")
    _grad_check(x, a, 0.8, x.cuda())
    wide = torch.zeros(*x.shape[:2], A + 5, dtype=dtype, device="cuda")
    wide[..., 2:A + 2] = x.cuda()
    _grad_check(x, a, 0.8, wide[..., 2:A + 2])


def test_gradient_against_differences():
    """Directional differences of the float64 definition: (f(x + h d) - f(x - h d)) / 2h, h = 1e-4."""
    x, a = _make((4, 6), 50, 11, torch.float32)
    g = torch.Generator().manual_seed(4)
    gl, ge = torch.randn(a.shape, generator=g), torch.randn(a.shape, generator=g)
    d = torch.randn(x.shape, generator=g).double()
    xd = x.cuda().requires_grad_()
    outs = policy.compute_action_log_probs(xd, a.cuda(), 1.3)
    got, = torch.autograd.grad(outs, xd, (gl.cuda(), ge.cuda()))

    def f(y):
        lp, ent, *_ = softmax_rows(y, a, 1.3)
        return float((lp * gl).sum() + (ent * ge).sum())

    h = 1e-4
    diff = (f(x.double() + h * d) - f(x.double() - h * d)) / (2 * h)
    dot = float((got.cpu().double() * d).sum())
    # differences: h^2 times a third derivative of size ~1 per logit (1200 of them); gradient: E of its size
    assert abs(diff - dot) < 1e-8 * 1200 + 4 * E * float((got.cpu().double() * d).abs().sum())


def test_empty_rows_have_no_gradient():
    x = torch.full((1, 2, 40), -math.inf)
    x[0, 1, 3] = 0.0
    a = torch.tensor([[5, 3]])
    xd = x.cuda().requires_grad_()
    lp, ent = policy.compute_action_log_probs(xd, a.cuda())
    g, = torch.autograd.grad((lp, ent), xd, (torch.ones(1, 2, device="cuda"),) * 2)
    assert bool((g == 0).all())


def test_no_rows():
    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        lp, ent = policy.compute_action_log_probs(x, torch.zeros(shape[:2], dtype=torch.int64, device="cuda"))
        assert lp.shape == ent.shape == shape[:2]
        assert torch.autograd.grad(lp.sum(), x)[0].shape == shape


def test_other_stream_and_graph():
    x, a = _make((8, 16), 18, 5, torch.float32)
    xd, ad = x.cuda(), a.cuda()
    want = policy.compute_action_log_probs(xd, ad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = policy.compute_action_log_probs(xd, ad)
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    import os
    os.environ["RL_TRITON_CORRECTNESS_WARNINGS"] = "0"
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = policy.compute_action_log_probs(xd, ad)
    for seed in (1, 2, 3):
        xd.copy_(_make((8, 16), 18, seed, torch.float32)[0])
        graph.replay()
        torch.cuda.synchronize()
        eager = policy.compute_action_log_probs(xd, ad)
        assert all(torch.equal(u, v) for u, v in zip(out, eager))
