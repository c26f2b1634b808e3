"""compute_linear_attention and compute_linear_attention_step against the float64 recurrence, step by step.

Error bounds.  Let Y be the recurrence run on absolute values: the sum of the sizes of all terms of a result.  float32:
every term carries a power of the decay (off by less than 24 u where the power is above 1e-6), three products and at
most T + 64 additions, so the result is within (T + 128) u Y, u = 2^-24.  bfloat16: products of queries and keys are rounded
to 8 bits after weighting, the state where outputs are read from it: U16 Y, and the output itself U16 |y|, U16 = 2^-8; a
state is float32 throughout but for its weighted terms, kept as two such numbers: U16^2 Y."""
import math

import pytest
import torch

import rl_triton.policy as policy
from _policy_reference import U16, U32, attention, attention_grads

pytestmark = pytest.mark.gpu


def _make(E, T, H, dk, dv, seed, dtype, ends=0.05, state=True):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(E, T, H, d, generator=g).to(dtype) for d in (dk, dk, dv))
    decay = torch.tensor([0.999, 0.5, 1.0, 0.05, 0.9, 0.0])[torch.arange(H) % 6]
    dones = (torch.rand(E, T, generator=g) < ends).float() if ends is not None else None
    s = torch.randn(E, H, dk, dv, generator=g) if state else None
    return q, k, v, decay, dones, s


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _bounds(args, dtype, T):
    q, k, v, decay, dones, s, scale = args
    y, S = attention(q.abs(), k.abs(), v.abs(), decay, dones, None if s is None else s.abs(), abs(scale))
    exact = (T + 128) * U32
    return (y * (exact + (U16 if dtype == torch.bfloat16 else 0)), S * (exact + (U16 * U16 if dtype == torch.bfloat16 else 0)))


def _within(got, want, bound, unit=0.0):
    err = (got.detach().cpu().double() - want).abs()
    tol = bound + unit * want.abs() + 1e-30
    assert bool((err <= tol).all()), float((err / tol).max())


SHAPES = [(1, 1, 1, 1, 1), (2, 2, 2, 3, 5), (3, 63, 2, 16, 16), (2, 64, 3, 16, 40), (2, 65, 6, 64, 64), (3, 127, 2, 72, 24),
          (1, 130, 2, 128, 128), (2, 333, 4, 40, 72), (1, 1000, 2, 64, 64), (1, 1025, 1, 128, 128), (1, 700, 1, 100, 100),
          (300, 5, 1, 33, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sequences(shape, dtype):
    E, T, H, dk, dv = shape
    for ends, state, scale in ((None, False, None), (0.03, True, 0.3), (0.5, True, None)):
        q, k, v, decay, dones, s = _make(*shape, T + dk, dtype, ends, state)
        out, last = policy.compute_linear_attention(*_cuda(q, k, v, decay, dones, s), scale)
        args = (q, k, v, decay, dones, s, dk ** -0.5 if scale is None else scale)
        want, wlast = attention(*args)
        by, bs = _bounds(args, dtype, T)
        assert out.dtype == dtype and last.dtype == torch.float32
        _within(out, want, by, U16 if dtype == torch.bfloat16 else 0)
        _within(last, wlast, bs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(shape, dtype):
    E, T, H, dk, dv = shape
    for ends, state in ((0.03, True), (None, False)):
        q, k, v, decay, dones, s = _make(*shape, 2 * T + dk, dtype, ends, state)
        g = torch.Generator().manual_seed(T)
        go, gs = torch.randn(E, T, H, dv, generator=g).to(dtype), torch.randn(E, H, dk, dv, generator=g)
        scale = 0.4
        d = [t.requires_grad_() if t is not None else None for t in _cuda(q, k, v, s)]
        out, last = policy.compute_linear_attention(d[0], d[1], d[2], *_cuda(decay, dones), d[3], scale)
        leaves = [t for t in d if t is not None]
        for use_last in (True, False):
            outs, ups = ((out, last), _cuda(go, gs)) if use_last else ((out,), _cuda(go))
            got = torch.autograd.grad(outs, leaves, ups, retain_graph=True)
            w = attention_grads(q, k, v, decay, dones, s, scale, go, gs if use_last else None)
            b = attention_grads(q.abs(), k.abs(), v.abs(), decay, dones, None if s is None else s.abs(), scale, go.abs(),
                                gs.abs() if use_last else None)
            for i, (x, want, size) in enumerate(zip(got, w, b)):
                low = dtype == torch.bfloat16
                unit = (U16 * U16 if i == 3 else U16) if low else 0
                _within(x, want, size * ((T + 128) * U32 + unit), U16 if low and i < 3 else U32)


def test_gradients_against_differences():
    """Directional differences of the float64 recurrence, h = 1e-4: exact but for h^2 (the results are cubic)."""
    q, k, v, decay, dones, s = _make(2, 150, 2, 20, 12, 5, torch.float32)
    g = torch.Generator().manual_seed(6)
    go, gs = torch.randn(2, 150, 2, 12, generator=g), torch.randn(2, 2, 20, 12, generator=g)
    leaves = [t.requires_grad_() for t in _cuda(q, k, v, s)]
    outs = policy.compute_linear_attention(leaves[0], leaves[1], leaves[2], *_cuda(decay, dones), leaves[3], 0.2)
    grads = torch.autograd.grad(outs, leaves, _cuda(go, gs))
    q, k, v, s = (t.detach().double() for t in (q, k, v, s))

    def f(q, k, v, s):
        y, last = attention(q, k, v, decay, dones, s, 0.2)
        return float((y * go).sum() + (last * gs).sum())

    xs = [q, k, v, s]
    for i, grad in enumerate(grads):
        d = torch.randn(xs[i].shape, generator=g).double()
        h = 1e-4
        hi, lo = (f(*[x + sign * h * d if j == i else x for j, x in enumerate(xs)]) for sign in (1, -1))
        prod = grad.cpu().double() * d
        # linear in each argument: the difference is exact to float64; the gradient to (T + 128) u of sizes, here below 1e-4
        assert abs((hi - lo) / (2 * h) - float(prod.sum())) < 1e-4 * float(prod.abs().sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """Time-major views, slices of a joint projection, shared heads, misaligned and element-strided tensors."""
    E, T, H, d = 3, 90, 4, 32
    q, k, v, decay, dones, s = _make(E, T, H, d, d, 3, dtype)
    dev = _cuda(q, k, v, decay, dones, s)
    want = policy.compute_linear_attention(*dev)
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in dev[:3]]
    joint = torch.cat(dev[:3], -1)
    slices = [joint[..., i * d:(i + 1) * d] for i in range(3)]
    strided = [torch.stack([t, t], -1)[..., 0] for t in dev[:3]]
    for views in (major, slices, strided):
        got = policy.compute_linear_attention(*views, *dev[3:])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = []
    for t in dev[:3]:
        buf = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        odd.append(buf[1:].view(t.shape))
    got = policy.compute_linear_attention(*odd, *dev[3:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one key and value head for all: its gradient is the sum over the heads
    k1, v1 = (t[:, :, :1].contiguous().requires_grad_() for t in dev[1:3])
    shared = policy.compute_linear_attention(dev[0], k1.expand(-1, -1, H, -1), v1.expand(-1, -1, H, -1), *dev[3:])
    kf, vf = (t.detach().expand(-1, -1, H, -1).contiguous().requires_grad_() for t in (k1, v1))
    full = policy.compute_linear_attention(dev[0], kf, vf, *dev[3:])
    assert torch.equal(shared[0], full[0])
    up = torch.randn(full[0].shape, device="cuda").to(dtype)
    gk, gv = torch.autograd.grad(shared[0], (k1, v1), up)
    fk, fv = torch.autograd.grad(full[0], (kf, vf), up)
    for a, b in ((gk, fk), (gv, fv)):
        assert torch.allclose(a.float(), b.float().sum(2, keepdim=True), rtol=2 ** -7, atol=2 ** -7 * float(b.abs().max()))
    # the flags in other types
    for flags in (dev[4].bool(), dev[4].bfloat16()):
        got = policy.compute_linear_attention(*dev[:4], flags, dev[5])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_windows_join(dtype):
    """Two windows with the state handed over, and single steps, stay within the bounds of the whole (a state handed over
    carries its own bound into the next window: twice)."""
    E, T, H, dk, dv = 3, 140, 2, 24, 40
    host = _make(E, T, H, dk, dv, 9, dtype)
    q, k, v, decay, dones, s = _cuda(*host)
    want, wlast = attention(*host, dk ** -0.5)
    by, bs = _bounds((*host, dk ** -0.5), dtype, T)
    unit = U16 if dtype == torch.bfloat16 else 0
    for at in (1, 64, 77):
        a, mid = policy.compute_linear_attention(q[:, :at], k[:, :at], v[:, :at], decay, dones[:, :at], s)
        b, end = policy.compute_linear_attention(q[:, at:], k[:, at:], v[:, at:], decay, dones[:, at:], mid)
        _within(torch.cat([a, b], 1), want, 2 * by, unit)
        _within(end, wlast, 2 * bs)
    st, outs = s, []
    for t in range(T):
        o, st = policy.compute_linear_attention_step(q[:, t], k[:, t], v[:, t], decay, st, dones[:, t - 1] if t else None)
        outs.append(o)
    _within(torch.stack(outs, 1), want, by, unit)
    _within(torch.where(dones[:, -1, None, None, None] != 0, 0.0, st), wlast, bs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,H,dk,dv", [(1, 1, 1, 1), (3, 2, 5, 3), (4, 6, 64, 64), (2, 3, 40, 72), (2, 2, 128, 128), (5, 1, 100, 33)])
def test_step(E, H, dk, dv, dtype):
    """In float32: a product, a sum and dk products and sums of them: (dk + 8) u of the sizes; bfloat16 rounds the output."""
    q, k, v, decay, dones, s = _make(E, 1, H, dk, dv, dk, dtype, 0.5)
    q, k, v, dones = q[:, 0], k[:, 0], v[:, 0], dones[:, 0]
    for flags in (dones, None):
        args = _cuda(q, k, v, decay, s, flags)
        keep = args[4].clone()
        out, new = policy.compute_linear_attention_step(*args)
        assert torch.equal(args[4], keep)
        lam = decay.double()[None].expand(E, H)
        lam = lam if flags is None else torch.where(flags[:, None] != 0, 0.0, lam)
        S = s.double() * lam[..., None, None] + k.double()[..., :, None] * v.double()[..., None, :]
        size = s.double().abs() * lam[..., None, None] + k.double().abs()[..., :, None] * v.double().abs()[..., None, :]
        _within(new, S, 4 * U32 * size)
        y = (q.double()[..., :, None] * S).sum(-2) * dk ** -0.5
        ysize = (q.double().abs()[..., :, None] * size).sum(-2) * dk ** -0.5
        _within(out, y, (dk + 8) * U32 * ysize, U16 if dtype == torch.bfloat16 else 0)
        out2, new2 = policy.compute_linear_attention_step(*args, out_state=args[4])
        assert new2 is args[4] and torch.equal(new2, new) and torch.equal(out2, out)


def test_a_cut_state_has_no_part():
    """Whatever the state held, NaN included, does not pass an episode's end."""
    q, k, v, decay, _, s = _make(2, 70, 2, 16, 16, 4, torch.float32)
    dones = torch.zeros(2, 70)
    dones[0, 63] = 1
    s[0] = math.nan
    out, last = policy.compute_linear_attention(*_cuda(q, k, v, decay, dones, s))
    assert bool(out[0, :64].isnan().any()) and bool(out[0, 64:].isfinite().all()) and bool(last.isfinite().all())
    o, new = policy.compute_linear_attention_step(*_cuda(q[:, 0], k[:, 0], v[:, 0], decay, s, torch.tensor([1.0, 0.0])))
    assert bool(o.isfinite().all()) and bool(new.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [24, 64, 100, 128])
def test_values_that_are_not_finite_stay_where_they_belong(d, dtype):
    """An inf, a NaN or a value whose products overflow, in q, k, v or an upstream gradient (garbage in padded steps is such a
    value), reaches what it reaches in the recurrence: nothing before it, nothing past its episode's end."""
    E, T, H = 2, 200, 2
    q, k, v, decay, _, s = _make(E, T, H, d, d, 7, dtype)
    dones = torch.zeros(E, T)
    dones[:, [59, 70, 71, 150]] = 1
    gen = torch.Generator().manual_seed(1)
    go, gs = torch.randn(E, T, H, d, generator=gen).to(dtype), torch.randn(E, H, d, d, generator=gen)
    # head 0 of environment 0, the episode of the steps 60..70: what is not finite
    q[0, 65, 0, 3], k[0, 66, 0, 1], v[0, 67, 0, 2], v[0, 68, 0, 5], go[0, 66, 0, 0] = math.nan, math.inf, -math.inf, math.nan, math.inf
    k[0, 70, 0] = math.nan
    # head 1 of environment 1: the type's lowest and largest values
    low = torch.finfo(dtype).min
    q[1, 65:68, 1], k[1, 65:68, 1], v[1, 65:68, 1], go[1, 65:68, 1] = low, low, -low, -low
    huge = torch.zeros(E, T, H, dtype=torch.bool)
    huge[1, 60:71, 1] = True

    leaves = [t.requires_grad_() for t in _cuda(q, k, v, s)]
    out, last = policy.compute_linear_attention(leaves[0], leaves[1], leaves[2], *_cuda(decay, dones), leaves[3], 0.3)
    got = (out, last, *torch.autograd.grad((out, last), leaves, _cuda(go, gs)))
    q, k, v, s = (t.detach() for t in (q, k, v, s))
    args = (q, k, v, decay, dones, s, 0.3)
    want = (*attention(*args), *attention_grads(*args, go, gs))
    by, bs = _bounds(args, dtype, T)
    sizes = attention_grads(q.abs(), k.abs(), v.abs(), decay, dones, s.abs(), 0.3, go.abs(), gs.abs())
    wide = dtype == torch.bfloat16
    bounds = (by, bs, *[x * ((T + 128) * U32 + ((U16 * U16 if i == 3 else U16) if wide else 0)) for i, x in enumerate(sizes)])
    for i, (x, w, bound) in enumerate(zip(got, want, bounds)):
        unit = (U16 if wide and i not in (1, 5) else 0) + U32
        x = x.detach().cpu().double()
        if i not in (1, 5):  # (a state belongs to no step)
            before = huge.clone()
            before[:, 65:] = False  # outputs and their queries' gradients from before them
            seen = ~huge | before if i == 0 else ~huge
            x, w, bound = x[seen], w[seen], bound[seen]
        kept = w.isfinite()
        assert bool((x.isfinite() == kept).all()), i
        _within(x[kept], w[kept], bound[kept], unit)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [40, 128])
def test_values_that_are_not_finite_in_sequences_cut_into_segments(d, dtype):
    """The same over 20 chunks of one environment and head, whose segments' states are found first.  A NaN without an episode's
    end after it reaches every later step, past the point where its decay is too small for float32."""
    E, T, H = 1, 1280, 2
    q, k, v, _, _, s = _make(E, T, H, d, d, 8, dtype)
    decay = torch.tensor([0.99, 0.5])
    dones = torch.zeros(E, T)
    dones[0, [300, 420]] = 1
    gen = torch.Generator().manual_seed(2)
    go, gs = torch.randn(E, T, H, d, generator=gen).to(dtype), torch.randn(E, H, d, d, generator=gen)
    k[0, 330, 0, 3], v[0, 350, 0, 2], k[0, 500, 1, 5], go[0, 310, 1, 1] = math.nan, math.inf, math.nan, -math.inf
    leaves = [t.requires_grad_() for t in _cuda(q, k, v, s)]
    out, last = policy.compute_linear_attention(leaves[0], leaves[1], leaves[2], *_cuda(decay, dones), leaves[3], 0.3)
    got = (out, last, *torch.autograd.grad((out, last), leaves, _cuda(go, gs)))
    q, k, v, s = (t.detach() for t in (q, k, v, s))
    args = (q, k, v, decay, dones, s, 0.3)
    want = (*attention(*args), *attention_grads(*args, go, gs))
    assert bool(want[0][0, -1, 1].isnan().any()) and not bool(want[0][0, 421:, 0].isnan().any())
    by, bs = _bounds(args, dtype, T)
    sizes = attention_grads(q.abs(), k.abs(), v.abs(), decay, dones, s.abs(), 0.3, go.abs(), gs.abs())
    wide = dtype == torch.bfloat16
    bounds = (by, bs, *[x * ((T + 128) * U32 + ((U16 * U16 if i == 3 else U16) if wide else 0)) for i, x in enumerate(sizes)])
    for i, (x, w, bound) in enumerate(zip(got, want, bounds)):
        x, kept = x.detach().cpu().double(), w.isfinite()
        assert bool((x.isfinite() == kept).all()), i
        _within(x[kept], w[kept], bound[kept], (U16 if wide and i not in (1, 5) else 0) + U32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_of_large_states(dtype):
    """States of 256 MB and more, which take another path through the caches; bounds as above."""
    E, H, d = 4096 + 3, 1, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(E, H, d, generator=g, device="cuda").to(dtype) for _ in range(3))
    s, decay = torch.randn(E, H, d, d, generator=g, device="cuda"), torch.tensor([0.75], device="cuda")
    done = (torch.rand(E, generator=g, device="cuda") < 0.25).float()
    out, new = policy.compute_linear_attention_step(q, k, v, decay, s, done, 0.5)
    lam = torch.where(done != 0, 0.0, 0.75)[:, None, None, None]
    for part in (slice(0, 300), slice(E - 300, E)):
        S = s[part].double() * lam[part] + k[part].double()[..., :, None] * v[part].double()[..., None, :]
        size = s[part].double().abs() * lam[part] + k[part].double().abs()[..., :, None] * v[part].double().abs()[..., None, :]
        assert bool(((new[part].double() - S).abs() <= 4 * U32 * size).all())
        y = (q[part].double()[..., :, None] * S).sum(-2) * 0.5
        bound = (d + 8) * U32 * (q[part].double().abs()[..., :, None] * size).sum(-2) * 0.5
        assert bool(((out[part].double() - y).abs() <= bound + (U16 if dtype == torch.bfloat16 else 0) * y.abs()).all())
    again, same = policy.compute_linear_attention_step(q, k, v, decay, s, done, 0.5, out_state=s)
    assert same is s and torch.equal(again, out) and torch.equal(s, new)


def test_more_pairs_than_a_launch_takes():
    """Two million sequences of two steps, nine million single steps: several launches over ranges of environments.  Two
    products and a sum a result: 8 u of the sizes."""
    E, g = (1 << 21) + 77, torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v, s = n(E, 2, 1, 1), n(E, 2, 1, 1), n(E, 2, 1, 1), n(E, 1, 1, 1)
    decay = torch.tensor([0.5], device="cuda")
    out, last = policy.compute_linear_attention(q, k, v, decay, None, s, 1.0)
    s1 = 0.5 * s[:, 0].double() + (k * v)[:, 0].double()
    s2 = 0.5 * s1 + (k * v)[:, 1].double()
    for got, want in ((out[:, 0], q[:, 0] * s1), (out[:, 1], q[:, 1] * s2), (last[:, 0], s2)):
        assert bool(((got.double() - want).abs() <= 8 * U32 * 8 * (1 + want.abs())).all())
    E = (1 << 23) + 77
    q, k, v, s = n(E, 1, 1), n(E, 1, 1), n(E, 1, 1), n(E, 1, 1, 1)
    out, new = policy.compute_linear_attention_step(q, k, v, decay, s, None, 1.0)
    s1 = 0.5 * s[:, 0].double() + (k * v).double()
    assert bool(((new[:, 0].double() - s1).abs() <= 64 * U32 * (1 + s1.abs())).all())
    assert bool(((out.double() - q * s1).abs() <= 64 * U32 * (1 + (q * s1).abs())).all())


def test_nothing_to_do():
    z = torch.zeros(2, 0, 3, 8, device="cuda", requires_grad=True)
    s = torch.randn(2, 3, 8, 8, device="cuda")
    out, last = policy.compute_linear_attention(z, z, z, torch.ones(3, device="cuda"), None, s)
    assert out.shape == z.shape and torch.equal(last, s)
    z = torch.zeros(0, 5, 3, 8, device="cuda")
    out, last = policy.compute_linear_attention(z, z, z, torch.ones(3, device="cuda"))
    assert out.shape == z.shape and last.shape == (0, 3, 8, 8)
    z = torch.zeros(0, 3, 8, device="cuda")
    out, last = policy.compute_linear_attention_step(z, z, z, torch.ones(3, device="cuda"), torch.zeros(0, 3, 8, 8, device="cuda"))
    assert out.shape == z.shape


def test_graph():
    import os
    os.environ["RL_TRITON_CORRECTNESS_WARNINGS"] = "0"
    dev = _cuda(*_make(1, 700, 2, 32, 32, 9, torch.bfloat16))  # few rows: segments and their workspace

    def call():
        out, last = policy.compute_linear_attention(*dev)
        return out, last, *policy.compute_linear_attention_step(dev[0][:, 0], dev[1][:, 0], dev[2][:, 0], dev[3], last)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (1, 2, 3):
        for t, n in zip(dev, _make(1, 700, 2, 32, 32, seed, torch.bfloat16)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call()))
