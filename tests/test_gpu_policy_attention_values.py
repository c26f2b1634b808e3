"""Linear attention at values and sizes where one path of it could answer otherwise than another: infinities at head dims that fill
no whole tile, decays of 0, sequences of no steps, and how exact bfloat16 calls are."""
import ctypes
import math

import pytest
import torch

import rl_triton.policy as policy
from _policy_reference import U16, U32, attention, attention_grads
from rl_triton.policy import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", [(24, 24), (40, 72), (64, 64), (100, 33), (128, 128), (1, 1)])
def test_infinities_stay_infinities(dk, dv, dtype):
    """Where the recurrence gives inf the call does, and NaN where it gives NaN: dims that do not exist have no part in it.
    (Queries and values have no zeros, so that inf times one of them is inf.)"""
    E, T, H = 2, 90, 2
    g = torch.Generator().manual_seed(dk)
    n = lambda *s: (torch.rand(s, generator=g) + 0.5).to(dtype)  # noqa: E731
    q, k, v, go = n(E, T, H, dk), n(E, T, H, dk), n(E, T, H, dv), n(E, T, H, dv)
    decay = torch.tensor([0.9, 1.0])
    dones = torch.zeros(E, T)
    dones[:, 80] = 1
    k[0, 70, 0, 0] = math.inf
    v[0, 75, 1, dv - 1] = -math.inf
    k[1, 66, 0, dk - 1], v[1, 67, 0, 0] = math.inf, math.nan
    q[1, 72, 1, 0] = math.inf
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, last = policy.compute_linear_attention(*leaves, decay.cuda(), dones.cuda(), None, 0.5)
    got = (out, last, *torch.autograd.grad(out, leaves, go.cuda()))
    want = (*attention(q, k, v, decay, dones, None, 0.5), *attention_grads(q, k, v, decay, dones, None, 0.5, go, None)[:3])
    for i, (x, w) in enumerate(zip(got, want)):
        x = x.detach().cpu().double()
        assert torch.equal(x.isnan(), w.isnan()), i
        assert torch.equal(x == math.inf, w == math.inf) and torch.equal(x == -math.inf, w == -math.inf), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_decay_of_zero_forgets_what_is_not_finite(bad, dtype):
    """A head that forgets everything forgets a state that is not finite too, in whole sequences (one segment and several) and in
    single steps alike."""
    for T in (3, 700):
        g = torch.Generator().manual_seed(T)
        q, k, v = (torch.randn(1, T, 2, 24, generator=g).to(dtype) for _ in range(3))
        s = torch.randn(1, 2, 24, 24, generator=g)
        s[0, 0, 3] = bad
        decay = torch.tensor([0.0, 0.5])
        out, last = policy.compute_linear_attention(*(t.cuda() for t in (q, k, v, decay)), None, s.cuda())
        zero = torch.where(decay[None, :, None, None] == 0, 0.0, s)
        want, wlast = policy.compute_linear_attention(*(t.cuda() for t in (q, k, v, decay)), None, zero.cuda())
        assert bool(out.isfinite().all()) and torch.equal(out, want) and torch.equal(last, wlast)
        o, new = policy.compute_linear_attention_step(*(t[:, 0].cuda() for t in (q, k, v)), decay.cuda(), s.cuda())
        wo, wnew = policy.compute_linear_attention_step(*(t[:, 0].cuda() for t in (q, k, v)), decay.cuda(), zero.cuda())
        assert bool(o.isfinite().all()) and torch.equal(o, wo) and torch.equal(new, wnew)


@pytest.mark.parametrize("reverse", [0, 1])
@pytest.mark.parametrize("transposed", [0, 1])
def test_the_c_entry_writes_the_states_of_no_steps(reverse, transposed):
    """The header: empty inputs launch nothing, but for states, which are written."""
    E, H, dk, dv = 3, 2, 5, 7
    state = torch.randn(E, H, dk, dv, device="cuda")
    given = state.transpose(-1, -2).contiguous() if transposed else state
    decay = torch.tensor([0.5, 0.25], device="cuda")
    none = _native.Sequence(None, 0, 0, 0)
    for enters, want in ((given, state * 3), (None, torch.zeros_like(state))):
        out = torch.full_like(state, 7.0)
        call = _native.Attention(none, none, none, none, E, 0, H, dk, dv, decay.data_ptr(), None, None if enters is None else enters.data_ptr(),
                                 transposed, out.data_ptr(), 1.0, 2.0, 1.5, reverse, 0, None, 0)
        assert _native.load().rlk_linear_attention(ctypes.byref(call), 1, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, want)


@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (40, 72)])
def test_states_of_bfloat16_calls_are_float32(dims):
    """A state is sums of products of bfloat16 values with float32 powers of the decay, as exact as float32 sums of them are: the
    root mean square of its error is that of the additions of one chunk's 64 terms and of some 20 chunks, each off by at
    most U32 of a partial sum, with the powers' 24 U32: far below 16 U32 of the largest value, 9.5e-7.  (Weighted terms kept as
    two bfloat16 numbers were off by 2.5e-6 of it, as three by 3e-7.)"""
    E, T, H, (dk, dv) = 2, 1280, 2, dims
    g = torch.Generator().manual_seed(dk)
    q, k, v = (torch.randn(E, T, H, d, generator=g).bfloat16() for d in (dk, dk, dv))
    go, gs = torch.randn(E, T, H, dv, generator=g).bfloat16(), torch.randn(E, H, dk, dv, generator=g)
    s = torch.randn(E, H, dk, dv, generator=g)
    decay = torch.tensor([0.99, 0.999])
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, s)]
    out, last = policy.compute_linear_attention(*leaves[:3], decay.cuda(), None, leaves[3], 0.3)
    got = last, torch.autograd.grad((out, last), leaves, (go.cuda(), gs.cuda()))[3]
    want = attention(q, k, v, decay, None, s, 0.3)[1], attention_grads(q, k, v, decay, None, s, 0.3, go, gs)[3]
    for x, w in zip(got, want):
        for h in range(H):
            err = (x.detach().cpu().double() - w)[:, h].square().mean().sqrt() / w[:, h].abs().max()
            assert float(err) < 16 * U32, float(err)


@pytest.mark.parametrize("E,T,H,dk,dv", [(2, 3, 2, 8, 8), (2, 65, 6, 64, 64), (3, 127, 2, 72, 24), (1, 130, 2, 128, 128), (2, 333, 4, 40, 72),
                                         (1, 1000, 2, 64, 64), (1, 1025, 1, 128, 128), (2, 700, 2, 33, 16)])
def test_outputs_of_bfloat16_calls_are_rounded_once(E, T, H, dk, dv):
    """Outputs and gradients of bfloat16 calls: sums as exact as float32's, of which two factors in each term (the state, the weighted
    product of query and key) are held in two bfloat16 numbers (the upper 8 bits leave less than 2^-7 of a number, 8 bits of that leave
    2^-8 of it: 2^-15), and one rounding to bfloat16 at the end."""
    g = torch.Generator().manual_seed(T)
    q, k, v, go = (torch.randn(E, T, H, d, generator=g).bfloat16() for d in (dk, dk, dv, dv))
    s, gs = torch.randn(E, H, dk, dv, generator=g), torch.randn(E, H, dk, dv, generator=g)
    decay = torch.tensor([0.999, 0.5, 1.0, 0.05, 0.9, 0.0])[:H]
    dones = (torch.rand(E, T, generator=g) < 0.01).float()
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, last = policy.compute_linear_attention(*leaves, decay.cuda(), dones.cuda(), s.cuda(), 0.3)
    got = out, *torch.autograd.grad((out, last), leaves, (go.cuda(), gs.cuda()))
    args, sizes = (q, k, v, decay, dones, s, 0.3), (q.abs(), k.abs(), v.abs(), decay, dones, s.abs(), 0.3)
    want = attention(*args)[0], *attention_grads(*args, go, gs)[:3]
    size = attention(*sizes)[0], *attention_grads(*sizes, go.abs(), gs.abs())[:3]
    for i, (x, w, y) in enumerate(zip(got, want, size)):
        err = (x.detach().cpu().double() - w).abs()
        bound = y * ((T + 128) * U32 + 2.0 ** -15) + U16 * w.abs() + 1e-30
        assert bool((err <= bound).all()), (i, float((err / bound).max()))


def test_a_state_that_is_not_finite_in_bfloat16():
    """An inf that a sequence goes on from is in every output that reads it, until its episode's end, as it is in float32."""
    g = torch.Generator().manual_seed(1)
    for d in (64, 128):
        q, k, v = ((torch.rand(2, 300, 2, d, generator=g) + 0.5).bfloat16() for _ in range(3))
        s = torch.randn(2, 2, d, d, generator=g)
        s[0, 1, 3, 5], s[1, 0, 2, 40], s[1, 0, 7, 41] = math.inf, -math.inf, math.nan
        decay, dones = torch.tensor([0.99, 0.95]), torch.zeros(2, 300)
        dones[:, 200] = 1
        out, last = policy.compute_linear_attention(*(t.cuda() for t in (q, k, v, decay, dones, s)))
        want, wlast = attention(q, k, v, decay, dones, s, d ** -0.5)
        x = out.cpu().double()
        assert torch.equal(x.isnan(), want.isnan()) and torch.equal(x == math.inf, want == math.inf) and torch.equal(x == -math.inf, want == -math.inf)
        assert bool(x[:, 201:].isfinite().all()) and bool(last.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [24, 64, 128])
def test_products_that_a_scale_takes_out_of_range(d, dtype):
    """Queries and keys whose products float32 holds, but not `scale` times them, with values that bring the output back into range: the
    recurrence forms k v first.  (T + 128) u of the sizes, the output's rounding, and in bfloat16 2^-15 of the sizes."""
    g = torch.Generator().manual_seed(d)
    E, T, H = 1, 100, 2
    q, k, v = ((torch.rand(E, T, H, d, generator=g) * 0.5 + 0.5).to(dtype) for _ in range(3))
    q, k, v, scale = q * 2.0 ** 57, k * 2.0 ** 57, v * 2.0 ** -100, 2.0 ** 9 * 128 / d
    decay = torch.tensor([0.9, 1.0])
    out, last = policy.compute_linear_attention(*(t.cuda() for t in (q, k, v, decay)), scale=scale)
    want, wlast = attention(q, k, v, decay, None, None, scale)
    low = dtype == torch.bfloat16
    assert bool(out.isfinite().all())
    err = (out.cpu().double() - want).abs()
    assert bool((err <= want * ((T + 128) * U32 + (2.0 ** -15 + U16 if low else 0))).all()), float((err / want).max())
    assert bool(((last.cpu().double() - wlast).abs() <= (T + 128) * U32 * wlast).all())
