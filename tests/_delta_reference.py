"""The gated delta rule in float64 on the CPU, a step after the other, with its derivative, and what its results are held to.

Roundings.  Keys here have length at most 1 and betas lie in [0, 1], so a step's map of the state, a (1 - b k k^T), has a norm of at most 1: what a
rounding adds is not enlarged later.  A float32 result is the end of a chain of T steps and sums of up to dim + 64 terms, each rounding at most
u = 2^-24 of its term and of either sign: n of them add up to about sqrt(n) u.  A term can be some times the result (a value and what is
already read for it are taken from each other), for which a factor of 8 stands: 8 sqrt(T + dim + 64) u, relative to the array's norm.
(Two bfloat16 numbers for a factor in place of three would be off by 2^-16: 5 times this at T = 128, dim = 64.)
A bfloat16 result is rounded once more, 2^-8 of itself; where only outputs are formed from them, factors are two bfloat16 numbers, 2^-15."""
import math

import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8


def inputs(E, T, H, dk, dv, dtype, seed, ends=0.05, state=True, gates=True, length=1.0):
    g = torch.Generator().manual_seed(seed)

    def n(*shape):
        return torch.randn(shape, generator=g)

    common = 0.5 * n(E, 1, 1, dk)
    q, k = ((n(E, T, H, dk) + common) for _ in range(2))
    # (a rounding to bfloat16 may lengthen a key by 2^-8)
    q, k = ((x * (0.99 * length) / x.norm(dim=-1, keepdim=True)).to(dtype) for x in (q, k))
    v = n(E, T, H, dv).to(dtype)
    rates = torch.tensor([0.01, 1.0, 0.0, 20.0, 0.1])[torch.arange(H) % 5]
    gd = -rates * torch.rand(E, T, H, generator=g) if gates else None
    if gates and T > 3:
        gd[0, T // 2, 0] = -math.inf  # nothing stays
        gd[-1, T // 3, -1] = -200.0
    betas = torch.rand(E, T, H, generator=g)
    betas[:, ::7] = 0.0  # steps that write nothing
    dones = (torch.rand(E, T, generator=g) < ends).float() if ends is not None else None
    s = n(E, H, dk, dv) if state else None
    return q, k, v, gd, betas, dones, s


def rule(q, k, v, g, beta, dones, state, scale, up=None, up_last=None):
    """(out, last) and, for upstream gradients, those of q, k, v, g, beta and the state."""
    q, k, v, beta = (x.double() for x in (q, k, v, beta))
    E, T, H, dk = q.shape
    a = torch.ones(E, T, H, dtype=torch.float64) if g is None else torch.where(g < -104, 0.0, g.double().exp())
    stays = torch.ones(E, T + 1, dtype=torch.float64)
    if dones is not None:
        stays[:, 1:] = (dones == 0).double()
    if T:
        a = a * torch.cat([torch.ones(E, 1, dtype=torch.float64), stays[:, 1:T]], 1)[..., None]
    S = torch.zeros(E, H, dk, v.shape[-1], dtype=torch.float64) if state is None else state.double()
    out, before, err = torch.zeros(v.shape, dtype=torch.float64), [], []
    for t in range(T):
        B = torch.where(a[:, t, :, None, None] == 0, 0.0, S * a[:, t, :, None, None])
        e = v[:, t] - (k[:, t, :, :, None] * B).sum(-2)
        S = B + k[:, t, :, :, None] * (beta[:, t, :, None] * e)[..., None, :]
        out[:, t] = scale * (q[:, t, :, :, None] * S).sum(-2)
        before.append(B), err.append(e)
    last = S * stays[:, T, None, None, None]
    if up is None and up_last is None:
        return out, last
    grads = [torch.zeros_like(x) for x in (q, k, v, beta, beta)]
    d = torch.zeros_like(S) if up_last is None else up_last.double() * stays[:, T, None, None, None]
    for t in range(T - 1, -1, -1):
        B, e, kt, b = before[t], err[t], k[:, t], beta[:, t, :, None]
        gt = torch.zeros_like(out[:, t]) if up is None else up[:, t].double()
        S = B + kt[..., None] * (b * e)[..., None, :]
        grads[0][:, t] = scale * (S * gt[..., None, :]).sum(-1)
        d = d + scale * q[:, t, :, :, None] * gt[..., None, :]
        du = (kt[..., None] * d).sum(-2)
        grads[4][:, t] = (du * e).sum(-1)
        grads[2][:, t] = b * du
        grads[1][:, t] = (d * (b * e)[..., None, :]).sum(-1) - (B * (b * du)[..., None, :]).sum(-1)
        d = d - kt[..., None] * (b * du)[..., None, :]
        grads[3][:, t] = (d * B).sum((-1, -2))
        d = torch.where(a[:, t, :, None, None] == 0, 0.0, d * a[:, t, :, None, None])
    return out, last, (*grads, d)


def relative(T, dim):
    return 8 * math.sqrt(T + dim + 64) * U32


def held(got, want, tol, what="", size=0.0):
    """Float32 results: in the array's norm, and no element off by more than 8 times that of the largest.  `size`: of terms that leave a
    smaller result."""
    got, want = got.detach().cpu().double(), want.double()
    if want.numel() == 0:
        return
    err = got - want
    scale = float(want.norm()) + size
    assert bool(torch.isfinite(got).all()), what
    assert float(err.norm()) <= tol * scale + 1e-30, (what, float(err.norm()) / max(scale, 1e-300), tol)
    assert float(err.abs().max()) <= 8 * tol * (float(want.abs().max()) + size) + 1e-30, what


def held_rounded(got, want, tol, what=""):
    """bfloat16 results: rounded once, and before that as float32 ones are but for factors of two numbers, some terms' sizes together."""
    got, want = got.detach().cpu().double(), want.double()
    if want.numel() == 0:
        return
    assert bool(torch.isfinite(got).all()), what
    slack = (8 * tol + 16 * 2.0 ** -15) * float(want.abs().max()) + 1e-30
    over = (got - want).abs() - U16 * want.abs() * 1.01
    assert float(over.max()) <= slack, (what, float(over.max()) / slack)
