"""The learner's operators (rl_triton.policy) written out in float64, step by step, with the sizes that their
error bounds are taken from."""
import math

import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8  # unit roundoffs: significands of 24 bits (float32) and 8 (bfloat16)
UNIT = {torch.float32: U32, torch.bfloat16: U16}


def softmax_rows(logits, actions, temperature):
    """(log p of the action, entropy, p, log p) in float64; empty rows: -inf, 0, zeros."""
    x = logits.double() / temperature
    top = x.amax(-1, keepdim=True)
    empty = (top == -math.inf).squeeze(-1)
    z = x - torch.where(top == -math.inf, 0.0, top)
    e = z.exp()
    s = e.sum(-1, keepdim=True)
    logp = torch.where(empty[..., None], -math.inf, z - s.log())
    p = torch.where(empty[..., None], 0.0, e / s)
    entropy = -torch.where(p == 0, 0.0, p * logp).sum(-1)
    inside = (actions >= 0) & (actions < logits.shape[-1])
    lp = logp.gather(-1, torch.where(inside, actions, 0)[..., None]).squeeze(-1)
    return torch.where(inside, lp, math.nan), entropy, p, logp


def logits_grad(p, logp, entropy, actions, g, h, temperature):
    """d/d logits of sum g log p_a + h H."""
    d = -g[..., None] * p - torch.where(p == 0, 0.0, h[..., None] * p * (logp + entropy[..., None]))
    at = torch.zeros_like(d).scatter_(-1, actions[..., None], torch.where(p.sum(-1) == 0, 0.0, g)[..., None])
    return (d + at) / temperature


def policy_loss(lp, old, adv, ref, mask, clip_low, clip_high, dual_clip, kl_coef, reduction):
    """(loss, d loss / d lp, means, weights) in float64, by a loop-free transcription of the definition."""
    lp, old, adv = lp.double(), old.double(), adv.double()
    kept = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask != 0
    w = torch.zeros_like(lp)
    if reduction == "rows":
        rows = [e for e in range(lp.shape[0]) if bool(kept[e].any())]
        for e in rows:
            w[e] = kept[e].double() / (int(kept[e].sum()) * len(rows))
    elif bool(kept.any()):
        w = kept.double() / int(kept.sum())
    d = lp - old
    r = d.exp()
    a, b = -adv * r, -adv * r.clamp(1 - clip_low, 1 + clip_high)
    pg = torch.maximum(a, b)
    flat = b > a
    if dual_clip is not None:
        cap = (adv < 0) & (pg > -adv * dual_clip)
        pg, flat = torch.where(cap, -adv * dual_clip, pg), flat | cap
    slope = torch.where(flat, 0.0, -adv * r)
    kl = torch.zeros_like(lp)
    if ref is not None:
        e = ref.double() - lp
        kl = torch.expm1(e) - e
        slope = slope - kl_coef * torch.expm1(e)
    terms = [pg, kl, flat.double(), torch.expm1(d) - d]
    means = torch.stack([torch.where(kept, w * t, 0.0).sum() for t in terms])
    sizes = torch.stack([torch.where(kept, w * t.abs(), 0.0).sum() for t in terms])
    return means[0] + kl_coef * means[1], torch.where(kept, w * slope, 0.0), means, sizes, w


def recurrence(a, b, c, decay, cut, state, reverse=False):
    """y_t = S_t^T a_t, S_t = decay (1 - cut_t) S_{t-1} + b_t c_t^T: (y, last S), [E, T, H, dim]."""
    E, T, H, _ = a.shape
    S = torch.zeros(E, H, b.shape[-1], c.shape[-1], dtype=torch.float64) if state is None else state.double()
    y = torch.zeros(E, T, H, c.shape[-1], dtype=torch.float64)
    first = True
    for t in reversed(range(T)) if reverse else range(T):
        lam = decay[None, :].expand(E, H) if not (reverse and first) else torch.ones(E, H, dtype=torch.float64)
        lam = torch.where(cut[:, t, None] != 0, 0.0, lam)
        S = torch.where(lam[..., None, None] == 0, 0.0, S * lam[..., None, None]) + b[:, t, :, :, None] * c[:, t, :, None, :]
        y[:, t] = (a[:, t, :, :, None] * S).sum(-2)
        first = False
    return y, S


def attention(q, k, v, decay, dones, state, scale):
    q, k, v, decay = q.double(), k.double(), v.double(), decay.double()
    E, T = q.shape[:2]
    done = torch.zeros(E, T) if dones is None else (dones != 0).float()
    cut = torch.cat([torch.zeros(E, 1), done[:, :-1]], 1)
    y, S = recurrence(q, k, v, decay, cut, state)
    return y * scale, S * (1 - done[:, -1].double())[:, None, None, None]


def attention_grads(q, k, v, decay, dones, state, scale, g, g_last):
    """Gradients of q, k, v and state for upstream gradients of both results."""
    q, k, v, decay, g = q.double(), k.double(), v.double(), decay.double(), g.double()
    E, T = q.shape[:2]
    done = torch.zeros(E, T) if dones is None else (dones != 0).float()
    cut = torch.cat([torch.zeros(E, 1), done[:, :-1]], 1)
    dq = recurrence(g, v, k, decay, cut, None if state is None else state.transpose(-1, -2))[0] * scale
    last = None if g_last is None else g_last.double() / scale
    dk = recurrence(v, g, q, decay, done, None if last is None else last.transpose(-1, -2), reverse=True)[0] * scale
    dv, R = recurrence(k, q, g, decay, done, last, reverse=True)
    return dq, dk, dv * scale, R * decay[None, :, None, None] * scale
