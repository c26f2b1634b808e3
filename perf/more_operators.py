"""A policy's operators between its projections and its actions, as cases that can be timed and compared.

A case is one pass of a user's program through one operator of rl_triton.policy:

  op       "sample"        actions drawn from logits [envs, steps, actions] by given uniform numbers, truncated to the likeliest
           "norms"         queries and keys [envs, steps, heads, dim] normed head by head and rotated by their positions
           "norms_train"   the same, forward and backward
           "delta"         the gated delta rule over whole sequences [envs, steps, heads, dim]
           "delta_train"   the same, forward and backward
           "delta_step"    one step of it for every environment, its state read and written
  dtype    of the logits, or of queries, keys and values

The plain forms are the formulas in elementary torch operations, computed in 32 bits; in 64 where 32 lose what matters (angles of far
positions; sums of probabilities, next to which a uniform number falls).
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
TEMPERATURE, BASE, EPS = 0.9, 10000.0, 1e-6


def _api():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rl-triton_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rl_triton.policy
    return rl_triton.policy


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def _sample(envs, steps, actions, dtype="float32", invalid=False, top_k=None, top_p=None, min_p=None):
    """invalid: some actions are not allowed (logits of -inf)."""
    return {"op": "sample", "envs": envs, "steps": steps, "actions": actions, "dtype": dtype, "invalid": invalid, "top_k": top_k,
            "top_p": top_p, "min_p": min_p}


def _norms(op, envs, steps, heads, key_heads, dim, dtype="bfloat16", rotary=None, far=0):
    """rotary: how many of the dims are rotated (all).  far: the largest position that an environment has reached before the window."""
    return {"op": op, "envs": envs, "steps": steps, "heads": heads, "key_heads": key_heads, "dim": dim, "dtype": dtype,
            "rotary": dim if rotary is None else rotary, "far": far}


def _delta(op, envs, steps, heads, dim_k, dim_v, dtype="bfloat16", ends=0.0, state=False):
    """ends: the share of steps that end an episode.  state: the sequences go on from an earlier window."""
    return {"op": op, "envs": envs, "steps": steps, "heads": heads, "dim_k": dim_k, "dim_v": dim_v, "dtype": dtype, "ends": ends,
            "state": state}


def listed():
    return [
        # one acting step of a vectorised simulator, some buttons not allowed: latency
        dict(_sample(256, 1, 18, invalid=True), name="sample_acting"),
        # the next token of some responses, with every truncation that a sampler is asked for
        dict(_sample(64, 1, 131072, dtype="bfloat16", top_k=50, top_p=0.95, min_p=0.02), name="sample_tokens"),
        # the next token of many responses, the likeliest nine tenths, an odd vocabulary
        dict(_sample(512, 1, 50001, top_p=0.9), name="sample_nucleus"),
        # one acting step of a policy with a memory
        dict(_norms("norms", 512, 1, 16, 16, 128, far=100000), name="norms_acting"),
        # one long history taken in at once, keys shared by groups of heads
        dict(_norms("norms", 1, 16384, 16, 4, 128), name="norms_history"),
        # an update on the rollouts of a vectorised simulator
        dict(_norms("norms_train", 64, 1024, 8, 8, 64, far=1000), name="norms_train_rollout"),
        # odd lengths and head sizes in 32 bits, rotated in part
        dict(_norms("norms_train", 37, 333, 4, 2, 72, dtype="float32", rotary=40, far=1000000), name="norms_train_ragged"),
        # one acting step of a policy with a memory, few environments: latency
        dict(_delta("delta_step", 8, 1, 4, 64, 64, ends=0.01), name="delta_step_few"),
        # the same for many environments
        dict(_delta("delta_step", 512, 1, 16, 128, 128, ends=0.01), name="delta_step_many"),
        # one long history taken in at once
        dict(_delta("delta", 1, 16384, 16, 128, 128), name="delta_history"),
        # an update of a policy with a memory on the rollouts of a vectorised simulator
        dict(_delta("delta_train", 64, 1024, 8, 64, 64, ends=0.005, state=True), name="delta_train_rollout"),
        # odd lengths and head sizes in 32 bits
        dict(_delta("delta_train", 37, 333, 4, 40, 72, dtype="float32", ends=0.01, state=True), name="delta_train_ragged"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, uniform over the logarithm; round ones are as likely as odd ones."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 16:
        n = n // 16 * 16
    return max(lo, min(hi, n))


def draw(rng):
    """Few actions and many environments, or a vocabulary and some responses; sequences of one step to long histories."""
    op = rng.choice(("sample", "norms", "norms_train", "delta", "delta_train", "delta_step"))
    dtype = rng.choice(("float32", "bfloat16"))
    while True:
        if op == "sample":
            few = rng.random() < 0.5
            actions = _spread(rng, 2, 256) if few else _spread(rng, 256, 131072)
            c = _sample(_spread(rng, 1, 4096 if few else 512), _spread(rng, 1, 16) if few else 1, actions, dtype=dtype,
                        invalid=few and rng.random() < 0.5, top_k=rng.choice((None, None, 1, 7, 50, 400)),
                        top_p=rng.choice((None, 0.5, 0.9, 0.95, 0.99)), min_p=rng.choice((None, None, 0.01, 0.1)))
        elif op.startswith("norms"):
            dim, heads = rng.choice((16, 32, 40, 64, 72, 96, 128)), rng.choice((1, 2, 4, 8, 16))
            c = _norms(op, _spread(rng, 1, 512), _spread(rng, 1, 16384 if op == "norms" else 2048), heads, rng.choice((1, heads)), dim, dtype=dtype,
                       rotary=rng.choice((dim, dim // 2)), far=rng.choice((0, 1000, 1000000)))
        else:
            steps = 1 if op == "delta_step" else _spread(rng, 1, 16384) if op == "delta" else _spread(rng, 1, 2048)
            dims = (16, 24, 32, 40, 64, 72, 96, 100, 128)
            c = _delta(op, _spread(rng, 1, 512), steps, rng.choice((1, 2, 4, 8, 16)), rng.choice(dims), rng.choice(dims), dtype=dtype,
                       ends=rng.choice((0.0, 0.005, 0.05)), state=rng.random() < 0.5)
        # no more than the largest listed case of the kind
        if all(work(c)[k] <= max(work(l)[k] for l in listed() if l["op"] == op) for k in ("bytes", "flops")):
            return c


def work(case):
    n, size = case["envs"] * case["steps"], 4 if case["dtype"] == "float32" else 2
    op = case["op"]
    if op == "sample":  # logits and a uniform number in, an action and its log-probability out.  A difference, an exp, a sum and a comparison
        return {"bytes": n * (case["actions"] * size + 4 + 8 + 4), "flops": 6 * n * case["actions"]}
    if op.startswith("norms"):
        rows = n * (case["heads"] + case["key_heads"])
        train = op == "norms_train"  # in and out; back: the outputs' gradients in, the inputs' out
        return {"bytes": rows * case["dim"] * size * (4 if train else 2) + n * 8 + 8 * case["dim"] * (2 if train else 1),
                "flops": rows * case["dim"] * (22 if train else 7)}
    dk, dv = case["dim_k"], case["dim_v"]
    rows, tokens = case["envs"] * case["heads"], n * case["heads"]
    state = 4 * rows * dk * dv
    if op == "delta_step":
        return {"bytes": 2 * state + tokens * (size * 2 * (dk + dv) + 8), "flops": rows * 7 * dk * dv}
    if op == "delta":  # what a key reads from the state, what is written there, what a query reads: three products, each a multiplication and a sum
        return {"bytes": tokens * (size * 2 * (dk + dv) + 8) + (1 + case["state"]) * state, "flops": 7 * tokens * dk * dv}
    # backward: the state's gradient and its two readings, the state once more, what is read from it for the gradients of q and k, the decay's sum
    return {"bytes": tokens * (size * 4 * (dk + dv) + 16) + (1 + case["state"]) * state, "flops": 24 * tokens * dk * dv}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    op, E, T = case["op"], case["envs"], case["steps"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    s = {"case": case}
    if op == "sample":
        A = case["actions"]
        # a policy that has learned something: a few actions stand out, more of a vocabulary's
        logits = normal(E, T, A, scale=2.0)
        if A > 256:
            logits = logits + 8.0 * (uniform(E, T, A) < 20.0 / A)
        if case["invalid"]:
            logits[uniform(E, T, A) < 0.2] = -math.inf
            logits[..., 0] = normal(E, T)  # there is always one that is allowed
        s["logits"], s["uniforms"] = logits.to(dt), uniform(E, T)
    elif op.startswith("norms"):
        H, K, d = case["heads"], case["key_heads"], case["dim"]
        shape = (E,) if op == "norms" and T == 1 else (E, T)
        # slices of a joint projection
        joint = normal(*shape, H + K, d, scale=1.5).to(dt)
        s["q"], s["k"] = joint[..., :H, :], joint[..., H:, :]
        s["q_weight"], s["k_weight"] = 1 + normal(d, scale=0.1), 1 + normal(d, scale=0.1)
        start = (uniform(E, 1) * (case["far"] + 1)).long()
        s["positions"] = (start + torch.arange(T, device="cuda")).view(shape)
        if op == "norms_train":
            s["q"], s["k"] = s["q"].contiguous(), s["k"].contiguous()
            s["grad_q"], s["grad_k"] = normal(*shape, H, d).to(dt), normal(*shape, K, d).to(dt)
            for name in ("q", "k", "q_weight", "k_weight"):
                s[name].requires_grad_()
    else:
        H, dk, dv = case["heads"], case["dim_k"], case["dim_v"]
        shape = (E, H) if op == "delta_step" else (E, T, H)
        # keys and queries of length 1, as the rule wants them; a policy's steps resemble each other
        common = normal(E, *(1,) * (len(shape) - 1), dk, scale=0.5)
        for name in "qk":
            x = normal(*shape, dk) + common
            s[name] = (x / x.square().sum(-1, keepdim=True).sqrt()).to(dt)
        s["v"] = normal(*shape, dv).to(dt)
        # heads that forget within some steps to some thousand, more or less of it at each step
        rate = torch.exp2(-torch.linspace(1, 11, H, device="cuda"))
        s["log_decays"] = -rate * torch.log1p(torch.exp(normal(*shape)))
        s["betas"] = torch.sigmoid(normal(*shape))
        s["scale"] = 1.0
        s["dones"] = (uniform(*shape[:-1]) < case["ends"]).float() if case["ends"] else None
        s["state"] = normal(E, H, dk, dv, scale=0.5) if case["state"] or op == "delta_step" else None
        if op == "delta_train":
            s["grad_out"] = normal(*shape, dv).to(dt)
            for name in _LEAVES:
                s[name].requires_grad_()
    return s


_LEAVES = ("q", "k", "v", "log_decays", "betas")


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    return _OWN[op](state, _api()) if own else _PLAIN[op](state)


def _own_sample(s, api):
    c = s["case"]
    return api.compute_sampled_actions(s["logits"], s["uniforms"], TEMPERATURE, top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"])


def _own_norms(s, api):
    return api.compute_query_key_norms(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], base=BASE,
                                       rotary_dim=s["case"]["rotary"], eps=EPS)


def _own_norms_train(s, api):
    q, k = _own_norms(s, api)
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"], s["q_weight"], s["k_weight"]), (s["grad_q"], s["grad_k"])))


def _own_delta(s, api):
    return api.compute_gated_delta_rule(s["q"], s["k"], s["v"], s["log_decays"], s["betas"], s["dones"], s["state"], s["scale"])


def _own_delta_train(s, api):
    out, state = _own_delta(s, api)
    return (out.detach(), state.detach(), *torch.autograd.grad(out, [s[n] for n in _LEAVES], s["grad_out"]))


def _own_delta_step(s, api):
    return api.compute_gated_delta_rule_step(s["q"], s["k"], s["v"], s["log_decays"], s["betas"], s["state"], s["dones"], s["scale"])


_OWN = {"sample": _own_sample, "norms": _own_norms, "norms_train": _own_norms_train, "delta": _own_delta, "delta_train": _own_delta_train,
        "delta_step": _own_delta_step}


def _plain_sample(s):
    """The likeliest actions, as many as the truncations leave, and of these the first whose probabilities add up to more than the uniform
    number's share.  In 64 bits: a border lies somewhere between two of a hundred thousand sums."""
    c, x = s["case"], s["logits"]
    A = x.shape[-1]
    z = (x.double() - x.double().amax(-1, keepdim=True)) / TEMPERATURE
    w = torch.exp(z)
    if c["top_k"] is not None or c["top_p"] is not None:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices  # (of equal ones the first)
        ranked = w.gather(-1, order)
        if c["top_k"] is not None:
            ranked[..., c["top_k"]:] = 0.0
        if c["top_p"] is not None:
            before = ranked.cumsum(-1) - ranked
            ranked = torch.where(before < c["top_p"] * ranked.sum(-1, keepdim=True), ranked, 0.0)
        w = torch.zeros_like(w).scatter_(-1, order, ranked)
    if c["min_p"] is not None:
        w = torch.where(w >= c["min_p"], w, 0.0)
    sums = w.cumsum(-1)
    total = sums[..., -1:]
    beyond = sums > s["uniforms"].double()[..., None] * total
    actions = torch.where(beyond, torch.arange(A, device=x.device), A).amin(-1).clamp_max(A - 1)
    return actions, (torch.log(w.gather(-1, actions[..., None])) - torch.log(total)).squeeze(-1).float()


def _angles(positions, rotary):
    i = torch.arange(rotary // 2, dtype=torch.float64, device=positions.device)
    a = positions.double()[..., None, None] * BASE ** (-2.0 * i / rotary)
    return torch.cos(a), torch.sin(a)


def _rotated(x, cos, sin):
    h = cos.shape[-1]
    a, b, rest = x[..., :h], x[..., h:2 * h], x[..., 2 * h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_normed(x, weight, cos, sin):
    x = x.float()
    return _rotated(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight, cos, sin)


def _plain_norms(s):
    cos, sin = (x.float() for x in _angles(s["positions"], s["case"]["rotary"]))
    return tuple(_plain_normed(s[n], s[n + "_weight"], cos, sin).to(s[n].dtype) for n in "qk")


def _plain_norms_train(s):
    cos, sin = (x.float() for x in _angles(s["positions"], s["case"]["rotary"]))
    x = [s[n].detach().float().requires_grad_() for n in ("q", "k", "q_weight", "k_weight")]
    outs = [_plain_normed(x[i], x[2 + i], cos, sin) for i in range(2)]
    grads = torch.autograd.grad(outs, x, (s["grad_q"].float(), s["grad_k"].float()))
    dt = s["q"].dtype
    return (*(o.detach().to(dt) for o in outs), grads[0].to(dt), grads[1].to(dt), *grads[2:])


_CHUNK = 64


def _unit_lower_inverse(a):
    """(1 + a)^-1 for strictly lower triangular a: blocks of 1, 2, 4, ... from the blocks of half the size."""
    C = a.shape[-1]
    lead, size, x = a.shape[:-2], 1, torch.ones(*a.shape[:-2], C, 1, 1, device=a.device)
    while size < C:
        n = C // (2 * size)
        i = torch.arange(n, device=a.device)
        low = a.view(*lead, n, 2 * size, n, 2 * size).movedim(-2, -4)[..., i, i, :, :] if n > 1 else a.unsqueeze(-3)
        low = low[..., size:, :size]
        first, second = x[..., 0::2, :, :], x[..., 1::2, :, :]
        below = -(second @ (low @ first))
        x = torch.cat([torch.cat([first, torch.zeros_like(first)], -1), torch.cat([below, second], -1)], -2)
        size *= 2
    return x.squeeze(-3)


def _chunked_delta(q, k, v, log_decays, betas, dones, state, scale):
    """Chunks of steps at once: a chunk's corrections are a triangular system of its keys, solved for all chunks; then the states, one
    after the other."""
    E, T, H, dk = q.shape
    C = _CHUNK
    N = -(-T // C)
    pad = N * C - T
    dev = q.device

    def chunks(x):  # [E, T, H, ...] -> [E, H, N, C, ...]
        x = torch.cat([x, x.new_zeros(E, pad, *x.shape[2:])], 1) if pad else x
        return x.reshape(E, N, C, *x.shape[2:]).movedim(3, 1).contiguous()

    q, k, v, g, beta = chunks(q * scale), chunks(k), chunks(v), chunks(log_decays), chunks(betas)[..., None]
    done = torch.zeros(E, N * C, device=dev)
    if dones is not None:
        done[:, :T] = (dones != 0).float()
    before = (done.cumsum(1) - done).view(E, 1, N, C)  # episodes that have ended before each step
    first = before[..., :1].clone()
    first[:, :, 1:, 0] -= done.view(E, 1, N, C)[:, :, :-1, -1]  # ... before the chunk's state was made
    last = before[..., -1:]
    G = g.cumsum(-1)
    i = torch.arange(C, device=dev)
    seen = (i[:, None] >= i) & (before[..., :, None] == before[..., None, :])
    among = torch.where(seen, torch.exp(torch.where(seen, G[..., :, None] - G[..., None, :], 0.0)), 0.0)  # [E, H, N, C, C]
    back = torch.exp(G)[..., None] * (before == first)[..., None]
    into = torch.exp(G[..., -1:] - G)[..., None] * (before == last)[..., None]
    keep = torch.exp(G[..., -1:])[..., None] * (last == first)[..., None]
    resemble = (k @ k.transpose(-1, -2)) * among * (i[:, None] > i)
    solve = _unit_lower_inverse(beta * resemble)
    read = (q @ k.transpose(-1, -2)) * among
    from_keys, from_queries, to_state = k * back, q * back, (k * into).transpose(-1, -2)
    S = torch.zeros(E, H, dk, v.shape[-1], device=dev) if state is None else state
    outs = []
    for n in range(N):
        u = solve[:, :, n] @ (beta[:, :, n] * (v[:, :, n] - from_keys[:, :, n] @ S))
        outs.append(from_queries[:, :, n] @ S + read[:, :, n] @ u)
        S = keep[:, :, n] * S + to_state[:, :, n] @ u
    out = torch.stack(outs, 2).movedim(1, 3).reshape(E, N * C, H, v.shape[-1])[:, :T]
    if dones is not None:
        S = S * (dones[:, -1] == 0)[:, None, None, None]
    return out, S


def _plain_delta(s):
    out, state = _chunked_delta(*(s[n].float() for n in _LEAVES), s["dones"], s["state"], s["scale"])
    return out.to(s["v"].dtype), state


def _plain_delta_train(s):
    x = [s[n].detach().float().requires_grad_() for n in _LEAVES]
    out, state = _chunked_delta(*x, s["dones"], s["state"], s["scale"])
    grads = torch.autograd.grad(out, x, s["grad_out"].float())
    dt = s["q"].dtype
    return (out.detach().to(dt), state.detach(), *(g.to(dt) for g in grads[:3]), *grads[3:])


def _plain_delta_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    lam = torch.exp(s["log_decays"])
    if s["dones"] is not None:
        lam = torch.where(s["dones"][:, None] != 0, 0.0, lam)
    state = s["state"] * lam[..., None, None]
    u = s["betas"][..., None] * (v - (k[..., :, None] * state).sum(-2))
    state = state + k[..., :, None] * u[..., None, :]
    return ((q * s["scale"])[..., :, None] * state).sum(-2).to(s["v"].dtype), state


_PLAIN = {"sample": _plain_sample, "norms": _plain_norms, "norms_train": _plain_norms_train, "delta": _plain_delta,
          "delta_train": _plain_delta_train, "delta_step": _plain_delta_step}


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["op"]](s)


def _exact_sample(s):
    """Row by row as it is said: an action is kept while fewer than top_k come before it, those hold less than top_p of what top_k leaves, and
    it is at least min_p times as likely as the first."""
    c = s["case"]
    E, T, A = s["logits"].shape
    actions = torch.empty(E * T, dtype=torch.int64, device="cuda")
    log_probs = torch.empty(E * T, dtype=torch.float64, device="cuda")
    rows, u = s["logits"].reshape(-1, A), s["uniforms"].reshape(-1).double()
    at_once = max(1, (1 << 24) // A)
    for lo in range(0, E * T, at_once):
        x = rows[lo:lo + at_once].double() / TEMPERATURE
        p = torch.softmax(x, -1)
        value, place = torch.sort(x, dim=-1, descending=True, stable=True)
        sorted_p = torch.softmax(value, -1)
        kept = torch.ones_like(place, dtype=torch.bool)
        if c["top_k"] is not None:
            kept &= torch.arange(A, device="cuda") < c["top_k"]
        if c["top_p"] is not None:
            q = sorted_p * kept
            q = q / q.sum(-1, keepdim=True)
            kept &= torch.cat([torch.zeros_like(q[:, :1]), q.cumsum(-1)[:, :-1]], -1) < c["top_p"]
        if c["min_p"] is not None:
            kept &= value - value[:, :1] >= math.log(c["min_p"])
        mine = torch.zeros_like(kept).scatter_(1, place, kept)
        p = p * mine
        p = p / p.sum(-1, keepdim=True)
        chosen = (p.cumsum(-1) <= u[lo:lo + at_once, None]).sum(-1).clamp_max(A - 1)
        actions[lo:lo + at_once] = chosen
        log_probs[lo:lo + at_once] = p.gather(-1, chosen[:, None]).squeeze(-1).log()
    return actions.view(E, T), log_probs.view(E, T)


def _turned(x, positions, rotary, sign=1.0):
    """Pairs as complex numbers, multiplied by e^(i angle)."""
    h = rotary // 2
    freq = torch.exp(torch.arange(h, dtype=torch.float64, device="cuda") * (-2.0 * math.log(BASE) / rotary))
    angle = sign * positions.double()[..., None] * freq
    turn = torch.complex(angle.cos(), angle.sin()).unsqueeze(-2)
    y = torch.complex(x[..., :h].contiguous(), x[..., h:rotary].contiguous()) * turn
    return torch.cat([y.real, y.imag, x[..., rotary:]], -1)


def _exact_norms(s, backward=False):
    outs, grads, weights = [], [], []
    r = s["case"]["rotary"]
    for n in "qk":
        x, w = s[n].detach().double(), s[n + "_weight"].detach().double()
        length = (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
        unit = x / length
        outs.append(_turned(unit * w, s["positions"], r))
        if backward:
            g = _turned(s["grad_" + n].double(), s["positions"], r, -1.0)
            weights.append((g * unit).reshape(-1, x.shape[-1]).sum(0))
            g = g * w
            grads.append((g - unit * (g * unit).mean(-1, keepdim=True)) / length)
    return (*outs, *grads, *weights)


def _exact_delta(s, backward=False):
    """Step after step; back: the derivative of each step from the last to the first."""
    q, k, v, g, beta = (s[n].detach().double() for n in _LEAVES)
    E, T, H, dk = q.shape
    scale = s["scale"]
    stays = torch.ones(E, T + 1, dtype=torch.float64, device="cuda")
    if s["dones"] is not None:
        stays[:, 1:] = (s["dones"] == 0).double()
    alpha = g.exp()
    S = torch.zeros(E, H, dk, v.shape[-1], dtype=torch.float64, device="cuda") if s["state"] is None else s["state"].double()
    out = torch.empty(E, T, H, v.shape[-1], dtype=torch.float64, device="cuda")
    decayed = []
    for t in range(T):
        S = S * (alpha[:, t] * (stays[:, t:t + 1] if t else 1.0))[..., None, None]
        if backward:
            decayed.append(S)
        u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None, :] @ S).squeeze(-2))
        S = S + k[:, t, :, :, None] * u[:, :, None, :]
        out[:, t] = scale * (q[:, t, :, None, :] @ S).squeeze(-2)
    outs = [out, S * stays[:, T, None, None, None]]
    if backward:
        grads = [torch.empty_like(x) for x in (q, k, v, g, beta)]
        d = torch.zeros_like(S)
        for t in range(T - 1, -1, -1):
            B, kt, bt, gt = decayed.pop(), k[:, t], beta[:, t, :, None], s["grad_out"][:, t].double()
            e = v[:, t] - (kt[:, :, None, :] @ B).squeeze(-2)
            S = B + kt[..., None] * (bt * e)[:, :, None, :]
            grads[0][:, t] = scale * (S @ gt[..., None]).squeeze(-1)
            d = d + scale * q[:, t, :, :, None] * gt[:, :, None, :]
            du = (kt[:, :, None, :] @ d).squeeze(-2)
            grads[4][:, t] = (du * e).sum(-1)
            grads[2][:, t] = bt * du
            grads[1][:, t] = (d @ (bt * e)[..., None]).squeeze(-1) - (B @ (bt * du)[..., None]).squeeze(-1)
            d = d - kt[..., None] * (bt * du)[:, :, None, :]
            grads[3][:, t] = (d * B).sum((-1, -2))
            d = d * (alpha[:, t] * (stays[:, t:t + 1] if t else 1.0))[..., None, None]
        outs += grads
    return tuple(outs)


def _exact_delta_step(s):
    keep = s["log_decays"].double().exp()
    if s["dones"] is not None:
        keep = keep * (s["dones"] == 0).double()[:, None]
    q, k, v = (s[n].double() for n in "qkv")
    S = s["state"].double() * keep[..., None, None]
    S = S + k[..., None] * (s["betas"].double()[..., None] * (v - (k[..., None, :] @ S).squeeze(-2)))[..., None, :]
    return s["scale"] * (q[..., None, :] @ S).squeeze(-2), S


_EXACT = {"sample": _exact_sample, "norms": _exact_norms, "norms_train": lambda s: _exact_norms(s, backward=True), "delta": _exact_delta,
          "delta_train": lambda s: _exact_delta(s, backward=True), "delta_step": _exact_delta_step}
