"""compute_sampled_actions against its definition in float64.

Actions are equal: a uniform number would have to lie within some 1e-13 of a border to come out otherwise, which a float32 number
(a multiple of 2^-24 at the least) does for less than one in a hundred million borders.  Log-probabilities are formed in float64 and rounded
once to float32."""
import math

import pytest
import torch

import rl_triton.policy as policy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


def definition(logits, uniforms, temperature=1.0, top_k=None, top_p=None, min_p=None):
    x = logits.double()
    A = x.shape[-1]
    top = x.amax(-1, keepdim=True)
    z = torch.where(x == top, 0.0, (x - top) / temperature)
    w = z.exp()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ranked = w.gather(-1, order)
    kept = torch.ones_like(ranked, dtype=torch.bool)
    if top_k is not None:
        kept &= torch.arange(A, device=x.device) < top_k
    if top_p is not None:
        r = ranked * kept
        kept &= r.cumsum(-1) - r < top_p * r.sum(-1, keepdim=True)
    if min_p is not None:
        kept &= ranked >= min_p
    w = torch.zeros_like(w).scatter_(-1, order, ranked * kept)
    sums = w.cumsum(-1)
    total = sums[..., -1]
    action = (sums <= (uniforms.double() * total)[..., None]).sum(-1).clamp_max(A - 1)
    log_prob = z.gather(-1, action[..., None]).squeeze(-1) - total.log()
    empty = (top == -math.inf).squeeze(-1)
    nan = x.isnan().any(-1)
    action = torch.where(empty | nan, -1, action)
    return action, torch.where(nan, math.nan, torch.where(empty, -math.inf, log_prob))


def _hold(logits, uniforms, **kw):
    got, want = policy.compute_sampled_actions(logits, uniforms, **kw), definition(logits, uniforms, **kw)
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.float32 and got[0].shape == uniforms.shape
    assert torch.equal(got[0], want[0]), (kw, got[0][got[0] != want[0]][:5], want[0][got[0] != want[0]][:5])
    assert torch.allclose(got[1].double(), want[1], rtol=2.0 ** -24, atol=1e-12, equal_nan=True)
    return got


TRUNCATIONS = [{}, {"top_k": 1}, {"top_k": 7}, {"top_p": 0.9}, {"top_p": 1e-9}, {"min_p": 0.05}, {"min_p": 1.0},
               {"top_k": 50, "top_p": 0.8, "min_p": 0.01, "temperature": 0.7}, {"top_k": 400, "top_p": 0.99}, {"top_p": 0.999, "temperature": 1.5},
               {"top_k": 10 ** 6, "top_p": 1.0, "min_p": 0.0}]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("actions", [1, 2, 3, 16, 17, 32, 33, 64, 65, 127, 500, 1025, 4096, 4097, 16384, 16385, 50001, 131072, 131077])
def test_distributions(actions, dtype):
    """Spread out ones, peaked ones, and ones full of equal logits (bfloat16 and whole numbers)."""
    g = torch.Generator(device="cuda").manual_seed(actions)
    rows = 40 if actions < 1000 else 6
    for kind in ("spread", "peaked", "whole"):
        x = torch.randn(rows, 2, actions, generator=g, device="cuda") * 2
        if kind == "peaked":
            x = x + 12 * (torch.rand(x.shape, generator=g, device="cuda") < 8 / actions)
        elif kind == "whole":
            x = x.round()
        x = x.to(dtype)
        u = torch.rand(rows, 2, generator=g, device="cuda")
        for kw in TRUNCATIONS:
            _hold(x, u, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("actions", [5, 64, 700, 20000])
def test_edges(actions, dtype):
    """Equal rows, masked actions, rows of nothing, NaN, infinities, the largest and lowest values, and uniform numbers at the ends."""
    g = torch.Generator(device="cuda").manual_seed(actions)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.randn(14, actions, generator=g, device="cuda").to(dtype)
    x[0] = 0.0
    x[1] = low
    x[2] = -math.inf
    x[3, 1:] = -math.inf
    x[4, :-1] = -math.inf
    x[5, actions // 2] = math.nan
    x[6, 2] = math.inf
    x[7, 1::2] = math.inf
    x[8] = high
    x[9, ::3] = low
    x[10] = 1000.0
    x[10, 3] = 1001.0
    x[11, ::2] = -0.0
    x[11, 1::2] = 0.0
    x[12] = -math.inf
    x[12, 1] = math.nan
    x[13, 1:] = x[13, 0] - 60.0  # (below the last bit of the weights)
    for value in (0.0, 0.5, 1.0 - 2.0 ** -24, 2.0 ** -30):
        u = torch.full((14,), value, device="cuda")
        for kw in ({}, {"top_k": 3}, {"top_p": 0.5}, {"min_p": 0.9}, {"top_k": 2, "top_p": 0.7, "min_p": 0.1}):
            _hold(x, u, **kw)
    u = torch.tensor([1.0, 5.0, math.inf, -1.0, -math.inf, math.nan], device="cuda")
    near = torch.tensor([1.0 - 2.0 ** -24] * 3 + [0.0] * 3, device="cuda")
    rows = x[9].expand(6, -1)
    a = policy.compute_sampled_actions(rows, u)
    # (a number of 1 stands for the last action that has a weight)
    b = policy.compute_sampled_actions(rows, near)
    assert torch.equal(a[0][3:], b[0][3:]) and bool((a[0][:3] >= b[0][:3]).all())


@pytest.mark.parametrize("temperature", [1e-38, 1e-3, 0.5, 100.0, 1e38])
def test_temperatures(temperature):
    g = torch.Generator(device="cuda").manual_seed(1)
    for actions in (30, 3001):
        x, u = torch.randn(20, actions, generator=g, device="cuda"), torch.rand(20, generator=g, device="cuda")
        for kw in ({}, {"top_k": 5}, {"top_p": 0.6}):
            _hold(x, u, temperature=temperature, **kw)


def test_an_action_lies_in_its_share():
    """Uniform numbers over a fine grid: each action as often as its probability says."""
    x = torch.randn(9, generator=torch.Generator().manual_seed(2)).cuda()
    n = 1 << 16
    u = (torch.arange(n, device="cuda").float() + 0.5) / n
    a, lp = policy.compute_sampled_actions(x.expand(n, 9), u, 0.8, top_k=6)
    w = torch.exp(x.double() / 0.8)
    w[x.argsort(descending=True)[6:]] = 0.0
    p = w / w.sum()
    assert bool(((torch.bincount(a, minlength=9).double() / n - p).abs() <= 1.0 / n).all())
    assert torch.allclose(lp.double(), p[a].log(), rtol=2.0 ** -23)
    assert bool((a[1:] >= a[:-1]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_and_ranks(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    for actions in (18, 300, 9000):
        x, u = torch.randn(6, 5, actions, generator=g, device="cuda").to(dtype), torch.rand(6, 5, generator=g, device="cuda")
        kw = dict(top_k=20, top_p=0.9)
        want = _hold(x, u, **kw)
        wide = torch.randn(6, 5, actions + 3, device="cuda").to(dtype)
        wide[..., 1:-2] = x
        for y in (x.transpose(0, 1).contiguous().transpose(0, 1), wide[..., 1:-2], torch.stack([x, x], -1)[..., 0]):
            got = policy.compute_sampled_actions(y, u, **kw)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got = policy.compute_sampled_actions(x, u.t().contiguous().t(), **kw)
        assert torch.equal(got[0], want[0])
        for shape in ((30,), (1, 2, 3, 5), ()):
            y, v = (x.reshape(*shape, actions), u.reshape(shape)) if shape else (x[2, 3], u[2, 3])
            got = policy.compute_sampled_actions(y, v, **kw)
            assert torch.equal(got[0], want[0].reshape(shape) if shape else want[0][2, 3])
        same = x[:1, :1].expand(6, 5, actions)  # one row for all
        _hold(same, u, **kw)


def test_log_probs_are_those_of_the_untruncated_policy():
    """Without a truncation they are compute_action_log_probs' (float32 sums: 2^-20 of a log-probability of some units)."""
    x, u = torch.randn(8, 40, 777, device="cuda"), torch.rand(8, 40, device="cuda")
    a, lp = policy.compute_sampled_actions(x, u, 0.9)
    assert torch.allclose(lp, policy.compute_action_log_probs(x, a, 0.9)[0], rtol=0, atol=16 * 2.0 ** -20)


def test_empty_calls():
    for shape in ((0, 4, 10), (4, 0, 10)):
        a, lp = policy.compute_sampled_actions(torch.zeros(shape, device="cuda"), torch.zeros(shape[:2], device="cuda"), top_k=3)
        assert a.shape == shape[:2] and lp.shape == shape[:2]


def test_streams_and_graphs():
    x, u = torch.randn(16, 20000, device="cuda"), torch.rand(16, device="cuda")
    kw = dict(top_k=100, top_p=0.9, min_p=0.01)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = policy.compute_sampled_actions(x, u, **kw)
    side.synchronize()
    assert torch.equal(got[0], definition(x, u, **kw)[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = policy.compute_sampled_actions(x, u, **kw)
    for _ in range(3):
        x.normal_()
        u.uniform_()
        graph.replay()
        want = policy.compute_sampled_actions(x, u, **kw)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(outs[0], definition(x, u, **kw)[0])


def test_many_actions():
    """The most that there may be, nearly all alike, with an uneven row stride."""
    n = 1 << 20
    x = torch.zeros(2, n + 1, device="cuda")[:, :n]
    x[0, 5] = 1.0
    x[1] = torch.randn(n, device="cuda")
    u = torch.tensor([0.75, 0.3], device="cuda")
    for kw in ({}, {"top_p": 0.5}, {"top_k": 1000}, {"top_k": 4000, "top_p": 0.3}):
        _hold(x, u, **kw)


def test_values_are_checked_where_that_is_asked_for(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "1")
    x = torch.zeros(2, 5, device="cuda")
    policy.compute_sampled_actions(x, x[:, 0])
    with pytest.raises(AssertionError, match="uniforms must lie"):
        policy.compute_sampled_actions(x, torch.ones(2, device="cuda"))
