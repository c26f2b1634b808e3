"""The boundary of the gated delta rule, the head norms and the sampling of actions: structures, C entries, refusals before any launch."""
import ctypes
import os
import subprocess

import pytest
import torch

import rl_triton.policy as policy
from rl_triton.policy import _native
from test_policy_api_cpu import I64, ROOT, _Gpu


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")


def test_structures(tmp_path):
    structs = {"rlk_delta_rule": _native.DeltaRule, "rlk_delta_rule_gradients": _native.DeltaRuleGradients, "rlk_sampling": _native.Sampling,
               "rlk_head_norms": _native.HeadNorms}
    lines = [f'printf("%d\\n", (int)sizeof({n}));' + "".join(f'printf("%d\\n", (int)offsetof({n}, {f[0]}));' for f in s._fields_)
             for n, s in structs.items()]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rl_triton_policy.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [x for s in structs.values() for x in (ctypes.sizeof(s), *(getattr(s, f[0]).offset for f in s._fields_))]


def test_entries_refuse_without_launching():
    lib = _native.load()
    p = 4096  # never dereferenced
    seq, none = _native.Sequence(p, 0, 0, 0), _native.Sequence(None, 0, 0, 0)
    need = lib.rlk_delta_rule_workspace_bytes(2, 100, 3, 8, 8, 0)
    keep = lib.rlk_delta_rule_saved_bytes(2, 100, 3, 8, 8)
    back = lib.rlk_delta_rule_workspace_bytes(2, 100, 3, 8, 8, 1)
    assert need > 0 and keep > need and back > 0
    delta = lambda **kw: _native.DeltaRule(**{**dict(q=seq, k=seq, v=seq, out=seq, num_envs=2, seq_len=100, heads=3, dim_k=8, dim_v=8, betas=p,  # noqa: E731
                                                     state=p, state_out=p, scale=1.0, workspace=p, workspace_bytes=need), **kw})
    f = lambda **kw: lib.rlk_gated_delta_rule(ctypes.byref(delta(**kw)), None, 0, None)  # noqa: E731
    for bad in (dict(q=none), dict(k=_native.Sequence(p + 2, 0, 0, 0)), dict(out=none), dict(betas=None), dict(dim_k=0), dict(dim_v=129), dict(num_envs=-1),
                dict(heads=-1), dict(seq_len=-1), dict(scale=float("nan")), dict(heads=1 << 23), dict(seq_len=1 << 31), dict(seq_len=1 << 28, heads=64)):
        assert f(**bad) == -1, bad
    for bad in (dict(workspace=None), dict(workspace_bytes=need - 1), dict(workspace=p + 8)):
        assert f(**bad) == -2, bad
    assert lib.rlk_gated_delta_rule(ctypes.byref(delta()), p, keep - 1, None) == -2
    assert f(num_envs=0) == 0 and lib.rlk_gated_delta_rule(None, None, 0, None) == -1
    grads = _native.DeltaRuleGradients(seq, seq, seq, seq, None, None, None, None)
    b = lambda g=grads, n=keep, **kw: lib.rlk_gated_delta_rule_backward(ctypes.byref(delta(**{**dict(workspace_bytes=back), **kw})), ctypes.byref(g), p, n, None)  # noqa: E731
    assert b(n=keep - 1) == -2 and b(workspace_bytes=back - 1) == -2 and b(k=none) == -1
    assert b(_native.DeltaRuleGradients(none, seq, seq, seq, None, None, None, None)) == -1
    assert b(_native.DeltaRuleGradients(seq, _native.Sequence(p + 2, 0, 0, 0), seq, seq, None, None, None, None)) == -1
    step = lambda **kw: lib.rlk_gated_delta_rule_step(ctypes.byref(delta(**kw)), None)  # noqa: E731
    assert step(state=None) == -1 and step(state_out=None) == -1 and step(betas=None) == -1 and step(num_envs=0) == 0
    # memory stays bounded by environments that go one set after the other
    assert lib.rlk_delta_rule_workspace_bytes(1 << 20, 1024, 8, 128, 128, 1) < 16 << 30
    assert lib.rlk_delta_rule_workspace_bytes(1, 100, 1, 129, 8, 0) == 0 and lib.rlk_delta_rule_saved_bytes(0, 100, 1, 8, 8) == 0

    samp = lambda **kw: lib.rlk_sample_actions(ctypes.byref(_native.Sampling(**{**dict(  # noqa: E731
        logits=p, num_envs=2, seq_len=3, num_actions=5, env_stride=15, step_stride=5, uniforms=p, temperature=1.0, top_p=1.0, actions=p, log_probs=p), **kw})), None)
    for bad in (dict(logits=None), dict(uniforms=None), dict(actions=None), dict(log_probs=None), dict(num_actions=0), dict(num_actions=(1 << 20) + 1),
                dict(num_envs=-1), dict(temperature=0.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5),
                dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=2.0), dict(logits=p + 2), dict(logits=p + 1, bf16=1)):
        assert samp(**bad) == -1, bad
    assert samp(num_envs=0, logits=None) == 0 and lib.rlk_sample_actions(None, None) == -1

    base = dict(q=seq, k=seq, q_out=seq, k_out=seq, num_envs=2, seq_len=3, q_heads=4, k_heads=2, dim=8, rotary_dim=8, positions=p, base=1e4, eps=1e-6)
    norm = lambda **kw: lib.rlk_query_key_norms(ctypes.byref(_native.HeadNorms(**{**base, **kw})), None)  # noqa: E731
    for bad in (dict(q=none), dict(k=none), dict(q_out=none), dict(dim=0), dict(dim=257), dict(rotary_dim=7), dict(rotary_dim=10), dict(base=0.0),
                dict(base=float("inf")), dict(eps=-1.0), dict(eps=float("nan")), dict(q_heads=-1), dict(q_heads=1 << 17), dict(q=_native.Sequence(p + 2, 0, 0, 0))):
        assert norm(**bad) == -1, bad
    assert norm(num_envs=0) == 0 and norm(q_heads=0, k_heads=0) == 0
    call = _native.HeadNorms(**base)
    need = lib.rlk_head_norms_workspace_bytes(ctypes.byref(call))
    for ws, n, want in ((None, need, -2), (p, need - 1, -2), (p + 2, need, -2)):
        assert lib.rlk_query_key_norms_backward(ctypes.byref(call), seq, seq, p, p, ws, n, None) == want


def test_delta_rule_refusals():
    f = policy.compute_gated_delta_rule
    z = torch.zeros(1, 2, 3, 4)
    with pytest.raises(AssertionError, match="q must be on CUDA"):
        f(z, z, z, None, torch.zeros(1, 2, 3))
    x, b = _Gpu(1, 2, 3, 4), _Gpu(1, 2, 3)
    for args, match in (((_Gpu(1, 2, 3), x, x, b, b), "q must be"), ((x, _Gpu(1, 2, 3, 5), x, b, b), "k shape"), ((x, x, _Gpu(1, 2, 2, 4), b, b), "v shape"),
                        ((_Gpu(1, 2, 3, 4, dtype=torch.float16), x, x, b, b), "float32 or bfloat16"), ((x, x, _Gpu(1, 2, 3, 129), b, b), "head dimensions"),
                        ((x, x, x, _Gpu(1, 2), b), "log_decays shape"), ((x, x, x, b, _Gpu(3)), "betas shape"),
                        ((x, x, x, _Gpu(1, 2, 3, dtype=torch.bfloat16), b), "log_decays must be float32"), ((x, x, x, b, _Gpu(1, 2, 3, device=1)), "betas must be"),
                        ((x, x, x, b, b, _Gpu(1, 3)), "dones shape"), ((x, x, x, b, b, None, _Gpu(1, 3, 4, 5)), "state must have shape"),
                        ((x, x, x, b, b, None, None, float("nan")), "scale"), ((x, x, x, b, b, None, None, "1"), "scale")):
        with pytest.raises(AssertionError, match=match):
            f(*args)
    many = [_Gpu(1, 1 << 24, 64, 4)] * 3 + [_Gpu(1, 1 << 24, 64)] * 2
    with pytest.raises(AssertionError, match="heads times chunks"):
        f(*many)
    g, y, c = policy.compute_gated_delta_rule_step, _Gpu(1, 3, 4), _Gpu(1, 3)
    with pytest.raises(AssertionError, match="state is required"):
        g(y, y, y, c, c, None)
    with pytest.raises(AssertionError, match="q must be"):
        g(x, x, x, c, c, _Gpu(1, 3, 4, 4))
    with pytest.raises(AssertionError, match="betas shape"):
        g(y, y, y, c, b, _Gpu(1, 3, 4, 4))


def test_sampling_refusals():
    f = policy.compute_sampled_actions
    with pytest.raises(AssertionError, match="logits must be on CUDA"):
        f(torch.zeros(2, 4), torch.zeros(2))
    x, u = _Gpu(2, 3, 4), _Gpu(2, 3)
    for args, kw, match in (((_Gpu(2, 3, 4, dtype=torch.float16), u), {}, "float32 or bfloat16"), ((_Gpu(2, 3, 0), u), {}, "action axis"),
                            ((_Gpu(2, 3, (1 << 20) + 1), u), {}, "action axis"), ((x, _Gpu(2, 3, dtype=torch.float64)), {}, "uniforms: expected"),
                            ((x, _Gpu(2, 3, 1)), {}, "uniforms shape"), ((x, _Gpu(2, 3, device=1)), {}, "uniforms must be on"), ((x, u, 0.0), {}, "temperature"),
                            ((x, u), dict(top_k=0), "top_k"), ((x, u), dict(top_k=2.0), "top_k"), ((x, u), dict(top_k=True), "top_k"), ((x, u), dict(top_p=0.0), "top_p"),
                            ((x, u), dict(top_p=1.1), "top_p"), ((x, u), dict(top_p=float("nan")), "top_p"), ((x, u), dict(min_p=-0.1), "min_p"),
                            ((x, u), dict(min_p=1.5), "min_p"), ((x, u), dict(min_p="a"), "min_p")):
        with pytest.raises(AssertionError, match=match):
            f(*args, **kw)


def test_head_norms_refusals():
    f = policy.compute_query_key_norms
    z = torch.zeros(1, 2, 3, 4)
    with pytest.raises(AssertionError, match="q must be on CUDA"):
        f(z, z)
    x, p = _Gpu(1, 2, 3, 4), _Gpu(1, 2, dtype=I64)
    for args, kw, match in (((_Gpu(2, 3), x), {}, "q must be"), ((x, _Gpu(1, 2, 3, 8)), {}, "k shape"), ((x, _Gpu(1, 3, 3, 4)), {}, "k shape"),
                            ((x, _Gpu(1, 2, 3, 4, dtype=torch.bfloat16)), {}, "k: expected"), ((x, _Gpu(1, 2, 3, 4, device=1)), {}, "k must be on"),
                            ((_Gpu(1, 2, 3, 257), _Gpu(1, 2, 3, 257)), {}, "head dimensions"), ((x, x, _Gpu(5)), {}, "q_weight must have shape"),
                            ((x, x, None, _Gpu(4, dtype=torch.bfloat16)), {}, "k_weight must be float32"), ((x, x, None, None, _Gpu(1, 2)), {}, "positions: expected"),
                            ((x, x, None, None, _Gpu(2, dtype=I64)), {}, "positions shape"), ((x, x, None, None, p), dict(rotary_dim=3), "rotary_dim"),
                            ((x, x, None, None, p), dict(rotary_dim=6), "rotary_dim"), ((_Gpu(1, 2, 3, 5), _Gpu(1, 2, 3, 5), None, None, p), {}, "rotary_dim"),
                            ((x, x, None, None, p), dict(base=0), "base"), ((x, x, None, None, p), dict(eps=-1e-6), "eps"), ((x, x), dict(eps=float("nan")), "eps")):
        with pytest.raises(AssertionError, match=match):
            f(*args, **kw)


def test_head_norms_workspace_serves_either_side_alone():
    """A backward call with the gradient of one output has fewer blocks of heads, so more workgroups along the steps."""
    lib = _native.load()
    size = lambda q, k: lib.rlk_head_norms_workspace_bytes(ctypes.byref(_native.HeadNorms(  # noqa: E731
        q=_native.Sequence(4096, 0, 0, 0), k=_native.Sequence(4096, 0, 0, 0), num_envs=8, seq_len=8192, q_heads=q, k_heads=k, dim=64, base=1e4, eps=1e-6)))
    for q in (1, 2, 3, 5, 64, 4096):
        for k in (0, 1, 2, 7, 4096):
            assert size(q, k) >= max(size(q, 0), size(0, k) if k else 0) > 0
