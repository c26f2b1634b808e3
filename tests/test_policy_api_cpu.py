"""The boundary of rl_triton.policy: exported symbols, headers, and refusals, which come before any launch."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import rl_triton.policy as policy
from rl_triton.policy import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "rl_triton_policy.h")


def test_library_exports_every_declared_symbol():
    names = set(re.findall(r"^\s*(?:int|size_t)\s+(rlk_\w+)\s*\(", open(HEADER).read(), re.M))
    lib = _native.load()
    assert names == set(_native.SIGNATURES)
    assert all(hasattr(lib, n) for n in names)


@pytest.mark.parametrize("lang", ["c", "c++"])
def test_header_and_structures(lang, tmp_path):
    """The header is plain C; its structures have the binding's sizes and offsets."""
    structs = {"rlk_action_rows": _native.ActionRows, "rlk_policy_terms": _native.PolicyTerms, "rlk_sequence": _native.Sequence,
               "rlk_attention": _native.Attention}
    lines = [f'printf("%d\\n", (int)sizeof({n}));' + "".join(f'printf("%d\\n", (int)offsetof({n}, {f[0]}));' for f in s._fields_)
             for n, s in structs.items()]
    src = tmp_path / ("t.c" if lang == "c" else "t.cpp")
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rl_triton_policy.h"\nint main(void) {' + "\n".join(lines) +
                   "return 0; }\n")
    cc, std = ("gcc", "-std=c99") if lang == "c" else ("g++", "-std=c++17")
    subprocess.run([cc, std, "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout.split()]
    want = [x for s in structs.values() for x in (ctypes.sizeof(s), *(getattr(s, f[0]).offset for f in s._fields_))]
    assert got == want


def test_entry_points_refuse_without_launching():
    lib = _native.load()
    p = 4096  # never dereferenced
    rows = lambda **kw: _native.ActionRows(**{**dict(logits=p, actions=p, num_envs=2, seq_len=3, num_actions=5, env_stride=15,
                                                     step_stride=5, temperature=1.0, bf16=0), **kw})
    f = lambda r: lib.rlk_action_log_probs(ctypes.byref(r), p, p, None, None)
    for bad in (dict(logits=None), dict(actions=None), dict(num_envs=-1), dict(num_actions=0), dict(temperature=0.0),
                dict(temperature=float("nan")), dict(temperature=float("inf")), dict(logits=p + 2), dict(logits=p + 1, bf16=1)):
        assert f(rows(**bad)) == -1, bad
    assert f(rows(num_envs=0, logits=None)) == 0
    assert lib.rlk_action_log_probs(None, p, p, None, None) == -1
    assert lib.rlk_action_log_probs_backward(ctypes.byref(rows()), p, None, p, p, p, None) == -1
    need = lib.rlk_policy_workspace_bytes(2)
    terms = lambda **kw: _native.PolicyTerms(**{**dict(old_log_probs=p, advantages=p, clip_low=0.2, clip_high=0.2, loss=p, means=p,
                                                       workspace=p, workspace_bytes=need), **kw})
    f = lambda t: lib.rlk_policy_loss(p, 2, 3, ctypes.byref(t), None, None)
    for bad in (dict(old_log_probs=None), dict(advantages=None), dict(clip_low=-0.1), dict(clip_high=float("nan")),
                dict(dual_clip=0.5), dict(loss=None), dict()):  # (the last: no place for the gradient)
        assert f(terms(**bad)) == -1, bad
    for bad in (dict(workspace=None), dict(workspace_bytes=need - 1), dict(workspace=p + 4)):
        assert f(terms(**bad)) == -2, bad
    assert lib.rlk_policy_loss_from_logits(ctypes.byref(rows()), ctypes.byref(terms(bf16=1)), p, None) == -1
    seq = _native.Sequence(p, 0, 0, 0)
    att = lambda **kw: _native.Attention(**{**dict(q=seq, k=seq, v=seq, out=seq, num_envs=1, seq_len=4, heads=1, dim_k=8, dim_v=8,
                                                   decay=p, state=p, scale=1.0, state_scale=1.0, state_out_scale=1.0), **kw})
    none = _native.Sequence(None, 0, 0, 0)
    for bad in (dict(q=none), dict(out=none), dict(decay=None), dict(dim_k=0), dict(dim_v=129), dict(scale=float("inf")),
                dict(seq_len=-1), dict(num_envs=-2), dict(heads=1 << 21)):
        assert lib.rlk_linear_attention(ctypes.byref(att(**bad)), 1, None) == -1, bad
    assert lib.rlk_linear_attention(ctypes.byref(att()), 4, None) == -1
    two = (_native.Attention * 2)(att(), att(heads=2))
    assert lib.rlk_linear_attention(two, 2, None) == -1
    assert lib.rlk_linear_attention(ctypes.byref(att(seq_len=0)), 1, None) == 0
    assert lib.rlk_linear_attention_step(ctypes.byref(att(state=None)), None) == -1
    assert lib.rlk_linear_attention(ctypes.byref(att(seq_len=1 << 16)), 1, None) == -2  # segments without a workspace


class _Gpu:
    """A tensor's attributes, said to be on a GPU."""

    def __init__(self, *shape, dtype=torch.float32, device=0, grad=False):
        self.shape, self.dtype, self.is_cuda, self._device, self.requires_grad = torch.Size(shape), dtype, True, device, grad

    def dim(self):
        return len(self.shape)

    def get_device(self):
        return self._device

    def numel(self):
        return self.shape.numel()


I64 = torch.int64


def test_log_probs_refusals(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    f = policy.compute_action_log_probs
    with pytest.raises(AssertionError, match="logits must be on CUDA"):
        f(torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=I64))
    x, a = _Gpu(2, 3, 4), _Gpu(2, 3, dtype=I64)
    for args, match in (((_Gpu(2, 3, 4, dtype=torch.float16), a), "float32 or bfloat16"), ((_Gpu(2, 3, 0), a), "action axis"),
                        ((x, _Gpu(2, 3)), "int64"), ((x, _Gpu(2, 4, dtype=I64)), "actions shape"),
                        ((x, _Gpu(2, 3, dtype=I64, device=1)), "device"), ((x, a, 0.0), "temperature"),
                        ((x, a, float("nan")), "temperature"), ((x, a, torch.ones(1)), "temperature")):
        with pytest.raises(AssertionError, match=match):
            f(*args)


def test_loss_refusals(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    f = policy.compute_policy_loss
    z = torch.zeros(2, 3)
    with pytest.raises(AssertionError, match="log_probs must be on CUDA"):
        f(z, z, z)
    t = _Gpu(2, 3)
    for args, kw, match in (((_Gpu(2, 3, 1), t, t), {}, "num_envs, seq_len"), ((t, _Gpu(3, 2), t), {}, "old_log_probs shape"),
                            ((t, t, _Gpu(2, 3, dtype=torch.bfloat16)), {}, "advantages: expected"),
                            ((t, t, t, _Gpu(2, 3, device=1)), {}, "ref_log_probs must be on"), ((t, t, t), dict(mask=_Gpu(2)), "mask shape"),
                            ((t, t, t), dict(clip_low=-0.1), "clip_low"), ((t, t, t), dict(clip_high=float("inf")), "clip_high"),
                            ((t, t, t), dict(kl_coef="1"), "kl_coef"), ((t, t, t), dict(dual_clip=1.0), "dual_clip"),
                            ((t, t, t), dict(reduction="mean"), "reduction")):
        with pytest.raises(AssertionError, match=match):
            f(*args, **kw)
    g = policy.compute_policy_loss_from_logits
    x, a = _Gpu(2, 3, 4, dtype=torch.bfloat16), _Gpu(2, 3, dtype=I64)
    for args, kw, match in (((_Gpu(3, 4), a, t, t), {}, "logits must be"), ((x, a, _Gpu(2, 3, dtype=torch.bfloat16), t), {}, "old_log_probs: expected"),
                            ((x, a, t, t), dict(entropy_coef=float("nan")), "entropy_coef"), ((x, a, t, t), dict(temperature=-1), "temperature")):
        with pytest.raises(AssertionError, match=match):
            g(*args, **kw)


def test_attention_refusals(monkeypatch):
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    f = policy.compute_linear_attention
    z = torch.zeros(1, 2, 3, 4)
    with pytest.raises(AssertionError, match="q must be on CUDA"):
        f(z, z, z, torch.ones(3))
    x, d = _Gpu(1, 2, 3, 4), _Gpu(3)
    for args, match in (((_Gpu(1, 2, 3), x, x, d), "q must be"), ((x, _Gpu(1, 2, 3, 5), x, d), "k shape"), ((x, x, _Gpu(1, 2, 2, 4), d), "v shape"),
                        ((x, x, _Gpu(1, 2, 3, 4, dtype=torch.bfloat16), d), "v: expected"), ((x, x, _Gpu(1, 2, 3, 129), d), "head dimensions"),
                        ((x, x, x, _Gpu(4)), "decay must have shape"), ((x, x, x, _Gpu(3, grad=True)), "constant"),
                        ((x, x, x, d, _Gpu(1, 3)), "dones shape"), ((x, x, x, d, _Gpu(1, 2, dtype=I64)), "dones: expected"),
                        ((x, x, x, d, None, _Gpu(1, 3, 4, 5)), "state must have shape"), ((x, x, x, d, None, None, 0.0), "scale"),
                        ((x, x, x, d, None, None, float("nan")), "scale")):
        with pytest.raises(AssertionError, match=match):
            f(*args)
    g, y = policy.compute_linear_attention_step, _Gpu(1, 3, 4)
    with pytest.raises(AssertionError, match="state is required"):
        g(y, y, y, d, None)
    with pytest.raises(AssertionError, match="q must be"):
        g(x, x, x, d, _Gpu(1, 3, 4, 4))
    with pytest.raises(AssertionError, match="state must have shape"):
        g(y, y, y, d, _Gpu(1, 3, 4, 5))
