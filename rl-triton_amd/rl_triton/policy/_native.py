"""ctypes binding of the learner's operators (include/rl_triton_policy.h) in librl_triton_amd.so.

Tensors reaching this module are on one GPU, of the right type and shape; this turns them into
the C ABI's structures, launches on torch's current stream of their device and owns the
workspaces, one per (device, stream), as rl_triton._native does for the estimators.
"""
from __future__ import annotations

import ctypes
import threading

import torch
from torch.autograd import forward_ad

from rl_triton import _native

_P, _I64, _F, _D, _INT, _SZ = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_float, ctypes.c_double, ctypes.c_int,
                               ctypes.c_size_t)


class ActionRows(ctypes.Structure):
    _fields_ = [("logits", _P), ("actions", _P), ("num_envs", _I64), ("seq_len", _I64), ("num_actions", _I64),
                ("env_stride", _I64), ("step_stride", _I64), ("temperature", _D), ("bf16", _INT),
                ("workspace", _P), ("workspace_bytes", _SZ)]


ROWS_WORKSPACE_BYTES = 12288


class PolicyTerms(ctypes.Structure):
    _fields_ = [("old_log_probs", _P), ("advantages", _P), ("ref_log_probs", _P), ("mask", _P), ("clip_low", _D),
                ("clip_high", _D), ("dual_clip", _D), ("kl_coef", _D), ("entropy_coef", _D), ("per_row", _INT),
                ("bf16", _INT), ("loss", _P), ("means", _P), ("workspace", _P), ("workspace_bytes", _SZ)]


class Sequence(ctypes.Structure):
    _fields_ = [("data", _P), ("env_stride", _I64), ("step_stride", _I64), ("head_stride", _I64)]


class Attention(ctypes.Structure):
    _fields_ = [("q", Sequence), ("k", Sequence), ("v", Sequence), ("out", Sequence), ("num_envs", _I64),
                ("seq_len", _I64), ("heads", _I64), ("dim_k", _I64), ("dim_v", _I64), ("decay", _P), ("dones", _P),
                ("state", _P), ("state_transposed", _INT), ("state_out", _P), ("scale", _F), ("state_scale", _F),
                ("state_out_scale", _F), ("reverse", _INT), ("bf16", _INT), ("workspace", _P),
                ("workspace_bytes", _SZ)]


class DeltaRule(ctypes.Structure):
    _fields_ = [("q", Sequence), ("k", Sequence), ("v", Sequence), ("out", Sequence), ("num_envs", _I64),
                ("seq_len", _I64), ("heads", _I64), ("dim_k", _I64), ("dim_v", _I64), ("log_decays", _P), ("betas", _P),
                ("dones", _P), ("state", _P), ("state_out", _P), ("scale", _F), ("bf16", _INT), ("workspace", _P),
                ("workspace_bytes", _SZ)]


class DeltaRuleGradients(ctypes.Structure):
    _fields_ = [("out", Sequence), ("q", Sequence), ("k", Sequence), ("v", Sequence), ("state_out", _P), ("state", _P),
                ("log_decays", _P), ("betas", _P)]


class Sampling(ctypes.Structure):
    _fields_ = [("logits", _P), ("num_envs", _I64), ("seq_len", _I64), ("num_actions", _I64), ("env_stride", _I64),
                ("step_stride", _I64), ("bf16", _INT), ("uniforms", _P), ("temperature", _D), ("top_k", _I64), ("top_p", _D),
                ("min_p", _D), ("actions", _P), ("log_probs", _P)]


class HeadNorms(ctypes.Structure):
    _fields_ = [("q", Sequence), ("k", Sequence), ("q_out", Sequence), ("k_out", Sequence), ("num_envs", _I64),
                ("seq_len", _I64), ("q_heads", _I64), ("k_heads", _I64), ("dim", _I64), ("rotary_dim", _I64),
                ("interleaved", _INT), ("bf16", _INT), ("q_weight", _P), ("k_weight", _P), ("positions", _P), ("base", _D),
                ("eps", _D)]


# name -> argtypes (must match include/rl_triton_policy.h)
SIGNATURES = {
    "rlk_action_log_probs": [ctypes.POINTER(ActionRows), _P, _P, _P, _P],
    "rlk_action_log_probs_backward": [ctypes.POINTER(ActionRows), _P, _P, _P, _P, _P, _P],
    "rlk_policy_workspace_bytes": [_I64],
    "rlk_policy_loss": [_P, _I64, _I64, ctypes.POINTER(PolicyTerms), _P, _P],
    "rlk_policy_loss_from_logits": [ctypes.POINTER(ActionRows), ctypes.POINTER(PolicyTerms), _P, _P],
    "rlk_attention_workspace_bytes": [_I64, _I64, _I64, _I64, _I64],
    "rlk_linear_attention": [ctypes.POINTER(Attention), _INT, _P],
    "rlk_linear_attention_step": [ctypes.POINTER(Attention), _P],
    "rlk_delta_rule_workspace_bytes": [_I64, _I64, _I64, _I64, _I64, _INT],
    "rlk_delta_rule_saved_bytes": [_I64, _I64, _I64, _I64, _I64],
    "rlk_gated_delta_rule": [ctypes.POINTER(DeltaRule), _P, _SZ, _P],
    "rlk_gated_delta_rule_backward": [ctypes.POINTER(DeltaRule), ctypes.POINTER(DeltaRuleGradients), _P, _SZ, _P],
    "rlk_gated_delta_rule_step": [ctypes.POINTER(DeltaRule), _P],
    "rlk_sample_actions": [ctypes.POINTER(Sampling), _P],
    "rlk_query_key_norms": [ctypes.POINTER(HeadNorms), _P],
    "rlk_head_norms_workspace_bytes": [ctypes.POINTER(HeadNorms)],
    "rlk_query_key_norms_backward": [ctypes.POINTER(HeadNorms), Sequence, Sequence, _P, _P, _P, _SZ, _P],
}
_RESTYPES = {"rlk_policy_workspace_bytes": _SZ, "rlk_attention_workspace_bytes": _SZ, "rlk_delta_rule_workspace_bytes": _SZ,
             "rlk_delta_rule_saved_bytes": _SZ, "rlk_head_norms_workspace_bytes": _SZ}

_lib = None


def load():
    global _lib
    if _lib is None:
        lib = _native.load()
        for name, argtypes in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.argtypes = argtypes
            fn.restype = _RESTYPES.get(name, _INT)
        _lib = lib
    return _lib


_BF16 = torch.bfloat16
# Scratch memory, one of each kind per (device, stream): "sums" of the losses, whose head is zero between calls,
# "rows" of statistics of shared rows, and "states" of sequences cut into segments.
_workspaces: dict = {}
_launching = threading.Lock()  # from a workspace's choice to the launch: a backward pass runs on torch's own thread


def _workspace(kind: str, dev: int, stream: int, need: int):
    """Scratch memory of the current call, to be held until its launch: kept per (device, stream), grown by doubling, zero-filled
    when made.  A call being captured into a graph has memory of its own from the graph's pool, which keeps its place for the replays
    (other work of the same graph may have it in turn, in the stream's order) and goes with the graph; "sums" are zero-filled there by
    a kernel that the graph records, the others need no initial contents."""
    if need == 0:
        return None
    device = torch.device("cuda", dev)
    if _native._capturing():
        return (torch.zeros if kind == "sums" else torch.empty)(need, dtype=torch.uint8, device=device)
    ws = _workspaces.get((kind, dev, stream))
    if ws is None or ws.numel() < need:
        ws = torch.zeros(max(need, 2 * ws.numel() if ws is not None else 0), dtype=torch.uint8, device=device)
        _workspaces[(kind, dev, stream)] = ws
    return ws


def _on_device(fn):
    """Runs `fn(dev, stream, ...)` with its first tensor's device current."""
    def call(lead, *args):
        dev = lead.get_device()
        with _launching:
            if dev != _native._cur_device():
                with torch.cuda.device(dev):
                    return fn(dev, _native._raw_stream(dev), lead, *args)
            return fn(dev, _native._raw_stream(dev), lead, *args)
    return call


def refuse_forward_derivatives(*tensors):
    """Raises for dual tensors, whose tangents the kernels would drop (they need not require a gradient)."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("forward-mode derivatives of rl_triton.policy's functions are not implemented")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _bytes(ws):
    return 0 if ws is None else ws.numel()


def _rows(logits, actions, temperature):
    e, t, a = logits.shape
    se, st, _ = logits.stride()
    return ActionRows(logits.data_ptr(), actions.data_ptr(), e, t, a, se, st, temperature, logits.dtype is _BF16)


@_on_device
def action_log_probs(dev, stream, logits, actions, temperature, log_probs, entropies, norms):
    rows = _rows(logits, actions, temperature)
    if actions.numel() <= 256:
        ws = _workspace("rows", dev, stream, ROWS_WORKSPACE_BYTES)
        rows.workspace, rows.workspace_bytes = ws.data_ptr(), ws.numel()
    _native._check((_lib or load()).rlk_action_log_probs(ctypes.byref(rows),
                                                        log_probs.data_ptr(), entropies.data_ptr(), _ptr(norms), stream),
                   "rlk_action_log_probs")


@_on_device
def action_log_probs_backward(dev, stream, logits, actions, temperature, entropies, norms, grad_log_probs,
                              grad_entropies, grad_logits):
    _native._check((_lib or load()).rlk_action_log_probs_backward(
        ctypes.byref(_rows(logits, actions, temperature)), entropies.data_ptr(), norms.data_ptr(), _ptr(grad_log_probs),
        _ptr(grad_entropies), grad_logits.data_ptr(), stream), "rlk_action_log_probs_backward")


def _terms(dev, stream, num_envs, old, advantages, ref, mask, clip, kl_coef, entropy_coef, per_row, loss, means):
    ws = _workspace("sums", dev, stream, (_lib or load()).rlk_policy_workspace_bytes(num_envs))
    low, high, dual = clip
    return ws, PolicyTerms(old.data_ptr(), advantages.data_ptr(), _ptr(ref), _ptr(mask), low, high, dual, kl_coef,
                       entropy_coef, per_row, old.dtype is _BF16, loss.data_ptr(), means.data_ptr(), ws.data_ptr(), ws.numel())


@_on_device
def policy_loss(dev, stream, log_probs, old, advantages, ref, mask, clip, kl_coef, per_row, loss, means, grad):
    e, t = log_probs.shape
    ws, terms = _terms(dev, stream, e, old, advantages, ref, mask, clip, kl_coef, 0.0, per_row, loss, means)
    _native._check(_lib.rlk_policy_loss(log_probs.data_ptr(), e, t, ctypes.byref(terms), grad.data_ptr(), stream),
                   "rlk_policy_loss")


@_on_device
def policy_loss_from_logits(dev, stream, logits, actions, temperature, old, advantages, ref, mask, clip, kl_coef,
                            entropy_coef, per_row, loss, means, grad):
    ws, terms = _terms(dev, stream, logits.shape[0], old, advantages, ref, mask, clip, kl_coef, entropy_coef, per_row, loss,
                       means)
    _native._check(_lib.rlk_policy_loss_from_logits(ctypes.byref(_rows(logits, actions, temperature)),
                                                   ctypes.byref(terms), grad.data_ptr(), stream),
                   "rlk_policy_loss_from_logits")


def _sequence(t):
    if t.dim() == 3:  # one step: [num_envs, heads, dim]
        return Sequence(t.data_ptr(), t.stride(0), 0, t.stride(1))
    return Sequence(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


class Pass:
    """One recurrence of a linear attention call: arrays by role, states, scales and direction."""
    __slots__ = ("a", "b", "c", "y", "state", "transposed", "state_out", "scale", "state_scale", "out_scale", "reverse")

    def __init__(self, a, b, c, y, state, state_out, scale, transposed=False, reverse=False, state_scale=1.0, out_scale=1.0):
        self.a, self.b, self.c, self.y = a, b, c, y
        self.state, self.state_out, self.transposed = state, state_out, transposed
        self.scale, self.state_scale, self.out_scale, self.reverse = scale, state_scale, out_scale, reverse

    def struct(self, decay, dones, ws, wsb):
        a, y = self.a, self.y
        seq = a.shape[1] if a.dim() == 4 else 1
        return Attention(_sequence(a), _sequence(self.b), _sequence(self.c), _sequence(y), a.shape[0], seq, a.shape[-2],
                         a.shape[-1], y.shape[-1], decay.data_ptr(), _ptr(dones), _ptr(self.state), self.transposed,
                         _ptr(self.state_out), self.scale, self.state_scale, self.out_scale, self.reverse,
                         a.dtype is _BF16, ws, wsb)


@_on_device
def linear_attention(dev, stream, decay, dones, passes):
    lib = _lib or load()
    e, t, h = passes[0].a.shape[:3]
    need = sum(lib.rlk_attention_workspace_bytes(e, t, h, p.a.shape[-1], p.y.shape[-1]) for p in passes)
    ws = _workspace("states", dev, stream, need)
    calls = (Attention * len(passes))(*(p.struct(decay, dones, _ptr(ws), _bytes(ws)) for p in passes))
    _native._check(lib.rlk_linear_attention(calls, len(passes), stream), "rlk_linear_attention")


@_on_device
def linear_attention_step(dev, stream, decay, dones, step):
    _native._check((_lib or load()).rlk_linear_attention_step(ctypes.byref(step.struct(decay, dones, None, 0)), stream),
                   "rlk_linear_attention_step")


def _delta_rule(q, k, v, out, log_decays, betas, dones, state, state_out, scale, ws):
    seq = q.shape[1] if q.dim() == 4 else 1
    return DeltaRule(_sequence(q), _sequence(k), _sequence(v), _sequence(out), q.shape[0], seq, q.shape[-2], q.shape[-1], v.shape[-1],
                     _ptr(log_decays), betas.data_ptr(), _ptr(dones), _ptr(state), _ptr(state_out), scale, q.dtype is _BF16, _ptr(ws),
                     _bytes(ws))


_FORWARD, _BACKWARD, _FORWARD_SAVED = 0, 1, 2  # RLK_DELTA_*


def _scratch(need, like):
    """Memory of one call, from torch's allocator: it may be GBs (1, or what 512 pairs of environments and heads ask for, or one environment), so none is
    kept.  (Its later users follow on the stream.)"""
    return torch.empty(need, dtype=torch.uint8, device=like.device)


@_on_device
def gated_delta_rule(dev, stream, q, k, v, out, log_decays, betas, dones, state, state_out, scale, keep):
    """Returns what the backward pass reads (`keep`), else None."""
    lib = _lib or load()
    e, t, h, dk = q.shape
    saved = _scratch(lib.rlk_delta_rule_saved_bytes(e, t, h, dk, v.shape[-1]), q) if keep else None
    ws = _scratch(lib.rlk_delta_rule_workspace_bytes(e, t, h, dk, v.shape[-1], _FORWARD_SAVED if keep else _FORWARD), q)
    call = _delta_rule(q, k, v, out, log_decays, betas, dones, state, state_out, scale, ws)
    _native._check(lib.rlk_gated_delta_rule(ctypes.byref(call), _ptr(saved), _bytes(saved), stream), "rlk_gated_delta_rule")
    return saved


@_on_device
def gated_delta_rule_backward(dev, stream, q, k, v, log_decays, betas, dones, state, scale, saved, grad_out, grad_last, grads, grad_state):
    lib = _lib or load()
    e, t, h, dk = q.shape
    ws = _scratch(lib.rlk_delta_rule_workspace_bytes(e, t, h, dk, v.shape[-1], _BACKWARD), q)
    call = _delta_rule(q, k, v, grad_out, log_decays, betas, dones, state, None, scale, ws)
    none = Sequence(None, 0, 0, 0)
    gq, gk, gv, gg, gb = grads
    to = DeltaRuleGradients(_sequence(grad_out), *(none if g is None else _sequence(g) for g in (gq, gk, gv)), _ptr(grad_last),
                            _ptr(grad_state), _ptr(gg), _ptr(gb))
    _native._check(lib.rlk_gated_delta_rule_backward(ctypes.byref(call), ctypes.byref(to), _ptr(saved), _bytes(saved), stream),
                   "rlk_gated_delta_rule_backward")


@_on_device
def gated_delta_rule_step(dev, stream, q, k, v, out, log_decays, betas, dones, state, state_out, scale):
    call = _delta_rule(q, k, v, out, log_decays, betas, dones, state, state_out, scale, None)
    _native._check((_lib or load()).rlk_gated_delta_rule_step(ctypes.byref(call), stream), "rlk_gated_delta_rule_step")


@_on_device
def sample_actions(dev, stream, logits, uniforms, temperature, top_k, top_p, min_p, actions, log_probs):
    e, t, a = logits.shape
    se, st, _ = logits.stride()
    call = Sampling(logits.data_ptr(), e, t, a, se, st, logits.dtype is _BF16, uniforms.data_ptr(), temperature, top_k, top_p, min_p,
                    actions.data_ptr(), log_probs.data_ptr())
    _native._check((_lib or load()).rlk_sample_actions(ctypes.byref(call), stream), "rlk_sample_actions")


_NONE = Sequence(None, 0, 0, 0)


def _head_norms(q, k, q_out, k_out, q_weight, k_weight, positions, base, rotary_dim, eps, interleaved):
    steps = q.shape[1] if q.dim() == 4 else 1
    out = [_NONE if t is None else _sequence(t) for t in (q_out, k_out)]
    return HeadNorms(_sequence(q), _sequence(k), *out, q.shape[0], steps, q.shape[-2], k.shape[-2], q.shape[-1], rotary_dim, interleaved,
                     q.dtype is _BF16, _ptr(q_weight), _ptr(k_weight), _ptr(positions), base, eps)


@_on_device
def query_key_norms(dev, stream, q, k, q_out, k_out, *settings):
    call = _head_norms(q, k, q_out, k_out, *settings)
    _native._check((_lib or load()).rlk_query_key_norms(ctypes.byref(call), stream), "rlk_query_key_norms")


@_on_device
def query_key_norms_backward(dev, stream, q, k, grad_q, grad_k, to_q, to_k, to_q_weight, to_k_weight, *settings):
    lib = _lib or load()
    call = _head_norms(q, k, to_q, to_k, *settings)
    weights = to_q_weight is not None or to_k_weight is not None
    ws = _scratch(lib.rlk_head_norms_workspace_bytes(ctypes.byref(call)), q) if weights else None
    up = [_NONE if t is None else _sequence(t) for t in (grad_q, grad_k)]
    _native._check(lib.rlk_query_key_norms_backward(ctypes.byref(call), *up, _ptr(to_q_weight), _ptr(to_k_weight), _ptr(ws), _bytes(ws),
                                                    stream), "rlk_query_key_norms_backward")
