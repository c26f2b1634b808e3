// rlk_torch_policy.hpp -- the fast path of rl_triton.policy's functions, included by rlk_torch.cpp.
//
// As for the estimators: a call is taken when it can go to the C ABI (include/rl_triton_policy.h) as it stands; any other is
// declined and the Python implementation checks it, copies what it has to and raises.  Calls that need gradients
// are nodes of torch's graph from here too: a forward and backward pass of attention takes 68 us of host time and 158 through
// Python's functions (torch's own q * k takes 55 in the same loop).
#pragma once

// Checks of one call, on the device of its first tensor.
struct PolicyCall {
  c10::DeviceIndex dev = -1;
  bool ok = true;
  bool wants_grad = false;  // a gradient by one of the tensors looked at with `graph`

  const at::Tensor* fail() {
    ok = false;
    return nullptr;
  }
  // A tensor on the current GPU that is an ordinary one; `graph`: one whose derivatives are given, or refused where they are asked for.
  const at::Tensor* tensor(PyObject* o, bool graph) {
    if (!ok || !THPVariable_Check(o)) return fail();
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.is_neg()) return fail();
    if (graph) {
      if (t._fw_grad(0).defined()) return fail();  // (a dual tensor, which need not require a gradient: refused by the Python path)
      if (t.requires_grad() && at::GradMode::is_enabled()) wants_grad = true;
    }
    if (dev < 0) {
      dev = t.get_device();
      if (dev != c10::hip::current_device()) return fail();
    } else if (t.get_device() != dev) {
      return fail();
    }
    return &t;
  }
  const at::Tensor* array(PyObject* o, at::ScalarType st, at::IntArrayRef sizes, bool graph = false) {
    const at::Tensor* t = tensor(o, graph);
    if (!t || t->scalar_type() != st || !t->is_contiguous() || t->sizes() != sizes) return fail();
    return t;
  }
  const at::Tensor* opt(PyObject* o, at::ScalarType st, at::IntArrayRef sizes, bool graph = false) {
    return o == Py_None ? nullptr : array(o, st, sizes, graph);
  }
  double number(PyObject* o, double low) {
    double d = NAN;
    if (PyFloat_CheckExact(o)) d = PyFloat_AS_DOUBLE(o);
    else if (PyLong_CheckExact(o)) d = PyLong_AsDouble(o);
    if (PyErr_Occurred()) PyErr_Clear(), d = NAN;
    if (!std::isfinite(d) || d < low) fail();
    return d;
  }
  void* stream() const { return c10::hip::getCurrentHIPStream(dev).stream(); }
};

at::Tensor policy_output(at::IntArrayRef sizes, at::ScalarType st, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, st, like.device(), std::nullopt));
}

const void* data_or_null(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// Scratch memory, one of each kind per (device, stream), as rl_triton.policy._native keeps it; none (declined) while
// the stream is capturing a graph.  A backward pass asks for its own on torch's thread and without the interpreter lock, so the
// map has a lock of its own.  What it holds is guarded by kind: `sums` and `rows`, which calls from Python alone use, by the
// interpreter lock, `states` by StatesScratch's.  (An element stays where it is when others are added.)
struct PolicyScratch {
  at::Tensor sums, rows, states;
};
PolicyScratch& scratch_of(int dev, uintptr_t stream) {
  static auto* lock = new std::mutex;
  static auto* all = new std::map<std::pair<int, uintptr_t>, PolicyScratch>();
  const std::lock_guard<std::mutex> held(*lock);
  return (*all)[{dev, stream}];
}
bool policy_scratch(const PolicyCall& c, at::Tensor PolicyScratch::* kind, size_t need, const at::Tensor& like, void** ptr,
                    size_t* bytes) {
  *ptr = nullptr, *bytes = 0;
  if (need == 0) return true;
  hipStream_t s = static_cast<hipStream_t>(c.stream());
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &cs) != hipSuccess || cs != hipStreamCaptureStatusNone) return false;
  at::Tensor& buf = scratch_of((int)c.dev, reinterpret_cast<uintptr_t>(s)).*kind;
  if (!buf.defined() || (size_t)buf.numel() < need)
    buf = zeroed((int64_t)(buf.defined() ? std::max(need, 2 * (size_t)buf.numel()) : need), like);
  *ptr = buf.data_ptr(), *bytes = (size_t)buf.numel();
  return true;
}

// Scratch memory of sequences cut into segments, held from its choice to the launch: a backward pass runs on torch's own
// thread.  `own`: a call that is being captured has memory of its own, from the graph's pool, which keeps its place for the replays
// (others of the graph's may have it after the launch, in the stream's order) and goes with the graph; else there is none.
class StatesScratch {
 public:
  void* ptr = nullptr;
  size_t bytes = 0;
  bool ok = true;
  StatesScratch(const PolicyCall& c, size_t need, const at::Tensor& like, bool own) {
    if (!lock().try_lock()) {  // (whoever holds it may need the interpreter before they let go)
      PyThreadState* state = PyGILState_Check() ? PyEval_SaveThread() : nullptr;
      lock().lock();
      if (state) PyEval_RestoreThread(state);
    }
    try {
      ok = policy_scratch(c, &PolicyScratch::states, need, like, &ptr, &bytes);
      if (!ok && own) {
        captured = at::empty({(int64_t)need}, like.options().dtype(at::kByte));
        ptr = captured.data_ptr(), bytes = need, ok = true;
      }
    } catch (...) {
      lock().unlock();
      throw;
    }
  }
  ~StatesScratch() { lock().unlock(); }
  StatesScratch(const StatesScratch&) = delete;

 private:
  at::Tensor captured;
  static std::mutex& lock() {
    static auto* m = new std::mutex;
    return *m;
  }
};

// A node's results cannot be differentiated once more: they say so when that is tried, as Python's functions do.
struct DifferentiableOnce : torch::autograd::Function<DifferentiableOnce> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext*, const at::Tensor& x, const at::Tensor&) { return {x.detach()}; }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "trying to differentiate twice a function of rl_triton.policy, whose gradients are not differentiable");
  }
};
void once(torch::autograd::variable_list& grads, const torch::autograd::variable_list& from) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor& f : from)
    if (f.defined() && f.requires_grad()) {
      for (at::Tensor& g : grads)
        if (g.defined()) g = DifferentiableOnce::apply(g, f)[0];
      return;
    }
}

bool float_type(at::ScalarType st) { return st == at::kFloat || st == at::kBFloat16; }

// logits [envs, steps, actions] with contiguous actions, or contiguous ones of any other rank.
bool logit_layout(const at::Tensor& t, rlk_action_rows* r) {
  const int64_t n = t.size(-1);
  r->num_actions = n;
  r->logits = t.data_ptr(), r->bf16 = t.scalar_type() == at::kBFloat16;
  if (t.dim() == 3 && (t.stride(2) == 1 || n == 1)) {
    r->num_envs = t.size(0), r->seq_len = t.size(1), r->env_stride = t.stride(0), r->step_stride = t.stride(1);
  } else if (t.is_contiguous()) {
    r->num_envs = 1, r->seq_len = t.numel() / n, r->env_stride = t.numel(), r->step_stride = n;
  } else {
    return false;
  }
  return true;
}
bool logit_rows(PolicyCall& c, PyObject* logits, PyObject* actions, PyObject* temperature, bool graph, rlk_action_rows* r,
                const at::Tensor** x, const at::Tensor** a) {
  const at::Tensor* t = *x = c.tensor(logits, graph);
  if (!t || !float_type(t->scalar_type()) || t->dim() < 1 || t->numel() == 0 || !logit_layout(*t, r)) return false;
  *a = c.array(actions, at::kLong, t->sizes().slice(0, t->dim() - 1));
  const double tau = c.number(temperature, 0.0);
  if (!c.ok || !(tau >= RLK_LEAST_TEMPERATURE && tau <= RLK_LARGEST_TEMPERATURE)) return false;
  r->actions = static_cast<const int64_t*>((*a)->data_ptr());
  r->temperature = tau;
  return true;
}

struct ActionLogProbs : torch::autograd::Function<ActionLogProbs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& actions,
                                                const rlk_action_rows* r, void* stream) {
    std::vector<int64_t> two = actions.sizes().vec();
    at::Tensor lp = policy_output(two, at::kFloat, logits), ent = policy_output(two, at::kFloat, logits);
    two.push_back(2);
    at::Tensor norms = policy_output(two, at::kFloat, logits);
    const int st = rlk_action_log_probs(r, static_cast<float*>(lp.data_ptr()), static_cast<float*>(ent.data_ptr()),
                                        static_cast<float*>(norms.data_ptr()), stream);
    TORCH_CHECK(st == RLK_OK, "rlk_action_log_probs failed: ", rlk_status_string(st));
    ctx->save_for_backward({logits, actions, ent, norms});
    ctx->saved_data["temperature"] = r->temperature;
    ctx->set_materialize_grads(false);
    return {lp, ent};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], &actions = saved[1];
    torch::autograd::variable_list out(4);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    rlk_action_rows r = {};
    logit_layout(logits, &r);
    r.actions = static_cast<const int64_t*>(actions.data_ptr()), r.temperature = ctx->saved_data["temperature"].toDouble();
    at::Tensor up[2];
    const float* p[2] = {};
    for (int i = 0; i < 2; ++i)
      if (grads[i].defined()) up[i] = grads[i].contiguous(), p[i] = static_cast<const float*>(up[i].data_ptr());
    out[0] = policy_output(logits.sizes(), logits.scalar_type(), logits);
    const int st = rlk_action_log_probs_backward(&r, static_cast<const float*>(saved[2].data_ptr()), static_cast<const float*>(saved[3].data_ptr()),
                                                 p[0], p[1], out[0].data_ptr(), c10::hip::getCurrentHIPStream(logits.get_device()).stream());
    TORCH_CHECK(st == RLK_OK, "rlk_action_log_probs_backward failed: ", rlk_status_string(st));
    once(out, {logits, grads[0], grads[1]});
    return out;
  }
};

// action_log_probs(logits, actions, temperature)
PyObject* op_action_log_probs(PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || correctness_warnings()) return decline();
  PolicyCall c;
  rlk_action_rows r = {};
  const at::Tensor *x, *act;
  if (!logit_rows(c, a[0], a[1], a[2], true, &r, &x, &act)) return decline();
  if (act->numel() <= 256 && r.num_actions >= 32768 &&
      !policy_scratch(c, &PolicyScratch::rows, RLK_ROWS_WORKSPACE_BYTES, *x, &r.workspace, &r.workspace_bytes))
    return decline();
  if (c.wants_grad) {
    torch::autograd::variable_list o = ActionLogProbs::apply(*x, *act, &r, c.stream());
    return pair(o[0], o[1]);
  }
  at::Tensor lp = policy_output(act->sizes(), at::kFloat, *x), ent = policy_output(act->sizes(), at::kFloat, *x);
  const int st = rlk_action_log_probs(&r, static_cast<float*>(lp.data_ptr()), static_cast<float*>(ent.data_ptr()), nullptr, c.stream());
  return finish(st, "rlk_action_log_probs", pair(lp, ent));
}

// What both losses read: (old, advantages, ref, clip_low, clip_high, kl_coef, dual_clip, mask, reduction).
bool loss_terms(PolicyCall& c, PyObject* old, PyObject* adv, PyObject* ref, PyObject* low, PyObject* high, PyObject* kl, PyObject* dual,
                PyObject* mask, PyObject* reduction, at::ScalarType st, at::IntArrayRef sizes, const at::Tensor& like,
                rlk_policy_terms* t) {
  const at::Tensor *o = c.array(old, st, sizes), *ad = c.array(adv, st, sizes), *r = c.opt(ref, st, sizes), *m = c.opt(mask, st, sizes);
  t->clip_low = c.number(low, 0.0), t->clip_high = c.number(high, 0.0);
  t->kl_coef = c.number(kl, -HUGE_VAL);
  if (dual != Py_None) {
    const double d = c.number(dual, 1.0);
    if (!(d > 1.0)) return false;
    t->dual_clip = d;
  }
  if (!c.ok || !PyUnicode_Check(reduction)) return false;
  if (PyUnicode_CompareWithASCIIString(reduction, "rows") == 0) t->per_row = 1;
  else if (PyUnicode_CompareWithASCIIString(reduction, "steps") != 0) return false;
  t->old_log_probs = o->data_ptr(), t->advantages = ad->data_ptr(), t->ref_log_probs = data_or_null(r), t->mask = data_or_null(m);
  t->bf16 = st == at::kBFloat16;
  return policy_scratch(c, &PolicyScratch::sums, rlk_policy_workspace_bytes(sizes[0]), like, &t->workspace, &t->workspace_bytes);
}

PyObject* loss_result(int st, const char* what, at::Tensor& loss, at::Tensor& grad, at::Tensor& means) {
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(loss)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(grad)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(means)));
  return finish(st, what, r);
}

// policy_loss(log_probs, old_log_probs, advantages, ref_log_probs, clip_low, clip_high, kl_coef, dual_clip, mask, reduction)
PyObject* op_policy_loss(PyObject* const* a, Py_ssize_t n) {
  if (n != 10 || correctness_warnings()) return decline();
  PolicyCall c;
  const at::Tensor* lp = c.tensor(a[0], false);
  if (!lp || lp->dim() != 2 || !lp->is_contiguous() || !float_type(lp->scalar_type())) return decline();
  rlk_policy_terms t = {};
  if (!loss_terms(c, a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], lp->scalar_type(), lp->sizes(), *lp, &t)) return decline();
  at::Tensor loss = policy_output({}, at::kFloat, *lp), grad = policy_output(lp->sizes(), lp->scalar_type(), *lp),
             means = policy_output({4}, at::kFloat, *lp);
  t.loss = static_cast<float*>(loss.data_ptr()), t.means = static_cast<float*>(means.data_ptr());
  const int st = rlk_policy_loss(lp->data_ptr(), lp->size(0), lp->size(1), &t, grad.data_ptr(), c.stream());
  return loss_result(st, "rlk_policy_loss", loss, grad, means);
}

// policy_loss_from_logits(logits, actions, old_log_probs, advantages, ref_log_probs, clip_low, clip_high, kl_coef, entropy_coef,
//                         temperature, dual_clip, mask, reduction)
PyObject* op_policy_loss_from_logits(PyObject* const* a, Py_ssize_t n) {
  if (n != 13 || correctness_warnings()) return decline();
  PolicyCall c;
  rlk_action_rows r = {};
  const at::Tensor *x, *act;
  if (!logit_rows(c, a[0], a[1], a[9], false, &r, &x, &act) || x->dim() != 3) return decline();
  rlk_policy_terms t = {};
  t.entropy_coef = c.number(a[8], -HUGE_VAL);
  if (!loss_terms(c, a[2], a[3], a[4], a[5], a[6], a[7], a[10], a[11], a[12], at::kFloat, act->sizes(), *x, &t)) return decline();
  at::Tensor loss = policy_output({}, at::kFloat, *x), grad = policy_output(x->sizes(), x->scalar_type(), *x),
             means = policy_output({5}, at::kFloat, *x);
  t.loss = static_cast<float*>(loss.data_ptr()), t.means = static_cast<float*>(means.data_ptr());
  const int st = rlk_policy_loss_from_logits(&r, &t, grad.data_ptr(), c.stream());
  return loss_result(st, "rlk_policy_loss_from_logits", loss, grad, means);
}

// q, k, v of a sequence ([envs, steps, heads, dim]) or of a step ([envs, heads, dim]) and what goes with them.
bool attention_args(PolicyCall& c, PyObject* q_, PyObject* k_, PyObject* v_, PyObject* decay_, PyObject* dones_, PyObject* state_,
                    PyObject* scale_, bool steps, rlk_attention* t, const at::Tensor** v, at::Tensor* flags) {
  const at::Tensor *q = c.tensor(q_, true), *k = c.tensor(k_, true);
  *v = c.tensor(v_, true);
  if (!c.ok || !float_type(q->scalar_type()) || k->scalar_type() != q->scalar_type() || (*v)->scalar_type() != q->scalar_type()) return false;
  const int64_t rank = steps ? 4 : 3;
  if (q->dim() != rank || (*v)->dim() != rank || k->sizes() != q->sizes() ||
      (*v)->sizes().slice(0, rank - 1) != q->sizes().slice(0, rank - 1) || q->numel() == 0 || (*v)->numel() == 0)
    return false;
  t->num_envs = q->size(0), t->seq_len = steps ? q->size(1) : 1, t->heads = q->size(rank - 2);
  t->dim_k = q->size(rank - 1), t->dim_v = (*v)->size(rank - 1);
  if (t->dim_k > 128 || t->dim_v > 128) return false;
  auto seq = [&](const at::Tensor& x) {
    return rlk_sequence{x.data_ptr(), x.stride(0), steps ? x.stride(1) : 0, x.stride(rank - 2)};
  };
  for (const at::Tensor* x : {q, k, *v})
    if (x->size(rank - 1) > 1 && x->stride(rank - 1) != 1) return false;
  t->q = seq(*q), t->k = seq(*k), t->v = seq(**v);
  const at::Tensor* decay = c.array(decay_, at::kFloat, {t->heads}, true);
  const at::Tensor* dones = dones_ == Py_None ? nullptr : c.tensor(dones_, false);
  if (!c.ok || (dones && (dones->scalar_type() != at::kFloat || dones->sizes() != q->sizes().slice(0, steps ? 2 : 1)))) return false;
  if (dones && !dones->is_contiguous()) {  // (a step's column of a rollout buffer)
    *flags = dones->contiguous();
    dones = flags;
  }
  const at::Tensor* state = c.opt(state_, at::kFloat, {t->num_envs, t->heads, t->dim_k, t->dim_v}, true);
  if (!c.ok || decay->requires_grad()) return false;  // (refused by the Python path)
  const double scale = scale_ == Py_None ? 1.0 / std::sqrt((double)t->dim_k) : c.number(scale_, -HUGE_VAL);
  if (!c.ok || (float)scale == 0.f || !std::isfinite((float)scale)) return false;
  t->decay = static_cast<const float*>(decay->data_ptr()), t->dones = static_cast<const float*>(data_or_null(dones));
  t->state = static_cast<const float*>(data_or_null(state));
  t->scale = (float)scale, t->state_scale = t->state_out_scale = 1.f, t->bf16 = q->scalar_type() == at::kBFloat16;
  return true;
}

// The outputs: contiguous like v, and a state.
at::Tensor attention_out(const at::Tensor& v, rlk_attention* t) {
  at::Tensor out = policy_output(v.sizes(), v.scalar_type(), v);
  const bool steps = v.dim() == 4;
  t->out = {out.data_ptr(), out.stride(0), steps ? out.stride(1) : 0, out.stride(v.dim() - 2)};
  return out;
}

rlk_sequence steps_of(const at::Tensor& x) { return {x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)}; }

// What a call has beside its tensors of every call (a node's arguments are defined tensors: `state` is any where there is none).
struct AttentionCall {
  rlk_attention* t;
  at::Tensor dones;
  bool state;
  double scale;  // unrounded
  size_t need;   // of scratch memory
};

struct LinearAttention : torch::autograd::Function<LinearAttention> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                                                const at::Tensor& v, const at::Tensor& state, const at::Tensor& decay,
                                                const AttentionCall* call) {
    rlk_attention* t = call->t;
    at::Tensor out = attention_out(v, t), last = policy_output({t->num_envs, t->heads, t->dim_k, t->dim_v}, at::kFloat, v);
    t->state_out = static_cast<float*>(last.data_ptr());
    PolicyCall c;
    c.dev = q.get_device();
    const int st = [&] {
      const StatesScratch scratch(c, call->need, q, true);
      t->workspace = scratch.ptr, t->workspace_bytes = scratch.bytes;
      return rlk_linear_attention(t, 1, c.stream());
    }();
    TORCH_CHECK(st == RLK_OK, "rlk_linear_attention failed: ", rlk_status_string(st));
    ctx->save_for_backward({q, k, v, call->state ? state : at::Tensor(), decay, call->dones});
    ctx->saved_data["scale"] = call->scale;
    ctx->set_materialize_grads(false);
    return {out, last};
  }
  // The gradients are the same recurrence over other arrays (rlk_attention.hip): dq = (g, v, k) forward, and in
  // reverse dk = (v, g, q) and dv = (k, q, g), whose state at the first step is the state's gradient.
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &state = saved[3], &decay = saved[4], &dones = saved[5];
    torch::autograd::variable_list out(6);
    // the walks whose gradients are asked for (the state's comes with v's)
    const bool asked[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2) || ctx->needs_input_grad(3)};
    if ((!grads[0].defined() && !grads[1].defined()) || !(asked[0] || asked[1] || asked[2])) return out;
    const at::Tensor g = !grads[0].defined() ? at::zeros(v.sizes(), v.options())
                         : grads[0].stride(3) == 1 || v.size(3) == 1 ? grads[0] : grads[0].contiguous();
    const at::Tensor last = grads[1].defined() ? grads[1].contiguous() : grads[1];
    const double scale = ctx->saved_data["scale"].toDouble();
    rlk_attention t[3] = {};
    const at::Tensor* roles[3][3] = {{&g, &v, &k}, {&v, &g, &q}, {&k, &q, &g}};
    const at::Tensor* like[3] = {&q, &k, &v};
    int count = 0;
    for (int i = 0; i < 3; ++i) {
      if (!asked[i]) continue;
      rlk_attention& w = t[count++];
      out[i] = policy_output(like[i]->sizes(), like[i]->scalar_type(), *like[i]);
      w.q = steps_of(*roles[i][0]), w.k = steps_of(*roles[i][1]), w.v = steps_of(*roles[i][2]), w.out = steps_of(out[i]);
      w.num_envs = q.size(0), w.seq_len = q.size(1), w.heads = q.size(2);
      w.dim_k = roles[i][0]->size(3), w.dim_v = out[i].size(3);
      w.decay = static_cast<const float*>(decay.data_ptr()), w.dones = dones.defined() ? static_cast<const float*>(dones.data_ptr()) : nullptr;
      const at::Tensor& enters = i == 0 ? state : last;
      w.state = enters.defined() ? static_cast<const float*>(enters.data_ptr()) : nullptr;
      w.state_transposed = i < 2, w.reverse = i > 0, w.bf16 = q.scalar_type() == at::kBFloat16;
      w.scale = (float)scale, w.state_scale = i > 0 ? (float)(1.0 / scale) : 1.f, w.state_out_scale = i > 0 ? (float)scale : 1.f;
    }
    if (ctx->needs_input_grad(3)) {
      out[3] = policy_output({q.size(0), q.size(2), q.size(3), v.size(3)}, at::kFloat, q);
      t[count - 1].state_out = static_cast<float*>(out[3].data_ptr());
    }
    PolicyCall c;
    c.dev = q.get_device();
    size_t need = 0;
    for (int i = 0; i < count; ++i) {
      const rlk_attention& w = t[i];
      need += rlk_attention_workspace_bytes(w.num_envs, w.seq_len, w.heads, w.dim_k, w.dim_v);
    }
    const int st = [&] {
      const StatesScratch scratch(c, need, q, true);
      for (rlk_attention& w : t) w.workspace = scratch.ptr, w.workspace_bytes = scratch.bytes;
      return rlk_linear_attention(t, count, c.stream());
    }();
    TORCH_CHECK(st == RLK_OK, "rlk_linear_attention failed: ", rlk_status_string(st));
    once(out, {q, k, v, state, grads[0], grads[1]});
    return out;
  }
};

// linear_attention(q, k, v, decay, dones, state, scale)
PyObject* op_linear_attention(PyObject* const* a, Py_ssize_t n) {
  if (n != 7 || correctness_warnings()) return decline();
  PolicyCall c;
  rlk_attention t = {};
  const at::Tensor* v;
  at::Tensor flags;
  if (!attention_args(c, a[0], a[1], a[2], a[3], a[4], a[5], a[6], true, &t, &v, &flags)) return decline();
  const size_t need = rlk_attention_workspace_bytes(t.num_envs, t.seq_len, t.heads, t.dim_k, t.dim_v);
  if (c.wants_grad) {
    const bool state = a[5] != Py_None;
    const AttentionCall call{&t, flags.defined() ? flags : a[4] == Py_None ? at::Tensor() : THPVariable_Unpack(a[4]), state,
                             a[6] == Py_None ? 1.0 / std::sqrt((double)t.dim_k) : c.number(a[6], -HUGE_VAL), need};
    const at::Tensor& decay = THPVariable_Unpack(a[3]);
    torch::autograd::variable_list o = LinearAttention::apply(THPVariable_Unpack(a[0]), THPVariable_Unpack(a[1]), *v,
                                                              state ? THPVariable_Unpack(a[5]) : decay, decay, &call);
    return pair(o[0], o[1]);
  }
  const StatesScratch scratch(c, need, *v, false);
  if (!scratch.ok) return decline();
  t.workspace = scratch.ptr, t.workspace_bytes = scratch.bytes;
  at::Tensor out = attention_out(*v, &t), last = policy_output({t.num_envs, t.heads, t.dim_k, t.dim_v}, at::kFloat, *v);
  t.state_out = static_cast<float*>(last.data_ptr());
  return finish(rlk_linear_attention(&t, 1, c.stream()), "rlk_linear_attention", pair(out, last));
}

// A step's output where a gradient is wanted of it: it has none, and says so when it is asked for, not before.  The node's one input
// is a tensor of its own, so nothing of the steps before is held; the state goes on without a graph.
struct StepOutput : torch::autograd::Function<StepOutput> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext*, const at::Tensor&, const at::Tensor& v, rlk_attention* t) {
    return {attention_out(v, t)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "compute_linear_attention_step computes no gradient: a learner runs compute_linear_attention over the steps");
  }
};

// linear_attention_step(q, k, v, decay, state, dones, scale, out_state)
PyObject* op_linear_attention_step(PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || a[7] != Py_None || correctness_warnings()) return decline();
  PolicyCall c;
  rlk_attention t = {};
  const at::Tensor* v;
  at::Tensor flags;
  if (!attention_args(c, a[0], a[1], a[2], a[3], a[5], a[4], a[6], false, &t, &v, &flags) || !t.state) return decline();
  at::Tensor out = c.wants_grad ? StepOutput::apply(at::empty({0}, v->options()).requires_grad_(true), v->detach(), &t)[0] : attention_out(*v, &t);
  at::Tensor next = policy_output({t.num_envs, t.heads, t.dim_k, t.dim_v}, at::kFloat, *v);
  t.state_out = static_cast<float*>(next.data_ptr());
  return finish(rlk_linear_attention_step(&t, c.stream()), "rlk_linear_attention_step", pair(out, next));
}
