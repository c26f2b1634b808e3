// rlk_torch_operators.hpp -- the fast path of the gated delta rule, the head norms and the sampling of actions, included by rlk_torch.cpp
// after rlk_torch_policy.hpp, whose checks and manners they share: a call that can go to the C ABI as it stands is taken, any other
// declined.
#pragma once

// Scratch memory of one call from torch's allocator, which keeps it in the stream's order (and, captured, in the graph's pool).
at::Tensor call_scratch(size_t bytes, const at::Tensor& like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }

// ---- sampled_actions(logits, uniforms, temperature, top_k, top_p, min_p)
PyObject* op_sampled_actions(PyObject* const* a, Py_ssize_t n) {
  if (n != 6 || correctness_warnings()) return decline();
  PolicyCall c;
  const at::Tensor* x = c.tensor(a[0], true);
  if (!x || !float_type(x->scalar_type()) || x->dim() < 1 || x->numel() == 0 || x->size(-1) > RLK_MOST_SAMPLED_ACTIONS) return decline();
  rlk_action_rows rows = {};
  if (!logit_layout(*x, &rows)) return decline();
  const at::Tensor* u = c.array(a[1], at::kFloat, x->sizes().slice(0, x->dim() - 1));
  rlk_sampling s = {};
  s.temperature = c.number(a[2], 0.0);
  s.top_p = a[4] == Py_None ? 1.0 : c.number(a[4], 0.0);
  s.min_p = a[5] == Py_None ? 0.0 : c.number(a[5], 0.0);
  if (a[3] != Py_None) {
    if (!PyLong_CheckExact(a[3])) return decline();
    int over = 0;
    const long long k = PyLong_AsLongLongAndOverflow(a[3], &over);
    if (over < 0 || (over == 0 && k < 1)) return decline();
    s.top_k = over > 0 || k > RLK_MOST_SAMPLED_ACTIONS ? RLK_MOST_SAMPLED_ACTIONS : k;
  }
  if (!c.ok || !(s.temperature >= RLK_LEAST_TEMPERATURE && s.temperature <= RLK_LARGEST_TEMPERATURE) || !(s.top_p > 0.0 && s.top_p <= 1.0) || s.min_p > 1.0)
    return decline();
  s.logits = rows.logits, s.num_envs = rows.num_envs, s.seq_len = rows.seq_len, s.num_actions = rows.num_actions;
  s.env_stride = rows.env_stride, s.step_stride = rows.step_stride, s.bf16 = rows.bf16;
  s.uniforms = static_cast<const float*>(u->data_ptr());
  at::Tensor actions = policy_output(u->sizes(), at::kLong, *x), log_probs = policy_output(u->sizes(), at::kFloat, *x);
  s.actions = static_cast<int64_t*>(actions.data_ptr()), s.log_probs = static_cast<float*>(log_probs.data_ptr());
  return finish(rlk_sample_actions(&s, c.stream()), "rlk_sample_actions", pair(actions, log_probs));
}

// ---- query_key_norms(q, k, q_weight, k_weight, positions, base, rotary_dim, eps, interleaved)
rlk_sequence rows_of(const at::Tensor& x) {  // of a sequence or of a step
  const bool steps = x.dim() == 4;
  return {x.data_ptr(), x.stride(0), steps ? x.stride(1) : 0, x.stride(steps ? 2 : 1)};
}

// What a call has beside its tensors of every call (a node's arguments are defined tensors: where there is no weight, q stands).
struct NormsCall {
  rlk_head_norms* t;
  at::Tensor positions;
  bool weights[2];
};

struct QueryKeyNorms : torch::autograd::Function<QueryKeyNorms> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                                                const at::Tensor& q_weight, const at::Tensor& k_weight, const NormsCall* call) {
    rlk_head_norms* t = call->t;
    at::Tensor out[2] = {policy_output(q.sizes(), q.scalar_type(), q), policy_output(k.sizes(), k.scalar_type(), k)};
    t->q_out = rows_of(out[0]), t->k_out = rows_of(out[1]);
    const int st = rlk_query_key_norms(t, c10::hip::getCurrentHIPStream(q.get_device()).stream());
    TORCH_CHECK(st == RLK_OK, "rlk_query_key_norms failed: ", rlk_status_string(st));
    ctx->save_for_backward({q, k, call->weights[0] ? q_weight : at::Tensor(), call->weights[1] ? k_weight : at::Tensor(), call->positions});
    ctx->saved_data["base"] = t->base, ctx->saved_data["eps"] = t->eps;
    ctx->saved_data["rotary"] = t->rotary_dim, ctx->saved_data["interleaved"] = (int64_t)t->interleaved;
    ctx->set_materialize_grads(false);
    return {out[0], out[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &positions = saved[4];
    torch::autograd::variable_list out(5);
    rlk_head_norms t = {};
    const bool steps = q.dim() == 4;
    t.q = rows_of(q), t.k = rows_of(k);
    t.num_envs = q.size(0), t.seq_len = steps ? q.size(1) : 1, t.q_heads = q.size(-2), t.k_heads = k.size(-2), t.dim = q.size(-1);
    t.rotary_dim = ctx->saved_data["rotary"].toInt(), t.interleaved = (int)ctx->saved_data["interleaved"].toInt();
    t.base = ctx->saved_data["base"].toDouble(), t.eps = ctx->saved_data["eps"].toDouble(), t.bf16 = q.scalar_type() == at::kBFloat16;
    t.q_weight = saved[2].defined() ? static_cast<const float*>(saved[2].data_ptr()) : nullptr;
    t.k_weight = saved[3].defined() ? static_cast<const float*>(saved[3].data_ptr()) : nullptr;
    t.positions = positions.defined() ? static_cast<const int64_t*>(positions.data_ptr()) : nullptr;
    at::Tensor up[2];
    rlk_sequence from[2] = {}, *to[2] = {&t.q_out, &t.k_out};
    float* weights[2] = {};
    bool any = false;
    for (int i = 0; i < 2; ++i) {
      if (!grads[i].defined()) continue;
      up[i] = grads[i].stride(-1) == 1 || grads[i].size(-1) == 1 ? grads[i] : grads[i].contiguous();
      from[i] = rows_of(up[i]);
      if (ctx->needs_input_grad(i)) out[i] = policy_output(saved[i].sizes(), saved[i].scalar_type(), q), *to[i] = rows_of(out[i]), any = true;
      if (saved[2 + i].defined() && ctx->needs_input_grad(2 + i))
        out[2 + i] = policy_output({t.dim}, at::kFloat, q), weights[i] = static_cast<float*>(out[2 + i].data_ptr()), any = true;
    }
    if (!any) return out;
    const bool sums = weights[0] || weights[1];
    const at::Tensor scratch = sums ? call_scratch(rlk_head_norms_workspace_bytes(&t), q) : at::Tensor();
    const int st = rlk_query_key_norms_backward(&t, from[0], from[1], weights[0], weights[1], sums ? scratch.data_ptr() : nullptr,
                                                sums ? (size_t)scratch.numel() : 0, c10::hip::getCurrentHIPStream(q.get_device()).stream());
    TORCH_CHECK(st == RLK_OK, "rlk_query_key_norms_backward failed: ", rlk_status_string(st));
    once(out, {q, k, saved[2], saved[3], grads[0], grads[1]});
    return out;
  }
};

PyObject* op_query_key_norms(PyObject* const* a, Py_ssize_t n) {
  if (n != 9 || correctness_warnings()) return decline();
  PolicyCall c;
  const at::Tensor *q = c.tensor(a[0], true), *k = c.tensor(a[1], true);
  if (!c.ok || !float_type(q->scalar_type()) || k->scalar_type() != q->scalar_type() || (q->dim() != 3 && q->dim() != 4) || k->dim() != q->dim() ||
      q->numel() == 0 || k->numel() == 0)
    return decline();
  const int64_t rank = q->dim(), dim = q->size(-1);
  if (k->size(-1) != dim || k->sizes().slice(0, rank - 2) != q->sizes().slice(0, rank - 2) || dim > 256 || q->size(-2) > 65536 || k->size(-2) > 65536)
    return decline();
  for (const at::Tensor* x : {q, k})
    if (dim > 1 && x->stride(-1) != 1) return decline();
  const at::Tensor *qw = c.opt(a[2], at::kFloat, {dim}, true), *kw = c.opt(a[3], at::kFloat, {dim}, true);
  const at::Tensor* positions = c.opt(a[4], at::kLong, q->sizes().slice(0, rank - 2));
  rlk_head_norms t = {};
  t.base = c.number(a[5], 0.0), t.eps = c.number(a[7], 0.0);
  if (a[6] == Py_None) {
    t.rotary_dim = positions ? dim : 0;
  } else {
    if (!PyLong_CheckExact(a[6])) return decline();
    int over = 0;
    t.rotary_dim = PyLong_AsLongLongAndOverflow(a[6], &over);
    if (over != 0) return decline();
  }
  if (a[8] != Py_True && a[8] != Py_False) return decline();
  if (!c.ok || t.base <= 0.0 || t.eps > 3.4e38 || t.rotary_dim < 0 || t.rotary_dim > dim || t.rotary_dim % 2 != 0) return decline();
  t.interleaved = a[8] == Py_True, t.bf16 = q->scalar_type() == at::kBFloat16;
  t.q = rows_of(*q), t.k = rows_of(*k);
  t.num_envs = q->size(0), t.seq_len = rank == 4 ? q->size(1) : 1, t.q_heads = q->size(-2), t.k_heads = k->size(-2), t.dim = dim;
  t.q_weight = static_cast<const float*>(data_or_null(qw)), t.k_weight = static_cast<const float*>(data_or_null(kw));
  t.positions = static_cast<const int64_t*>(data_or_null(positions));
  if (c.wants_grad) {
    const NormsCall call{&t, positions ? *positions : at::Tensor(), {qw != nullptr, kw != nullptr}};
    torch::autograd::variable_list o = QueryKeyNorms::apply(*q, *k, qw ? *qw : *q, kw ? *kw : *q, &call);
    return pair(o[0], o[1]);
  }
  at::Tensor oq = policy_output(q->sizes(), q->scalar_type(), *q), ok = policy_output(k->sizes(), k->scalar_type(), *k);
  t.q_out = rows_of(oq), t.k_out = rows_of(ok);
  return finish(rlk_query_key_norms(&t, c.stream()), "rlk_query_key_norms", pair(oq, ok));
}

// ---- the gated delta rule
struct DeltaArgs {
  const at::Tensor *q, *k, *v, *decays, *betas, *state;
  at::Tensor dones;
};
// q, k, v of a sequence or of a step and what goes with them.
bool delta_args(PolicyCall& c, PyObject* const* a, PyObject* dones_, PyObject* state_, PyObject* scale_, bool steps, rlk_delta_rule* t, DeltaArgs* x) {
  x->q = c.tensor(a[0], true), x->k = c.tensor(a[1], true), x->v = c.tensor(a[2], true);
  if (!c.ok) return false;
  const at::Tensor &q = *x->q, &k = *x->k, &v = *x->v;
  const int64_t rank = steps ? 4 : 3;
  if (!float_type(q.scalar_type()) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || q.dim() != rank || v.dim() != rank ||
      k.sizes() != q.sizes() || v.sizes().slice(0, rank - 1) != q.sizes().slice(0, rank - 1) || q.numel() == 0 || v.numel() == 0)
    return false;
  t->num_envs = q.size(0), t->seq_len = steps ? q.size(1) : 1, t->heads = q.size(rank - 2), t->dim_k = q.size(rank - 1), t->dim_v = v.size(rank - 1);
  if (t->dim_k > 128 || t->dim_v > 128 || t->seq_len > (int64_t{1} << 30) || t->heads > (int64_t{1} << 22) ||
      (steps && t->heads * ((t->seq_len + 63) / 64) > (int64_t{1} << 22)))
    return false;
  for (const at::Tensor* y : {&q, &k, &v})
    if (y->size(rank - 1) > 1 && y->stride(rank - 1) != 1) return false;
  t->q = rows_of(q), t->k = rows_of(k), t->v = rows_of(v);
  x->decays = c.opt(a[3], at::kFloat, q.sizes().slice(0, rank - 1), true);
  x->betas = c.array(a[4], at::kFloat, q.sizes().slice(0, rank - 1), true);
  const at::Tensor* dones = dones_ == Py_None ? nullptr : c.tensor(dones_, false);
  if (!c.ok || (dones && (dones->scalar_type() != at::kFloat || dones->sizes() != q.sizes().slice(0, steps ? 2 : 1)))) return false;
  if (dones) x->dones = dones->contiguous();  // (a step's column of a rollout buffer)
  x->state = c.opt(state_, at::kFloat, {t->num_envs, t->heads, t->dim_k, t->dim_v}, true);
  const double scale = scale_ == Py_None ? 1.0 / std::sqrt((double)t->dim_k) : c.number(scale_, -HUGE_VAL);
  if (!c.ok || !(std::abs(scale) <= 3.4e38)) return false;
  t->log_decays = static_cast<const float*>(data_or_null(x->decays)), t->betas = static_cast<const float*>(x->betas->data_ptr());
  t->dones = dones ? static_cast<const float*>(x->dones.data_ptr()) : nullptr;
  t->state = static_cast<const float*>(data_or_null(x->state));
  t->scale = (float)scale, t->bf16 = q.scalar_type() == at::kBFloat16;
  return true;
}

// The launch of a sequence's forward pass; with `saved`, what the backward pass reads.
int delta_forward(rlk_delta_rule* t, const at::Tensor& out, const at::Tensor& last, const at::Tensor* saved) {
  t->out = rows_of(out), t->state_out = static_cast<float*>(last.data_ptr());
  const at::Tensor scratch = call_scratch(rlk_delta_rule_workspace_bytes(t->num_envs, t->seq_len, t->heads, t->dim_k, t->dim_v,
                                                                         saved ? RLK_DELTA_FORWARD_SAVED : RLK_DELTA_FORWARD), out);
  t->workspace = scratch.data_ptr(), t->workspace_bytes = (size_t)scratch.numel();
  return rlk_gated_delta_rule(t, saved ? saved->data_ptr() : nullptr, saved ? (size_t)saved->numel() : 0,
                              c10::hip::getCurrentHIPStream(out.get_device()).stream());
}

struct DeltaCall {
  rlk_delta_rule* t;
  at::Tensor dones;
  bool decays, state;
};

struct GatedDeltaRule : torch::autograd::Function<GatedDeltaRule> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                const at::Tensor& decays, const at::Tensor& betas, const at::Tensor& state, const DeltaCall* call) {
    rlk_delta_rule* t = call->t;
    at::Tensor out = policy_output(v.sizes(), v.scalar_type(), v), last = policy_output({t->num_envs, t->heads, t->dim_k, t->dim_v}, at::kFloat, v);
    const at::Tensor saved = call_scratch(rlk_delta_rule_saved_bytes(t->num_envs, t->seq_len, t->heads, t->dim_k, t->dim_v), q);
    const int st = delta_forward(t, out, last, &saved);
    TORCH_CHECK(st == RLK_OK, "rlk_gated_delta_rule failed: ", rlk_status_string(st));
    ctx->save_for_backward({q, k, v, call->decays ? decays : at::Tensor(), betas, call->state ? state : at::Tensor(), call->dones, saved});
    ctx->saved_data["scale"] = (double)t->scale;
    ctx->set_materialize_grads(false);
    return {out, last};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto kept = ctx->get_saved_variables();
    const at::Tensor &q = kept[0], &k = kept[1], &v = kept[2], &decays = kept[3], &betas = kept[4], &state = kept[5], &dones = kept[6], &saved = kept[7];
    torch::autograd::variable_list out(7);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const at::Tensor g = !grads[0].defined() ? at::zeros(v.sizes(), v.options())
                         : grads[0].stride(3) == 1 || v.size(3) == 1 ? grads[0] : grads[0].contiguous();
    const at::Tensor last = grads[1].defined() ? grads[1].contiguous() : grads[1];
    rlk_delta_rule t = {};
    t.q = rows_of(q), t.k = rows_of(k), t.v = rows_of(v);
    t.num_envs = q.size(0), t.seq_len = q.size(1), t.heads = q.size(2), t.dim_k = q.size(3), t.dim_v = v.size(3);
    auto floats = [](const at::Tensor& x) { return x.defined() ? static_cast<float*>(x.data_ptr()) : nullptr; };
    t.log_decays = floats(decays), t.betas = floats(betas), t.dones = floats(dones), t.state = floats(state);
    t.scale = (float)ctx->saved_data["scale"].toDouble(), t.bf16 = q.scalar_type() == at::kBFloat16;
    rlk_delta_rule_gradients to = {};
    to.out = rows_of(g), to.state_out = floats(last);
    const at::Tensor* like[6] = {&q, &k, &v, &decays, &betas, &state};
    bool any = false;
    for (int i = 0; i < 6; ++i)
      if (like[i]->defined() && ctx->needs_input_grad(i)) out[i] = policy_output(like[i]->sizes(), like[i]->scalar_type(), q), any = true;
    if (!any) return out;
    rlk_sequence* sequences[3] = {&to.q, &to.k, &to.v};
    for (int i = 0; i < 3; ++i)
      if (out[i].defined()) *sequences[i] = rows_of(out[i]);
    to.log_decays = floats(out[3]), to.betas = floats(out[4]), to.state = floats(out[5]);
    const at::Tensor scratch = call_scratch(rlk_delta_rule_workspace_bytes(t.num_envs, t.seq_len, t.heads, t.dim_k, t.dim_v, RLK_DELTA_BACKWARD), q);
    t.workspace = scratch.data_ptr(), t.workspace_bytes = (size_t)scratch.numel();
    const int st = rlk_gated_delta_rule_backward(&t, &to, saved.data_ptr(), (size_t)saved.numel(), c10::hip::getCurrentHIPStream(q.get_device()).stream());
    TORCH_CHECK(st == RLK_OK, "rlk_gated_delta_rule_backward failed: ", rlk_status_string(st));
    once(out, {q, k, v, decays, betas, state, grads[0], grads[1]});
    return out;
  }
};

// gated_delta_rule(q, k, v, log_decays, betas, dones, state, scale)
PyObject* op_gated_delta_rule(PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || correctness_warnings()) return decline();
  PolicyCall c;
  rlk_delta_rule t = {};
  DeltaArgs x;
  if (!delta_args(c, a, a[5], a[6], a[7], true, &t, &x)) return decline();
  if (c.wants_grad) {
    const DeltaCall call{&t, x.dones, x.decays != nullptr, x.state != nullptr};
    torch::autograd::variable_list o = GatedDeltaRule::apply(*x.q, *x.k, *x.v, x.decays ? *x.decays : *x.betas, *x.betas, x.state ? *x.state : *x.betas, &call);
    return pair(o[0], o[1]);
  }
  at::Tensor out = policy_output(x.v->sizes(), x.v->scalar_type(), *x.v), last = policy_output({t.num_envs, t.heads, t.dim_k, t.dim_v}, at::kFloat, *x.v);
  const int st = delta_forward(&t, out, last, nullptr);  // (before pair() takes the tensors: arguments have no order)
  return finish(st, "rlk_gated_delta_rule", pair(out, last));
}

// A step's output where a gradient is wanted of it (as StepOutput).
struct DeltaStepOutput : torch::autograd::Function<DeltaStepOutput> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext*, const at::Tensor&, const at::Tensor& v) {
    return {policy_output(v.sizes(), v.scalar_type(), v)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "compute_gated_delta_rule_step computes no gradient: a learner runs compute_gated_delta_rule over the steps");
  }
};

// gated_delta_rule_step(q, k, v, log_decays, betas, state, dones, scale, out_state)
PyObject* op_gated_delta_rule_step(PyObject* const* a, Py_ssize_t n) {
  if (n != 9 || a[8] != Py_None || correctness_warnings()) return decline();
  PolicyCall c;
  rlk_delta_rule t = {};
  DeltaArgs x;
  if (!delta_args(c, a, a[6], a[5], a[7], false, &t, &x) || !x.state) return decline();
  at::Tensor out = c.wants_grad ? DeltaStepOutput::apply(at::empty({0}, x.v->options()).requires_grad_(true), x.v->detach())[0]
                                : policy_output(x.v->sizes(), x.v->scalar_type(), *x.v);
  at::Tensor next = policy_output({t.num_envs, t.heads, t.dim_k, t.dim_v}, at::kFloat, *x.v);
  t.out = rows_of(out), t.state_out = static_cast<float*>(next.data_ptr());
  return finish(rlk_gated_delta_rule_step(&t, c.stream()), "rlk_gated_delta_rule_step", pair(out, next));
}
