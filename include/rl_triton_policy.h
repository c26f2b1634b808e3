/*
 * rl_triton_policy.h -- C ABI of the operators around the return estimators: what a learner computes
 * before them (heads normed and rotated by their positions, a memory over the steps of an episode, the
 * sampling of actions, log-probabilities of the taken ones) and after them (the clipped policy loss and its
 * gradient).  The reference has no counterpart of these.
 *
 * As in rl_triton_amd.h: device pointers, work enqueued on `stream` (a hipStream_t), nothing allocates or
 * synchronises, inputs are never written, RLK_OK or a negative RLK_ERR_* code comes back.  Empty inputs
 * return RLK_OK without a launch (losses, states and the weights' gradients of the norms excepted: those are written).  `bf16` non-zero: the arrays it names
 * are rlk_bf16, otherwise float.  Sizes are counted and strides given in elements; every offset is formed in 64 bits.
 */
#ifndef RL_TRITON_POLICY_H
#define RL_TRITON_POLICY_H

#include "rl_triton_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* What logits are divided by is held as a reciprocal in float: outside this range that would be infinite or lose its digits. */
#define RLK_LEAST_TEMPERATURE 1e-38
#define RLK_LARGEST_TEMPERATURE 1e38

/* Rows of logits: [num_envs, seq_len, num_actions], the actions of a row contiguous, and the action taken
 * at each step.  An action outside [0, num_actions) has a log-probability of NaN; nothing is read for it. */
typedef struct rlk_action_rows {
  const void *logits;
  const int64_t *actions; /* [num_envs, seq_len], contiguous */
  int64_t num_envs, seq_len, num_actions;
  int64_t env_stride, step_stride;
  double temperature; /* logits are divided by it */
  int bf16;          /* logits (and their gradient) */
  /* NULL, or RLK_ROWS_WORKSPACE_BYTES (no initial contents needed) with which log-probabilities of few long rows are
   * shared by several workgroups a row.  The losses use their own. */
  void *workspace;
  size_t workspace_bytes;
} rlk_action_rows;

#define RLK_ROWS_WORKSPACE_BYTES 12288

/* log_probs[e,t] = x_a - log sum_j exp x_j with x = logits / temperature, and the entropy of every row.
 * norms: NULL, or [num_envs, seq_len, 2] for the backward call: the row's largest logit and the binary
 * logarithm of its sum of exponentials. */
int rlk_action_log_probs(const rlk_action_rows *rows, float *log_probs, float *entropies, float *norms, void *stream);

/* grad_logits (contiguous, the logits' type) from the gradients of both outputs (either may be NULL). */
int rlk_action_log_probs_backward(const rlk_action_rows *rows, const float *entropies, const float *norms,
                                  const float *grad_log_probs, const float *grad_entropies, void *grad_logits,
                                  void *stream);

/* The clipped policy loss: what it reads beside the log-probabilities, and where it goes.  Arrays are
 * contiguous [num_envs, seq_len], of one type. */
typedef struct rlk_policy_terms {
  const void *old_log_probs, *advantages;
  const void *ref_log_probs; /* NULL: no KL term */
  const void *mask;          /* NULL: every step takes part; else those with mask != 0 */
  double clip_low, clip_high; /* ratios are held to [1 - clip_low, 1 + clip_high] */
  double dual_clip;           /* > 1: the least that negative advantages count with, -A * dual_clip; 0: none */
  double kl_coef, entropy_coef;
  int per_row; /* 0: mean over the steps that take part; 1: mean over rows of their means */
  int bf16;    /* the arrays above (rlk_policy_loss: log_probs and the gradient too) */
  float *loss;  /* [1] */
  float *means; /* [4]: policy term, KL term (without its coefficient), share of steps whose gradient the
                   clipping removed, KL estimate to the old policy; from logits a fifth: the entropy */
  void *workspace;
  size_t workspace_bytes; /* at least rlk_policy_workspace_bytes(num_envs); zero-filled before its first use
                             and left ready for the next call on its stream */
} rlk_policy_terms;

size_t rlk_policy_workspace_bytes(int64_t num_envs);

/* The loss of log_probs [num_envs, seq_len] and its gradient. */
int rlk_policy_loss(const void *log_probs, int64_t num_envs, int64_t seq_len, const rlk_policy_terms *terms,
                    void *grad_log_probs, void *stream);

/* The loss of logits, minus entropy_coef times the mean entropy, and the logits' gradient (contiguous). */
int rlk_policy_loss_from_logits(const rlk_action_rows *rows, const rlk_policy_terms *terms, void *grad_logits,
                                void *stream);

/* One array of a sequence operator: [num_envs, seq_len, heads, dim], the dim contiguous. */
typedef struct rlk_sequence {
  const void *data;
  int64_t env_stride, step_stride, head_stride;
} rlk_sequence;

/* S_t = decay_h (1 - cut_t) S_{t-1} + k_t v_t^T,  out_t = scale * S_t^T q_t, cut_t = (done_{t-1} != 0).
 * reverse non-zero runs the same recurrence from the last step to the first, with cut_t = (done_t != 0): with
 * (q, k, v) = (v, grad_out, q) and (k, q, grad_out) it gives the gradients of k and v, and forward with
 * (grad_out, v, k) that of q. */
typedef struct rlk_attention {
  rlk_sequence q, k, v, out; /* out.data is written */
  int64_t num_envs, seq_len, heads, dim_k, dim_v; /* dims 1..128 */
  const float *decay;        /* [heads], 0..1 */
  const float *dones;        /* NULL or [num_envs, seq_len], contiguous */
  /* [num_envs, heads, dim_k, dim_v], contiguous; NULL: zeros.  Forward: S before the first step.  Reverse: the
   * gradient of the state after the last one. */
  const float *state;
  int state_transposed; /* `state` is [num_envs, heads, dim_v, dim_k] */
  /* NULL, or the state after the last step, zero if that step is done (of no steps: `state`); reverse: the gradient of the
   * state before the first step. */
  float *state_out;
  float scale;                        /* of out */
  float state_scale, state_out_scale; /* what `state` is multiplied with when read, `state_out` when written (the
                                         gradients of states: 1 / scale and scale; else 1) */
  int reverse;
  int bf16;        /* q, k, v, out */
  void *workspace; /* rlk_attention_workspace_bytes(), no initial contents needed */
  size_t workspace_bytes;
} rlk_attention;

size_t rlk_attention_workspace_bytes(int64_t num_envs, int64_t seq_len, int64_t heads, int64_t dim_k, int64_t dim_v);
/* `count` (1..3) of them in as few launches; they share num_envs, seq_len, heads, decay, dones and bf16. */
int rlk_linear_attention(const rlk_attention *calls, int count, void *stream);

/* One step for every environment: q, k, v, out with step_stride unused, dones [num_envs] or NULL.  `state`
 * is read, `state_out` written; they may be the same. */
int rlk_linear_attention_step(const rlk_attention *call, void *stream);

/* The gated delta rule: S_t = a_t S_{t-1} + k_t u_t^T with u_t = beta_t (v_t - a_t S_{t-1}^T k_t), a_t = exp(log_decay_t), 0 where
 * done_{t-1}; out_t = scale * S_t^T q_t.  A log-decay below -104 leaves nothing of the state, as -inf does. */
typedef struct rlk_delta_rule {
  rlk_sequence q, k, v, out; /* out.data is written */
  int64_t num_envs, seq_len, heads, dim_k, dim_v; /* dims 1..128 */
  const float *log_decays; /* NULL (zeros) or [num_envs, seq_len, heads], contiguous */
  const float *betas;      /* [num_envs, seq_len, heads], contiguous */
  const float *dones;      /* NULL or [num_envs, seq_len], contiguous */
  const float *state;      /* before the first step, [num_envs, heads, dim_k, dim_v], contiguous; NULL: zeros */
  float *state_out;        /* NULL, or the state after the last step, zero if that step is done (of no steps: `state`) */
  float scale;
  int bf16;                /* q, k, v, out */
  void *workspace;         /* rlk_delta_rule_workspace_bytes(), 16-byte aligned, no initial contents needed */
  size_t workspace_bytes;
} rlk_delta_rule;

/* Upstream gradients in `out` and `state_out` (NULL: none), the others are written; NULL data or pointers: not wanted.  Arrays of the gates
 * are contiguous, those of states too. */
typedef struct rlk_delta_rule_gradients {
  rlk_sequence out, q, k, v;
  const float *state_out;
  float *state, *log_decays, *betas;
} rlk_delta_rule_gradients;

/* Of a forward call, of a backward one, of a forward call with `saved` (whose records lie there; NULL will do where 0 bytes are asked for). */
#define RLK_DELTA_FORWARD 0
#define RLK_DELTA_BACKWARD 1
#define RLK_DELTA_FORWARD_SAVED 2
size_t rlk_delta_rule_workspace_bytes(int64_t num_envs, int64_t seq_len, int64_t heads, int64_t dim_k, int64_t dim_v, int pass);
/* Of what a forward call leaves for the backward one (16-byte aligned). */
size_t rlk_delta_rule_saved_bytes(int64_t num_envs, int64_t seq_len, int64_t heads, int64_t dim_k, int64_t dim_v);
/* `saved`: NULL, or what the backward call is to read.  heads * ceil(seq_len / 64) is at most 2^22. */
int rlk_gated_delta_rule(const rlk_delta_rule *call, void *saved, size_t saved_bytes, void *stream);
/* `call` as the forward one was, with a workspace of its own; its out and state_out are not looked at, and of its
 * state only whether there is one. */
int rlk_gated_delta_rule_backward(const rlk_delta_rule *call, const rlk_delta_rule_gradients *grads, const void *saved, size_t saved_bytes,
                                  void *stream);
/* One step for every environment: step strides and seq_len unused, log_decays and betas [num_envs, heads], dones [num_envs].  `state` is
 * read, `state_out` written; they may be the same. */
int rlk_gated_delta_rule_step(const rlk_delta_rule *call, void *stream);

/* Actions drawn from softmax(logits / temperature), truncated: of the actions ordered by their logits, the largest first and of equal ones the
 * first, those are kept that top_k says, of these the shortest beginning that holds top_p of their probability, of these the ones at
 * least min_p times as likely as the first.  The action is the first, in the order of their numbers, up to which the kept ones hold more
 * than the uniform number's share.  Rows without an allowed action (all logits -inf) and rows with a NaN: -1. */
typedef struct rlk_sampling {
  const void *logits; /* [num_envs, seq_len, num_actions], the actions of a row contiguous */
  int64_t num_envs, seq_len, num_actions; /* num_actions: 1 .. 2^20 */
  int64_t env_stride, step_stride;
  int bf16;
  const float *uniforms; /* [num_envs, seq_len], contiguous, in [0, 1) */
  double temperature;
  int64_t top_k; /* 0: all */
  double top_p;  /* above 0, up to 1: all */
  double min_p;  /* 0 .. 1, 0: all */
  int64_t *actions; /* [num_envs, seq_len] */
  float *log_probs; /* of the actions among those kept: [num_envs, seq_len]; -inf without one, NaN in rows with a NaN */
} rlk_sampling;

#define RLK_MOST_SAMPLED_ACTIONS (1 << 20)

int rlk_sample_actions(const rlk_sampling *call, void *stream);

/* Queries and keys, head by head: x / sqrt(mean(x^2) + eps) * weight, then the pairs of the first rotary_dim elements turned by
 * position * base^(-2 i / rotary_dim): elements i and i + rotary_dim / 2, or 2 i and 2 i + 1 (`interleaved`). */
typedef struct rlk_head_norms {
  rlk_sequence q, k;         /* heads of q_heads and k_heads; either number may be 0 */
  rlk_sequence q_out, k_out; /* backward: gradients of q and k */
  int64_t num_envs, seq_len, q_heads, k_heads, dim, rotary_dim; /* dim: 1 .. 256; rotary_dim: even, 0 .. dim */
  int interleaved, bf16;
  const float *q_weight, *k_weight; /* [dim] or NULL (ones) */
  const int64_t *positions;         /* [num_envs, seq_len], contiguous; NULL: nothing is turned */
  double base, eps;
} rlk_head_norms;

int rlk_query_key_norms(const rlk_head_norms *call, void *stream);
/* Gradients: of q and k into q_out and k_out (NULL data: not wanted), of the weights into q_weight_grad and k_weight_grad (NULL: not
 * wanted).  A workspace of rlk_head_norms_workspace_bytes() (no initial contents needed) where weights' gradients are. */
size_t rlk_head_norms_workspace_bytes(const rlk_head_norms *call);
int rlk_query_key_norms_backward(const rlk_head_norms *call, rlk_sequence grad_q, rlk_sequence grad_k, float *q_weight_grad,
                                 float *k_weight_grad, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
