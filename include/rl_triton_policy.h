/*
 * rl_triton_policy.h -- C ABI of the operators around the return estimators: what a learner computes
 * before them (log-probabilities of the taken actions, a memory over the steps of an episode) and after
 * them (the clipped policy loss and its gradient).  The reference has no counterpart of these.
 *
 * As in rl_triton_amd.h: device pointers, work enqueued on `stream` (a hipStream_t), nothing allocates or
 * synchronises, inputs are never written, RLK_OK or a negative RLK_ERR_* code comes back.  Empty inputs
 * return RLK_OK without a launch (losses and states excepted: those are written).  `bf16` non-zero: the arrays it names
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

#ifdef __cplusplus
}
#endif
#endif
