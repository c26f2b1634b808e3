// rlk_policy_loss.hip -- the clipped policy loss from log-probabilities, and the counting and summing that
// the loss from logits shares (include/rl_triton_policy.h).
#include "rlk_policy.hpp"

namespace rlk {
namespace {

constexpr int kNT = 256;

// What the mean divides by: the steps with mask != 0 or, per_row, the rows that have any (and each row's
// number).  A wavefront per row, or the whole workgroup where there are few.
template <class E>
__global__ __launch_bounds__(kNT) void count_kernel(const E* __restrict__ mask, int64_t num_envs, int64_t seq_len,
                                                    int per_row, int64_t* __restrict__ parts, int* __restrict__ row_counts) {
  __shared__ int64_t s[kNT / 64];
  int64_t total = 0;
  if (!per_row) {
    const int64_t n = num_envs * seq_len, step = (int64_t)gridDim.x * kNT;
    for (int64_t i = (int64_t)blockIdx.x * kNT + threadIdx.x; i < n; i += step) total += load_one(mask + i) != 0.f;
  } else {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int64_t e = (int64_t)blockIdx.x * (kNT / 64) + wave; e < num_envs; e += (int64_t)gridDim.x * (kNT / 64)) {
      int n = 0;
      for (int64_t t = lane; t < seq_len; t += 64) n += load_one(mask + e * seq_len + t) != 0.f;
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
      if (lane == 0) {
        row_counts[e] = n;
        total += n > 0;
      }
    }
  }
  total = block_sum<kNT>(total, s);
  if (threadIdx.x == 0) parts[blockIdx.x] = total;
}

template <class E>
struct LossArgs {
  const E *lp, *old, *adv, *ref, *mask;
  E* grad;
  int64_t n, seq_len;
  LossConsts c;
  Weights w;
  double* partials;
};

template <class E>
__global__ __launch_bounds__(kNT) void loss_kernel(const LossArgs<E> a) {
  __shared__ int64_t sc[kNT / 64];
  __shared__ double sd[kNT / 64];
  const float scale = weight_scale<kNT>(a.w, sc);
  float acc[kTerms] = {};
  const int64_t step = (int64_t)gridDim.x * kNT;
  for (int64_t i = (int64_t)blockIdx.x * kNT + threadIdx.x; i < a.n; i += step) {
    float g = 0.f;
    if (a.mask == nullptr || load_one(a.mask + i) != 0.f) {
      float w = scale;
      if (a.w.row_counts != nullptr) w /= (float)a.w.row_counts[i / a.seq_len];
      const StepTerms t = step_terms(load_one(a.lp + i), load_one(a.old + i), load_one(a.adv + i),
                                     a.ref ? load_one(a.ref + i) : 0.f, a.ref != nullptr, a.c);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += w * t.v[k];
      g = w * t.slope;
    }
    a.grad[i] = from_f32<E>(g);
  }
  write_partials<kNT>(acc, a.partials, sd);
}

__global__ __launch_bounds__(kNT) void finish_kernel(const double* __restrict__ partials, int blocks, int means,
                                                     float kl_coef, float entropy_coef, float* __restrict__ loss,
                                                     float* __restrict__ out) {
  __shared__ double s[kNT / 64];
  double v[kTerms] = {};
  for (int b = threadIdx.x; b < blocks; b += kNT)
#pragma unroll
    for (int k = 0; k < kTerms; ++k) v[k] += partials[(int64_t)b * kTerms + k];
#pragma unroll
  for (int k = 0; k < kTerms; ++k) v[k] = block_sum<kNT>(v[k], s);
  if (threadIdx.x == 0) {
    *loss = (float)(v[0] + (double)kl_coef * v[1] - (double)entropy_coef * v[4]);
    for (int k = 0; k < means; ++k) out[k] = (float)v[k];
  }
}

template <class E>
int loss_impl(const void* lp, int64_t E_, int64_t T, const rlk_policy_terms* t, void* grad, hipStream_t s) {
  LossPlan plan;
  int st = plan_loss(t, E_, T, &plan);
  if (st != RLK_OK) return st;
  const int64_t n = E_ * T;
  if (n > 0 && (!lp || !grad)) return RLK_ERR_INVALID_ARGUMENT;
  if ((st = launch_count(t, E_, T, &plan, s)) != RLK_OK) return st;
  int64_t blocks = (n + kNT * 4 - 1) / (kNT * 4);
  blocks = blocks < 1 ? 1 : blocks > 2048 ? 2048 : blocks;
  LossArgs<E> a{static_cast<const E*>(lp), static_cast<const E*>(t->old_log_probs), static_cast<const E*>(t->advantages),
                static_cast<const E*>(t->ref_log_probs), static_cast<const E*>(t->mask), static_cast<E*>(grad),
                n, T, plan.consts, plan.weights, plan.partials};
  loss_kernel<E><<<dim3((unsigned)blocks), dim3(kNT), 0, s>>>(a);
  if (hipGetLastError() != hipSuccess) return RLK_ERR_LAUNCH;
  return launch_finish(t, plan, (int)blocks, 4, s);
}

}  // namespace

int plan_loss(const rlk_policy_terms* t, int64_t num_envs, int64_t seq_len, LossPlan* p) {
  if (!t || num_envs < 0 || seq_len < 0 || !t->loss || !t->means) return RLK_ERR_INVALID_ARGUMENT;
  if (num_envs * seq_len > 0 && (!t->old_log_probs || !t->advantages)) return RLK_ERR_INVALID_ARGUMENT;
  if (!(t->clip_low >= 0.f) || !(t->clip_high >= 0.f) || !(t->dual_clip == 0.f || t->dual_clip > 1.f))
    return RLK_ERR_INVALID_ARGUMENT;
  if (seq_len > (int64_t{1} << 30)) return RLK_ERR_INVALID_ARGUMENT;  // (a row's count is an int)
  if (!t->workspace || t->workspace_bytes < rlk_policy_workspace_bytes(num_envs) ||
      (reinterpret_cast<uintptr_t>(t->workspace) & 7u) != 0)
    return RLK_ERR_WORKSPACE;
  LossConsts& c = p->consts;
  c.low = 1.f - t->clip_low, c.high = 1.f + t->clip_high;
  c.log_low = t->clip_low < 1.f ? (float)std::log1p(-(double)t->clip_low) : -INFINITY;
  c.log_high = (float)std::log1p((double)t->clip_high);
  c.dual = t->dual_clip, c.log_dual = t->dual_clip > 0.f ? (float)std::log((double)t->dual_clip) : INFINITY;
  c.kl_coef = t->kl_coef, c.entropy_coef = t->entropy_coef;
  p->partials = static_cast<double*>(t->workspace);
  p->count_parts = reinterpret_cast<int64_t*>(p->partials + (int64_t)kMaxLossBlocks * kTerms);
  p->row_counts = reinterpret_cast<int*>(p->count_parts + kCountBlocks);
  Weights& w = p->weights;
  w.parts = nullptr, w.row_counts = nullptr, w.num_parts = 0, w.per_row = t->per_row != 0;
  const int64_t n = num_envs * seq_len;
  w.all = n > 0 ? (float)(1.0 / (double)n) : 0.f;  // (rows of one length: both means are the same)
  return RLK_OK;
}

int launch_count(const rlk_policy_terms* t, int64_t num_envs, int64_t seq_len, LossPlan* p, hipStream_t s) {
  if (t->mask == nullptr || num_envs * seq_len == 0) return RLK_OK;
  Weights& w = p->weights;
  const int64_t units = w.per_row ? (num_envs + kNT / 64 - 1) / (kNT / 64) : (num_envs * seq_len + kNT - 1) / kNT;
  const int blocks = (int)(units < kCountBlocks ? units : kCountBlocks);
  w.parts = p->count_parts, w.num_parts = blocks;
  if (w.per_row) w.row_counts = p->row_counts;
  if (t->bf16)
    count_kernel<bf16><<<dim3(blocks), dim3(kNT), 0, s>>>(static_cast<const bf16*>(t->mask), num_envs, seq_len, w.per_row,
                                                         p->count_parts, p->row_counts);
  else
    count_kernel<float><<<dim3(blocks), dim3(kNT), 0, s>>>(static_cast<const float*>(t->mask), num_envs, seq_len, w.per_row,
                                                          p->count_parts, p->row_counts);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

int launch_finish(const rlk_policy_terms* t, const LossPlan& p, int blocks, int means, hipStream_t s) {
  finish_kernel<<<dim3(1), dim3(kNT), 0, s>>>(p.partials, blocks, means, t->kl_coef, means > 4 ? t->entropy_coef : 0.f,
                                              t->loss, t->means);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

}  // namespace rlk

using namespace rlk;

extern "C" {

size_t rlk_policy_workspace_bytes(int64_t num_envs) {
  const size_t rows = num_envs > 0 ? (size_t)num_envs : 0;
  return sizeof(double) * kMaxLossBlocks * kTerms + sizeof(int64_t) * kCountBlocks + (sizeof(int) * rows + 7) / 8 * 8;
}

int rlk_policy_loss(const void* log_probs, int64_t num_envs, int64_t seq_len, const rlk_policy_terms* terms,
                    void* grad_log_probs, void* stream) {
  if (!terms) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return terms->bf16 ? loss_impl<bf16>(log_probs, num_envs, seq_len, terms, grad_log_probs, s)
                     : loss_impl<float>(log_probs, num_envs, seq_len, terms, grad_log_probs, s);
}

}  // extern "C"
