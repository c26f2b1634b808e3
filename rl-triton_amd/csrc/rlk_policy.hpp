// rlk_policy.hpp -- what the learner's operators share: 16-byte vectors of either storage type, group and
// workgroup reductions, the policy loss's terms, and the weights of its mean.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "rl_triton_policy.h"
#include "rlk_ops.hpp"

namespace rlk {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// N consecutive elements of E as they are stored, in words.
template <class E>
struct Words;
template <>
struct Words<float> {
  static constexpr int kPerWord = 1;
  __device__ static float get(uint32_t w, int) { return __uint_as_float(w); }
  __device__ static uint32_t put(float a, float) { return __float_as_uint(a); }
};
template <>
struct Words<bf16> {
  static constexpr int kPerWord = 2;
  __device__ static float get(uint32_t w, int i) { return __uint_as_float(i == 0 ? w << 16 : w & 0xffff0000u); }
  __device__ static uint32_t put(float a, float b) { return pack_bf16x2(a, b); }
};

__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const bf16* p) { return to_f32(*p); }

// The sum of `x` over a workgroup of NT threads, in a fixed order, in every thread.  `s`: NT / 64 elements.
template <int NT, class T>
__device__ __forceinline__ T block_sum(T x, T* s) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
  if constexpr (NT == 64) return x;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  T r = s[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) r += s[i];
  return r;
}

// ---------------------------------------------------------------------------------------
// The policy loss, step by step.
//
// With D = log pi - log pi_old, r = e^D and advantage A the loss of a step is max(-A r, -A clip(r)).  The
// maximum takes the clipped side only where A > 0 and r is above, or A < 0 and r below; which side is told by
// comparing D with the logarithms of the bounds, so no rounding of the exponential decides it.  On the
// clipped side, and where the dual clip caps it, the gradient is zero, elsewhere d/d(log pi) = -A r.  The KL
// term is e^d - 1 - d with d = log pi_ref - log pi, derivative 1 - e^d.
// ---------------------------------------------------------------------------------------

// The bounds come as two floats each: terms of both signs leave a loss that is far smaller than they are, and a bound rounded
// to one float is off alike in every step that it holds.  Their logarithms are one float each: a D that differs from one by
// less than its rounding differs in the term by no more.
struct LossConsts {
  float log_low, log_high, log_dual;  // thresholds of D; log_dual = inf: no cap
  float low, high, dual;              // the bounds, and what float32 leaves out of them
  float low_rest, high_rest, dual_rest;
  float kl;  // kl_coef
  double kl_coef, entropy_coef;
};

constexpr int kTerms = 5;  // policy, KL, clipped share, KL to the old policy, entropy

struct StepTerms {
  float policy, kl, clipped, old_kl;
  float slope;
};

// Adds a step's terms with weight w.
__device__ __forceinline__ void add_terms(double (&acc)[5], const StepTerms& t, float w) {
  acc[0] += (double)w * (double)t.policy;
  acc[1] += (double)(w * t.kl), acc[2] += (double)(w * t.clipped), acc[3] += (double)(w * t.old_kl);
}

// e^x - 1 - x >= 0 without the cancellation near zero: its series up to 1/2 in size (the first dropped
// term is below 2^-25 of the sum), the plain difference beyond, where it loses at most two bits.  From 64 on e^x is all that
// float32 holds of it (and infinity is, where the difference would be NaN).
__device__ __forceinline__ float exp_minus_linear(float x, float ex) {
  float p = 1.f / 362880.f;
  p = fmaf(p, x, 1.f / 40320.f);
  p = fmaf(p, x, 1.f / 5040.f);
  p = fmaf(p, x, 1.f / 720.f);
  p = fmaf(p, x, 1.f / 120.f);
  p = fmaf(p, x, 1.f / 24.f);
  p = fmaf(p, x, 1.f / 6.f);
  p = fmaf(p, x, 0.5f);
  return fabsf(x) < 0.5f ? p * x * x : x > 64.f ? ex : (ex - 1.f) - x;
}

__device__ __forceinline__ StepTerms step_terms(float lp, float old, float adv, float ref, bool has_ref,
                                                const LossConsts& c) {
  StepTerms t;
  const float d = lp - old;
  const float r = expf(d);
  const bool up = d > c.log_high && adv > 0.f, down = d < c.log_low && adv < 0.f;
  const bool cap = d > c.log_dual && adv < 0.f;
  const bool flat = up || down || cap;
  const float held = cap ? c.dual : up ? c.high : down ? c.low : r;
  const float rest = cap ? c.dual_rest : up ? c.high_rest : down ? c.low_rest : 0.f;
  t.policy = -fmaf(adv, held, adv * rest);
  t.slope = flat ? 0.f : -adv * r;
  t.clipped = flat ? 1.f : 0.f;
  t.old_kl = exp_minus_linear(d, r);
  t.kl = 0.f;
  if (has_ref) {
    const float e = ref - lp;
    const float ee = expf(e);
    t.kl = exp_minus_linear(e, ee);
    // e^e - 1: from the series near zero, else as it stands.  A reference far below (-inf: an action that it forbids) has a KL term
    // that holds nothing but -e, from which it could not be had again.  Without a coefficient there is none to follow.
    if (c.kl != 0.f) t.slope -= c.kl * (fabsf(e) < 0.5f ? t.kl + e : ee - 1.f);
  }
  return t;
}

// ---------------------------------------------------------------------------------------
// Weights of the mean.  `steps`: 1 / (number of steps that take part).  `rows`: 1 / (n_row * rows with any).
// With a mask these numbers come from count_kernel: a number per row, and per workgroup the sums of what
// the mean divides by, which every workgroup that needs them adds up in the same order (whole numbers: exact).
// ---------------------------------------------------------------------------------------
constexpr int kCountBlocks = 512;

struct Weights {
  const int64_t* parts;  // [kCountBlocks], or NULL: no mask
  const int* row_counts;  // [num_envs] (per_row with a mask)
  int num_parts;
  int per_row;
  float all;  // without a mask: every step's weight
};

// What all steps' weights have in common, in every thread of the workgroup.
template <int NT>
__device__ __forceinline__ float weight_scale(const Weights& w, int64_t* s) {
  if (w.parts == nullptr) return w.all;
  int64_t n = 0;
  for (int i = threadIdx.x; i < w.num_parts; i += NT) n += w.parts[i];
  n = block_sum<NT>(n, s);
  return n > 0 ? (float)(1.0 / (double)n) : 0.f;
}

// Partial sums of the loss's terms: one set of kTerms doubles per workgroup, at most this many.
constexpr int kMaxLossBlocks = 2048, kPartials = 8;  // (64 bytes each)

// The workgroups draw tickets in this many groups, and the last of each group draws one of the groups: 1024 draws
// from one word took 10 us more than the kernel around them.
constexpr int kTicketGroups = 32, kTicketStride = 16;
constexpr size_t kTicketBytes = (kTicketGroups + 1) * kTicketStride * sizeof(uint32_t);

// Where a call's sums meet and what they become.
struct LossOut {
  double* partials;  // [workgroups, kPartials]
  uint32_t* tickets;  // [kTicketGroups + 1], kTicketStride apart, 0 between calls
  float *loss, *means;
  int num_means;
};

struct LossPlan {
  LossConsts consts;
  Weights weights;
  LossOut out;
  int64_t* count_parts;
  int* row_counts;
  void* shares;  // kShareBytes for rows of logits that several workgroups share
};
constexpr size_t kShareBytes = RLK_ROWS_WORKSPACE_BYTES;

// Checks the terms and lays out the workspace; RLK_OK or an error.
int plan_loss(const rlk_policy_terms* t, int64_t num_envs, int64_t seq_len, int means, LossPlan* plan);
// Counts the steps that take part (when there is a mask).
int launch_count(const rlk_policy_terms* t, int64_t num_envs, int64_t seq_len, LossPlan* plan, hipStream_t s);
// Writes the loss and means of no steps: zeros.
int launch_no_steps(const LossPlan& plan, hipStream_t s);

// The sums of kTerms doubles over a workgroup of NT threads: term k in thread k.  `s`: NT / 64 * kTerms.  At each of the first
// three exchanges a lane keeps half of its terms and hands over the others: 10 additions and not 30 for the wavefront.
template <int NT>
__device__ __forceinline__ double sum_terms(const double (&v)[kTerms], double* s) {
  static_assert(kTerms <= 8);
  const int lane = threadIdx.x & 63;
  double w[4];
  const bool b5 = lane & 32, b4 = lane & 16, b3 = lane & 8;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const double high = 4 + k < kTerms ? v[4 + k < kTerms ? 4 + k : 0] : 0.0;
    w[k] = (b5 ? high : v[k]) + __shfl_xor(b5 ? v[k] : high, 32);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) w[k] = (b4 ? w[2 + k] : w[k]) + __shfl_xor(b4 ? w[k] : w[2 + k], 16);
  double x = (b3 ? w[1] : w[0]) + __shfl_xor(b3 ? w[0] : w[1], 8);
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) x += __shfl_xor(x, d);
  const int term = (b5 ? 4 : 0) + (b4 ? 2 : 0) + (b3 ? 1 : 0);
  __syncthreads();
  if ((lane & 7) == 0 && term < kTerms) s[(threadIdx.x >> 6) * kTerms + term] = x;
  __syncthreads();
  x = 0.0;
  if (threadIdx.x < kTerms)
    for (int i = 0; i < NT / 64; ++i) x += s[i * kTerms + threadIdx.x];
  return x;
}

// The end of a loss kernel: the workgroups' sums, and from the last one to arrive the loss and the means, added up in the
// workgroups' order whichever that is.  (A launch of its own for that took 2.7 us and a gap.)  The sums go through stores
// and loads at agent scope, which every XCD sees, and are complete before the ticket is drawn: the wait is all the order
// that takes.  A release at the ticket would also write back the L2's gradients, once per workgroup ([512,6000] 47 us of a
// kernel that takes 11).
template <int NT>
__device__ __forceinline__ void finish_loss(const double (&acc)[kTerms], const LossConsts& c, const LossOut& o) {
  __shared__ double s[NT / 64 * kTerms];
  __shared__ bool last;
  double x = sum_terms<NT>(acc, s);
  if (gridDim.x > 1) {
    if (threadIdx.x < kTerms)
      __hip_atomic_store(o.partials + (int64_t)blockIdx.x * kPartials + threadIdx.x, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (threadIdx.x == 0) {
      const uint32_t group = blockIdx.x % kTicketGroups, members = (gridDim.x - group + kTicketGroups - 1) / kTicketGroups;
      const bool grouped = gridDim.x > kTicketGroups;
      const uint32_t groups = grouped ? kTicketGroups : gridDim.x;
      uint32_t *mine = o.tickets + group * kTicketStride, *all = o.tickets + kTicketGroups * kTicketStride;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the wavefront's stores: the sums' among them)
      last = (!grouped || __hip_atomic_fetch_add(mine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == members - 1) &&
             __hip_atomic_fetch_add(all, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
    }
    __syncthreads();
    if (!last) return;
    double v[kTerms] = {};
    for (int b = threadIdx.x; b < (int)gridDim.x; b += NT)
#pragma unroll
      for (int k = 0; k < kTerms; ++k)
        v[k] += __hip_atomic_load(o.partials + (int64_t)b * kPartials + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = sum_terms<NT>(v, s);
    if (threadIdx.x <= kTicketGroups) o.tickets[threadIdx.x * kTicketStride] = 0;
  }
  if ((int)threadIdx.x < o.num_means) o.means[threadIdx.x] = (float)x;
  const double kl = __shfl(x, 1), entropy = __shfl(x, 4);
  // (a term without a coefficient has no part, infinite or not)
  if (threadIdx.x == 0) *o.loss = (float)(x + (c.kl_coef != 0.0 ? c.kl_coef * kl : 0.0) - (c.entropy_coef != 0.0 ? c.entropy_coef * entropy : 0.0));
}

}  // namespace rlk
