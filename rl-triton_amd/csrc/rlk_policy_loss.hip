// rlk_policy_loss.hip -- the clipped policy loss from log-probabilities, and the counting and summing that
// the loss from logits shares (include/rl_triton_policy.h).
//
// [512,6000] with mask, reference and row means: counts 4.7 us, loss 20.6 (floor 14 for both; bfloat16 the same, floor 7): two
// exponentials and two series a step keep the vector units busy for 57% of the time, then comes
// one exchange between workgroups through two levels of tickets.  [64,128]: 6.1 us, two loads' latencies, the reduction and the
// exchange.
#include "rlk_launch.hpp"
#include "rlk_policy.hpp"

namespace rlk {
namespace {

constexpr int kNT = 256;

// Four consecutive elements as floats; `whole`: one aligned access, else the `left` (1..4) that exist.
template <class E>
__device__ __forceinline__ float4 load4(const E* p, bool whole, int left) {
  if (whole) return load_quad<false>(p);
  return {load_one(p), left > 1 ? load_one(p + 1) : 0.f, left > 2 ? load_one(p + 2) : 0.f, left > 3 ? load_one(p + 3) : 0.f};
}

// What the mean divides by: the steps with mask != 0 or, per_row, the rows that have any (and each row's number: a
// wavefront per row for short rows, the workgroup for others).
template <class E, int ROW_LANES>  // 0: steps
__global__ __launch_bounds__(kNT) void count_kernel(const E* __restrict__ mask, int64_t num_envs, int64_t seq_len, bool whole,
                                                    int64_t* __restrict__ parts, int* __restrict__ row_counts) {
  __shared__ int64_t s[kNT / 64];
  __shared__ int part[2][kNT / 64];
  int64_t total = 0;
  auto kept = [](float4 m) { return (m.x != 0.f) + (m.y != 0.f) + (m.z != 0.f) + (m.w != 0.f); };
  if constexpr (ROW_LANES == 0) {
    const int64_t n = num_envs * seq_len, step = (int64_t)gridDim.x * kNT * 4;
    for (int64_t i = ((int64_t)blockIdx.x * kNT + threadIdx.x) * 4; i < n; i += step) {
      const int left = (int)(n - i < 4 ? n - i : 4);
      total += kept(load4(mask + i, whole && left == 4, left));
    }
  } else {
    constexpr int PER = kNT / ROW_LANES;
    const int lane = threadIdx.x % ROW_LANES;
    int turn = 0;
    for (int64_t e = (int64_t)blockIdx.x * PER + threadIdx.x / ROW_LANES; e < num_envs; e += (int64_t)gridDim.x * PER) {
      const E* row = mask + e * seq_len;
      int n = 0;
      for (int64_t t = lane * 4; t < seq_len; t += ROW_LANES * 4) {
        const int left = (int)(seq_len - t < 4 ? seq_len - t : 4);
        n += kept(load4(row + t, whole && left == 4, left));
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
      if constexpr (ROW_LANES > 64) {
        if ((threadIdx.x & 63) == 0) part[turn][threadIdx.x >> 6] = n;
        __syncthreads();
        n = 0;
        for (int i = 0; i < kNT / 64; ++i) n += part[turn][i];
        turn ^= 1;
      }
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
  bool whole;  // arrays aligned to 4 elements
  LossConsts c;
  Weights w;
  LossOut out;
};

// Steps i .. i + 3 (`left` of them exist).
struct FourSteps {
  float4 lp, old, adv, ref;
  template <class E>
  __device__ __forceinline__ void load(const LossArgs<E>& a, int64_t i, int left) {
    const bool whole = a.whole && left == 4;
    lp = load4(a.lp + i, whole, left), old = load4(a.old + i, whole, left), adv = load4(a.adv + i, whole, left);
    ref = a.ref ? load4(a.ref + i, whole, left) : float4{0.f, 0.f, 0.f, 0.f};
  }
};

// Their gradients, their terms added to `acc`.  weight(step, which of the four): what it counts for.
template <class E, class F>
__device__ __forceinline__ void four_steps(const LossArgs<E>& a, const FourSteps& x4, int64_t i, int left, float4 m, double (&acc)[kTerms],
                                           F weight) {
  const bool whole = a.whole && left == 4;
  const float4 &lp = x4.lp, &old = x4.old, &adv = x4.adv, &ref = x4.ref;
  float g[4], policy = 0.f, kl = 0.f, clipped = 0.f, old_kl = 0.f;
  const float *pl = &lp.x, *po = &old.x, *pa = &adv.x, *pr = &ref.x, *pm = &m.x;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    g[x] = 0.f;
    if (pm[x] != 0.f && x < left) {
      const float w = weight(i, x);
      const StepTerms t = step_terms(pl[x], po[x], pa[x], pr[x], a.ref != nullptr, a.c);
      policy = fmaf(w, t.policy, policy);
      kl = fmaf(w, t.kl, kl), clipped = fmaf(w, t.clipped, clipped), old_kl = fmaf(w, t.old_kl, old_kl);
      g[x] = w * t.slope;
    }
  }
  acc[0] += policy, acc[1] += kl, acc[2] += clipped, acc[3] += old_kl;
  if (whole) {
    store_quad(a.grad + i, float4{g[0], g[1], g[2], g[3]});
  } else {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (x < left) a.grad[i + x] = from_f32<E>(g[x]);
  }
}

constexpr float4 kAll{1.f, 1.f, 1.f, 1.f};

template <class E>
__global__ __launch_bounds__(kNT) void loss_kernel(const LossArgs<E> a) {
  __shared__ int64_t sc[kNT / 64];
  const int64_t step = (int64_t)gridDim.x * kNT * 4;
  int64_t i = ((int64_t)blockIdx.x * kNT + threadIdx.x) * 4;
  float4 m = kAll;
  FourSteps x;
  auto load = [&](int64_t at) {
    const int left = (int)(a.n - at < 4 ? a.n - at : 4);
    if (a.mask) m = load4(a.mask + at, a.whole && left == 4, left);
    x.load(a, at, left);
  };
  if (i < a.n) load(i);  // (on their way while the counts are added up)
  const float scale = weight_scale<kNT>(a.w, sc);
  double acc[kTerms] = {};
  for (; i < a.n; i += step) {
    const int left = (int)(a.n - i < 4 ? a.n - i : 4);
    if (a.w.row_counts == nullptr) {
      four_steps(a, x, i, left, m, acc, [&](int64_t, int) { return scale; });
    } else {
      int64_t row = a.n <= 0x7fffffff ? (int64_t)((uint32_t)i / (uint32_t)a.seq_len) : i / a.seq_len;
      int64_t ends = (row + 1) * a.seq_len;
      float w = scale / (float)a.w.row_counts[row];  // (a row of none is asked for nothing)
      four_steps(a, x, i, left, m, acc, [&](int64_t at, int which) {
        while (at + which >= ends) w = scale / (float)a.w.row_counts[++row], ends += a.seq_len;
        return w;
      });
    }
    if (i + step < a.n) load(i + step);
  }
  finish_loss<kNT>(acc, a.c, a.out);
}

// Small masked calls: one workgroup counts, computes and sums, in one launch ([16,128] 8.8 us in a graph, 10.7 in two; at
// [32,128] 10.3 and 10.7, at [64,128] 13.1 and 10.9).  Without a mask there is nothing to count, and loss_kernel is one launch.
constexpr int kSmallNT = 512, kSmallSteps = 4 * kSmallNT;

template <class E>
__global__ __launch_bounds__(kSmallNT) void small_loss_kernel(const LossArgs<E> a) {
  __shared__ int counts[kSmallSteps];
  __shared__ int sums[kSmallNT / 64];
  const int n = (int)a.n, T = (int)a.seq_len, i = 4 * threadIdx.x, left = n - i < 4 ? n - i : 4;
  const bool rows = a.w.per_row;
  float4 m{0.f, 0.f, 0.f, 0.f};
  if (i < n) m = load4(a.mask + i, a.whole && left == 4, left);
  int count = 0;
  if (rows) {
    for (int e = threadIdx.x; e * T < n; e += kSmallNT) counts[e] = 0;
    __syncthreads();
  }
  const float* pm = &m.x;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (pm[x] != 0.f) {
      if (rows) atomicAdd(&counts[(i + x) / T], 1);
      else ++count;
    }
  if (rows) {
    __syncthreads();
    for (int e = threadIdx.x; e * T < n; e += kSmallNT) count += counts[e] > 0;
  }
  count = block_sum<kSmallNT>(count, sums);
  const float scale = count > 0 ? 1.f / (float)count : 0.f;
  double acc[kTerms] = {};
  if (i < n) {
    FourSteps x;
    x.load(a, i, left);
    four_steps(a, x, i, left, m, acc, [&](int64_t at, int which) { return rows ? scale / (float)counts[((int)at + which) / T] : scale; });
  }
  finish_loss<kSmallNT>(acc, a.c, a.out);
}

__global__ void no_steps_kernel(LossOut o) {
  if (threadIdx.x == 0) *o.loss = 0.f;
  if ((int)threadIdx.x < o.num_means) o.means[threadIdx.x] = 0.f;
}

template <class E>
int loss_impl(const void* lp, int64_t E_, int64_t T, const rlk_policy_terms* t, void* grad, hipStream_t s) {
  LossPlan plan;
  int st = plan_loss(t, E_, T, 4, &plan);
  if (st != RLK_OK) return st;
  const int64_t n = E_ * T;
  if (n == 0) return launch_no_steps(plan, s);
  if (!lp || !grad) return RLK_ERR_INVALID_ARGUMENT;
  LossArgs<E> a{static_cast<const E*>(lp), static_cast<const E*>(t->old_log_probs), static_cast<const E*>(t->advantages),
                static_cast<const E*>(t->ref_log_probs), static_cast<const E*>(t->mask), static_cast<E*>(grad),
                n, T, false, plan.consts, plan.weights, plan.out};
  a.whole = quad_aligned(a.lp, a.old, a.adv, a.ref, a.mask, a.grad);
  a.c.entropy_coef = 0.0;  // (there are no entropies here)
  if (t->mask && n <= kSmallSteps) {
    small_loss_kernel<E><<<dim3(1), dim3(kSmallNT), 0, s>>>(a);
  } else {
    if ((st = launch_count(t, E_, T, &plan, s)) != RLK_OK) return st;
    a.w = plan.weights;
    // as many rounds as the most workgroups need, and as many workgroups as fill them
    // (4 workgroups a CU, each with as many rounds as it takes: [2048,2048] masked 28.6 us, 31.2 with up to 8; [4096,8192] 109 and 125)
    const int64_t most = 1024, units = (n + kNT * 4 - 1) / (kNT * 4), rounds = (units + most - 1) / most;
    loss_kernel<E><<<dim3((unsigned)((units + rounds - 1) / rounds)), dim3(kNT), 0, s>>>(a);
  }
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

template <class E>
int count_impl(const rlk_policy_terms* t, int64_t E_, int64_t T, LossPlan* p, hipStream_t s) {
  const E* mask = static_cast<const E*>(t->mask);
  Weights& w = p->weights;
  const bool whole = quad_aligned(mask) && (!w.per_row || T % 4 == 0);
  // a workgroup per row from rows that give each of its threads a quad
  const bool wide = T >= kNT * 4;
  const int64_t units = !w.per_row ? (E_ * T + kNT * 4 - 1) / (kNT * 4) : wide ? E_ : (E_ + kNT / 64 - 1) / (kNT / 64);
  const int blocks = (int)(units < kCountBlocks ? units : kCountBlocks);
  w.parts = p->count_parts, w.num_parts = blocks;
  if (w.per_row) w.row_counts = p->row_counts;
  const dim3 grid(blocks), block(kNT);
  if (!w.per_row) count_kernel<E, 0><<<grid, block, 0, s>>>(mask, E_, T, whole, p->count_parts, p->row_counts);
  else if (wide) count_kernel<E, kNT><<<grid, block, 0, s>>>(mask, E_, T, whole, p->count_parts, p->row_counts);
  else count_kernel<E, 64><<<grid, block, 0, s>>>(mask, E_, T, whole, p->count_parts, p->row_counts);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

}  // namespace

int plan_loss(const rlk_policy_terms* t, int64_t num_envs, int64_t seq_len, int means, LossPlan* p) {
  if (!t || num_envs < 0 || seq_len < 0 || !t->loss || !t->means) return RLK_ERR_INVALID_ARGUMENT;
  if (num_envs * seq_len > 0 && (!t->old_log_probs || !t->advantages)) return RLK_ERR_INVALID_ARGUMENT;
  if (!(t->clip_low >= 0.0) || !(t->clip_high >= 0.0) || !(t->dual_clip == 0.0 || t->dual_clip > 1.0))
    return RLK_ERR_INVALID_ARGUMENT;
  if (seq_len > (int64_t{1} << 30)) return RLK_ERR_INVALID_ARGUMENT;  // (a row's count is an int)
  if (!t->workspace || t->workspace_bytes < rlk_policy_workspace_bytes(num_envs) ||
      (reinterpret_cast<uintptr_t>(t->workspace) & 7u) != 0)
    return RLK_ERR_WORKSPACE;
  LossConsts& c = p->consts;
  const double low = 1.0 - t->clip_low, high = 1.0 + t->clip_high, dual = t->dual_clip;
  c.low = (float)low, c.high = (float)high, c.dual = (float)dual;
  c.low_rest = (float)(low - (double)c.low), c.high_rest = (float)(high - (double)c.high), c.dual_rest = (float)(dual - (double)c.dual);
  c.log_low = t->clip_low < 1.0 ? (float)std::log1p(-t->clip_low) : -INFINITY;
  c.log_high = (float)std::log1p(t->clip_high);
  c.log_dual = t->dual_clip > 0.0 ? (float)std::log(t->dual_clip) : INFINITY;
  c.kl = (float)t->kl_coef, c.kl_coef = t->kl_coef, c.entropy_coef = t->entropy_coef;
  char* ws = static_cast<char*>(t->workspace);
  p->out = {reinterpret_cast<double*>(ws + kTicketBytes), reinterpret_cast<uint32_t*>(ws), t->loss, t->means, means};
  p->count_parts = reinterpret_cast<int64_t*>(p->out.partials + (int64_t)kMaxLossBlocks * kPartials);
  p->shares = p->count_parts + kCountBlocks;
  p->row_counts = reinterpret_cast<int*>(static_cast<char*>(p->shares) + kShareBytes);
  Weights& w = p->weights;
  w.parts = nullptr, w.row_counts = nullptr, w.num_parts = 0, w.per_row = t->per_row != 0;
  const int64_t n = num_envs * seq_len;
  w.all = n > 0 ? (float)(1.0 / (double)n) : 0.f;  // (rows of one length: both means are the same)
  return RLK_OK;
}

int launch_count(const rlk_policy_terms* t, int64_t num_envs, int64_t seq_len, LossPlan* p, hipStream_t s) {
  if (t->mask == nullptr || num_envs * seq_len == 0) return RLK_OK;
  return t->bf16 ? count_impl<bf16>(t, num_envs, seq_len, p, s) : count_impl<float>(t, num_envs, seq_len, p, s);
}

int launch_no_steps(const LossPlan& p, hipStream_t s) {
  no_steps_kernel<<<dim3(1), dim3(64), 0, s>>>(p.out);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

}  // namespace rlk

using namespace rlk;

extern "C" {

size_t rlk_policy_workspace_bytes(int64_t num_envs) {
  const size_t rows = num_envs > 0 ? (size_t)num_envs : 0;
  return kTicketBytes + sizeof(double) * kMaxLossBlocks * kPartials + sizeof(int64_t) * kCountBlocks + kShareBytes +
         (sizeof(int) * rows + 7) / 8 * 8;
}

int rlk_policy_loss(const void* log_probs, int64_t num_envs, int64_t seq_len, const rlk_policy_terms* terms,
                    void* grad_log_probs, void* stream) {
  if (!terms) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return terms->bf16 ? loss_impl<bf16>(log_probs, num_envs, seq_len, terms, grad_log_probs, s)
                     : loss_impl<float>(log_probs, num_envs, seq_len, terms, grad_log_probs, s);
}

}  // extern "C"
