// rlk_logits_loss.hip -- the clipped policy loss from logits and the logits' gradient in one pass over them
// (include/rl_triton_policy.h; the mathematics is in rlk_action_rows.hpp and rlk_policy.hpp).
#include "rlk_action_rows.hpp"

namespace rlk {
namespace {

struct StepArrays {
  const float *old, *adv, *ref, *mask;
};

template <class E, int LANES, int NV>
__global__ __launch_bounds__(rows_threads<LANES>()) void logits_loss_kernel(const ActionRows<E> a, const StepArrays t,
                                                                             const LossConsts c, const Weights w,
                                                                             double* __restrict__ partials, E* __restrict__ grad) {
  constexpr int NT = rows_threads<LANES>(), PER = NT / LANES;
  __shared__ float lds[LANES > 64 ? 3 * (LANES / 64) + 2 : 1];
  __shared__ int64_t sc[NT / 64];
  __shared__ double sd[NT / 64];
  const float scale = weight_scale<NT>(w, sc);
  const int lane = threadIdx.x % LANES;
  float acc[kTerms] = {};
  for (int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / LANES; row < a.rows; row += (int64_t)gridDim.x * PER) {
    E* out = grad + row * a.A;
    if (t.mask != nullptr && t.mask[row] == 0.f) {  // (the same for the whole group)
      write_zeros<E, LANES>(out, a.A, lane);
      continue;
    }
    const float wt = w.row_counts != nullptr ? scale / (float)w.row_counts[row / a.seq_len] : scale;
    const Frame<E> f(row_base(a, row), a.A);
    const int64_t act = a.actions[row];
    const float x = act >= 0 && act < a.A ? load_one(f.base + act) : NAN;
    RowHolder<E, LANES, (NV > 0 ? NV : 1)> h;
    RowStats r;
    if constexpr (NV > 0) {
      h.load(f, lane);
      r = h.stats(f, lane, a.c, lds);
    } else {
      r = streamed_stats<E, LANES>(f, lane, a.c, lds);
    }
    const bool empty = r.s == 0.f;
    const float log2s = r.log2s();
    const float lp = empty && x == x ? -INFINITY : ((x - r.m) * a.c - log2s) * kLn2;
    const float entropy = empty ? 0.f : (log2s - r.u / r.s) * kLn2;
    const StepTerms st = step_terms(lp, t.old[row], t.adv[row], t.ref ? t.ref[row] : 0.f, t.ref != nullptr, c);
    const RowGrad g(wt * st.slope, -c.entropy_coef * wt, entropy, r.m, log2s, a.inv_tau, act, empty);
    if constexpr (NV > 0)
      write_grad<E, LANES, NV>(f, &h, out, g, a.c, lane);
    else
      write_grad<E, LANES, 0>(f, nullptr, out, g, a.c, lane);
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += wt * st.v[k];
      acc[4] += wt * entropy;
    }
    if constexpr (LANES > 64) __syncthreads();
  }
  write_partials<NT>(acc, partials, sd);
}

template <class E>
int impl(const rlk_action_rows* rows, const rlk_policy_terms* t, void* grad, hipStream_t s) {
  LossPlan plan;
  int st = plan_loss(t, rows->num_envs, rows->seq_len, &plan);
  if (st != RLK_OK) return st;
  const ActionRows<E> a = action_rows<E>(rows);
  if (a.rows == 0) return launch_finish(t, plan, 0, kTerms, s);
  if (!grad) return RLK_ERR_INVALID_ARGUMENT;
  if ((st = launch_count(t, rows->num_envs, rows->seq_len, &plan, s)) != RLK_OK) return st;
  const StepArrays arrays{static_cast<const float*>(t->old_log_probs), static_cast<const float*>(t->advantages),
                          static_cast<const float*>(t->ref_log_probs), static_cast<const float*>(t->mask)};
  constexpr int VEC = Frame<E>::VEC;
  int64_t blocks = 0;
  st = dispatch_row((a.A + VEC - 1) / VEC, [&](auto lanes, auto nv) {
    constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value, NT = rows_threads<L>();
    blocks = (a.rows + NT / L - 1) / (NT / L);
    if (blocks > kMaxLossBlocks) blocks = kMaxLossBlocks;
    logits_loss_kernel<E, L, NV><<<dim3((unsigned)blocks), dim3(NT), 0, s>>>(a, arrays, plan.consts, plan.weights, plan.partials,
                                                                           static_cast<E*>(grad));
    return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
  });
  return st != RLK_OK ? st : launch_finish(t, plan, (int)blocks, kTerms, s);
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" int rlk_policy_loss_from_logits(const rlk_action_rows* rows, const rlk_policy_terms* terms, void* grad_logits,
                                           void* stream) {
  if (!valid_rows(rows) || !terms || terms->bf16) return RLK_ERR_INVALID_ARGUMENT;  // (the step arrays are float)
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return rows->bf16 ? impl<bf16>(rows, terms, grad_logits, s) : impl<float>(rows, terms, grad_logits, s);
}
