// rlk_logits_loss.hip -- the clipped policy loss from logits and the logits' gradient in one pass over them
// (include/rl_triton_policy.h; the mathematics is in rlk_action_rows.hpp and rlk_policy.hpp).
// Bound by HBM where rows are long: [16,512] of 65536 bfloat16 378 us a call, 5.7 TB/s of reads and writes, [7,285] of 50001
// float32 139, 5.7 TB/s (a large copy 5.2).  [4096,128] of 18 float32: 22 to 23 us, 3.6 TB/s (floor 16), bfloat16 21 (8): a tile of
// 256 rows is loaded, computed on and stored in turn, two of them a workgroup.  Counters: the vector units are busy for 43% of the time that
// a CU has work (18 of the 23 us), wavefronts wait for 70% of theirs, for memory and for each other; LDS conflicts are 1%.
#include "rlk_action_rows.hpp"

namespace rlk {
namespace {

struct StepArrays {
  const float *old, *adv, *ref, *mask;
};

template <class E, int LANES, int NV>
__global__ __launch_bounds__(rows_threads<LANES>()) void logits_loss_kernel(const ActionRows<E> a, const StepArrays t,
                                                                             const LossConsts c, const Weights w,
                                                                             const LossOut sums, E* __restrict__ grad) {
  constexpr int NT = rows_threads<LANES>(), PER = NT / LANES;
  __shared__ float lds[LANES > 64 ? 3 * (LANES / 64) + 2 : 1];
  __shared__ int64_t sc[NT / 64];
  const float scale = weight_scale<NT>(w, sc);
  const int lane = threadIdx.x % LANES;
  // (a workgroup's rows: one thread adds, and in LDS, since the held row needs the registers)
  __shared__ double total[kTerms];
  double acc[kTerms] = {};
  if (LANES > 64 && threadIdx.x < kTerms) total[threadIdx.x] = 0.0;
  __syncthreads();
  for (int64_t row = first_row<LANES>(); row < a.rows; row += (int64_t)gridDim.x * PER) {
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
      r = streamed_stats<E, LANES>(f, lane, a.c, lds, Part{0, f.nfull, true});
    }
    const float entropy = r.entropy();
    const StepTerms st = step_terms(r.log_prob(x, a.c), t.old[row], t.adv[row], t.ref ? t.ref[row] : 0.f, t.ref != nullptr, c);
    const RowGrad g(wt * st.slope, -(float)c.entropy_coef * wt, entropy, r.m, a.c, r.log2s(), a.inv_tau, act, r.empty());
    if constexpr (NV > 0)
      write_grad<E, LANES, NV>(f, &h, out, g, lane, Part{0, f.nfull, true});
    else
      write_grad<E, LANES, 0>(f, nullptr, out, g, lane, Part{0, f.nfull, true});
    if (lane == 0) {
      if constexpr (LANES > 64) {
        add_terms(total, st, wt);
        total[4] += (double)(wt * entropy);
      } else {
        add_terms(acc, st, wt);
        acc[4] += (double)(wt * entropy);
      }
    }
    if constexpr (LANES > 64) __syncthreads();
  }
  if constexpr (LANES > 64) {
    if (threadIdx.x == 0)
#pragma unroll
      for (int k = 0; k < kTerms; ++k) acc[k] = total[k];
  }
  finish_loss<NT>(acc, c, sums);
}

// The second launch for rows that several workgroups share: the loss by the first part's, the gradient by each for its own.
template <class E>
__global__ __launch_bounds__(256) void join_loss_kernel(const ActionRows<E> a, const RowParts p, const StepArrays t, const LossConsts c,
                                                        const Weights w, const LossOut sums, E* __restrict__ grad) {
  __shared__ int64_t sc[4];
  const float scale = weight_scale<256>(w, sc);
  double acc[kTerms] = {};
  const int part = blockIdx.x % p.parts;
  const int64_t row = blockIdx.x / p.parts;
  E* out = grad + row * a.A;
  if (t.mask != nullptr && t.mask[row] == 0.f) {
    write_zeros<E, 256>(out, a.A, threadIdx.x, part, p.parts);
  } else {
    const float wt = w.row_counts != nullptr ? scale / (float)w.row_counts[row / a.seq_len] : scale;
    const Frame<E> f(row_base(a, row), a.A);
    const int64_t act = a.actions[row];
    const float x = act >= 0 && act < a.A ? load_one(f.base + act) : NAN;
    const RowStats r = join_parts(p, row, a.c);
    const float entropy = r.entropy();
    const StepTerms st = step_terms(r.log_prob(x, a.c), t.old[row], t.adv[row], t.ref ? t.ref[row] : 0.f, t.ref != nullptr, c);
    const RowGrad g(wt * st.slope, -(float)c.entropy_coef * wt, entropy, r.m, a.c, r.log2s(), a.inv_tau, act, r.empty());
    write_grad<E, 256, 0>(f, nullptr, out, g, threadIdx.x, p.part(part, f.nfull));
    if (threadIdx.x == 0 && part == 0) {
      add_terms(acc, st, wt);
      acc[4] = (double)(wt * entropy);
    }
  }
  finish_loss<256>(acc, c, sums);
}

template <class E, int K>
__global__ __launch_bounds__(kFewRows) void few_loss_kernel(const ActionRows<E> a, const FewRows f, const StepArrays t,
                                                            const LossConsts c, const Weights w, const LossOut sums,
                                                            E* __restrict__ grad) {
  extern __shared__ __align__(16) float lds[];
  __shared__ int64_t sc[kFewRows / 64];
  const float scale = weight_scale<kFewRows>(w, sc);
  double acc[kTerms] = {};
  for (int64_t row0 = (int64_t)blockIdx.x * kFewRows; row0 < a.rows; row0 += (int64_t)gridDim.x * kFewRows) {
    const int rows = (int)(a.rows - row0 < kFewRows ? a.rows - row0 : kFewRows);
    const int64_t row = row0 + threadIdx.x;
    const bool mine = (int)threadIdx.x < rows, kept = mine && (t.mask == nullptr || t.mask[row] != 0.f);
    int64_t act = 0;
    float old = 0.f, adv = 0.f, ref = 0.f, wt = scale;
    if (kept) {
      act = a.actions[row], old = t.old[row], adv = t.adv[row];
      if (t.ref) ref = t.ref[row];
      if (w.row_counts != nullptr) wt = scale / (float)w.row_counts[row / a.seq_len];
    }
    f.take(a.logits + row0 * a.A, rows * a.A, lds);
    __syncthreads();
    float* x = lds + threadIdx.x * f.pitch;
    if (kept) {
      FewLogits<K> h;
      h.load(x, a.A);
      const RowStats r = h.stats(a.c);
      const float xa = act >= 0 && act < a.A ? x[act] : NAN;
      const float entropy = r.entropy();
      const StepTerms st = step_terms(r.log_prob(xa, a.c), old, adv, ref, t.ref != nullptr, c);
      const RowGrad g(wt * st.slope, -(float)c.entropy_coef * wt, entropy, r.m, a.c, r.log2s(), a.inv_tau, act, r.empty());
      if (__any(r.empty())) {
#pragma unroll
        for (int j = 0; j < K; ++j) h.x[j] = r.empty() ? 0.f : g(h.x[j], j);
        h.store(x, a.A);
      } else {
#pragma unroll
        for (int j = 0; j < K; ++j) h.x[j] = g(h.x[j]);
        h.store(x, a.A);
        asm volatile("" ::: "memory");  // (the stores are of another type: the compiler might exchange them)
        if (g.action >= 0 && g.action < a.A) x[g.action] += g.at;
      }
      add_terms(acc, st, wt);
      acc[4] += (double)(wt * entropy);
    } else if (mine) {
      for (int j = 0; j < a.A; ++j) x[j] = 0.f;
    }
    __syncthreads();
    f.put(grad + row0 * a.A, rows * a.A, lds);
    __syncthreads();
  }
  finish_loss<kFewRows>(acc, c, sums);
}

template <class E>
int impl(const rlk_action_rows* rows, const rlk_policy_terms* t, void* grad, hipStream_t s) {
  LossPlan plan;
  int st = plan_loss(t, rows->num_envs, rows->seq_len, kTerms, &plan);
  if (st != RLK_OK) return st;
  const ActionRows<E> a = action_rows<E>(rows);
  if (a.rows == 0) return launch_no_steps(plan, s);
  if (!grad) return RLK_ERR_INVALID_ARGUMENT;
  if ((st = launch_count(t, rows->num_envs, rows->seq_len, &plan, s)) != RLK_OK) return st;
  const StepArrays arrays{static_cast<const float*>(t->old_log_probs), static_cast<const float*>(t->advantages),
                          static_cast<const float*>(t->ref_log_probs), static_cast<const float*>(t->mask)};
  FewRows few;
  if (few_rows(a, grad, &few)) {
    int64_t blocks = (a.rows + kFewRows - 1) / kFewRows;
    // Two tiles a workgroup and more where LDS would hold a workgroup for every tile: one's loads go on beside another's
    // sums ([4096,128], in a graph: 2 actions 17.2 -> 13.7 us, 18 28.7 -> 24.7; 28, of which fewer fit, 37.7 and 38.3).
    const int64_t most = a.A <= 24 ? 1024 : kMaxLossBlocks;
    if (blocks > most) blocks = most;
    return dispatch_few(a.A, [&](auto k) {
      few_loss_kernel<E, decltype(k)::value><<<dim3((unsigned)blocks), dim3(kFewRows), FewRows::bytes(few.pitch), s>>>(
          a, few, arrays, plan.consts, plan.weights, plan.out, static_cast<E*>(grad));
      return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
    });
  }
  constexpr int VEC = Frame<E>::VEC;
  const RowParts parts = plan_parts(a.rows, (a.A + VEC - 1) / VEC, true, plan.shares, kShareBytes);
  if (parts.parts > 0) {
    const dim3 grid((unsigned)(a.rows * parts.parts));
    part_stats_kernel<E><<<grid, dim3(256), 0, s>>>(a, parts, arrays.mask);
    join_loss_kernel<E><<<grid, dim3(256), 0, s>>>(a, parts, arrays, plan.consts, plan.weights, plan.out, static_cast<E*>(grad));
    return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
  }
  return dispatch_update((a.A + VEC - 1) / VEC, [&](auto lanes, auto nv, int64_t most) {
    constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value, NT = rows_threads<L>();
    int64_t blocks = (a.rows + NT / L - 1) / (NT / L);
    if (blocks > most) blocks = most;
    logits_loss_kernel<E, L, NV><<<dim3((unsigned)blocks), dim3(NT), 0, s>>>(a, arrays, plan.consts, plan.weights, plan.out,
                                                                           static_cast<E*>(grad));
    return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
  });
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
