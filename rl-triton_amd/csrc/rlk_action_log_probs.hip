// rlk_action_log_probs.hip -- log-probabilities and entropies of the taken actions
// (include/rl_triton_policy.h; the mathematics is in rlk_action_rows.hpp).
// Bound by HBM where rows are many and long ([16,1024] of 32768 bfloat16: 189 us, 5.7 TB/s read), by a launch and one
// load's latency where they are few ([256] of 18 float32: 2.6 us).
// Backward, nothing is reduced (the row's statistics were kept): one read and one write, at HBM's rate where rows are many
// and long ([16,1024] of 32768: bfloat16 382 us, float32 806, 5.3 TB/s), not elsewhere: [4096,128] of 18 27 us in either type (floors
// 8 and 15), a workgroup for each of [16] rows of 131072 40 (3), [512] of 300 3.4 and 4.6.
#include "rlk_action_rows.hpp"

namespace rlk {
namespace {

// What a row's statistics come to, and the logit of its action (NaN: there is no such action).
__device__ __forceinline__ void write_row(const RowStats& r, float x, float c, int64_t row, float* log_probs, float* entropies, float* norms) {
  log_probs[row] = r.log_prob(x, c);
  entropies[row] = r.entropy();
  if (norms) norms[2 * row] = r.m, norms[2 * row + 1] = r.empty() ? INFINITY : r.log2s();  // (inf: p = 0)
}
template <class E>
__device__ __forceinline__ void write_row(const ActionRows<E>& a, const E* base, int64_t row, const RowStats& r, float* log_probs,
                                          float* entropies, float* norms) {
  const int64_t act = a.actions[row];
  write_row(r, act >= 0 && act < a.A ? load_one(base + act) : NAN, a.c, row, log_probs, entropies, norms);
}

template <class E, int LANES, int NV>
__global__ __launch_bounds__(rows_threads<LANES>()) void log_probs_kernel(const ActionRows<E> a, float* __restrict__ log_probs,
                                                                           float* __restrict__ entropies,
                                                                           float* __restrict__ norms) {
  constexpr int NT = rows_threads<LANES>(), PER = NT / LANES;
  __shared__ float lds[LANES > 64 ? 3 * (LANES / 64) + 2 : 1];
  const int lane = threadIdx.x % LANES;
  for (int64_t row = first_row<LANES>(); row < a.rows; row += (int64_t)gridDim.x * PER) {
    const Frame<E> f(row_base(a, row), a.A);
    RowStats r;
    if constexpr (NV > 0) {
      RowHolder<E, LANES, NV> h;
      h.load(f, lane);
      r = h.stats(f, lane, a.c, lds);
    } else {
      r = streamed_stats<E, LANES>(f, lane, a.c, lds, Part{0, f.nfull, true});
    }
    if (lane == 0) write_row(a, f.base, row, r, log_probs, entropies, norms);
    if constexpr (LANES > 64) __syncthreads();
  }
}

template <class E>
__global__ __launch_bounds__(256) void join_log_probs_kernel(const ActionRows<E> a, const RowParts p, float* __restrict__ log_probs,
                                                             float* __restrict__ entropies, float* __restrict__ norms) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const RowStats r = join_parts(p, row, a.c);
  if ((threadIdx.x & 63) == 0) write_row(a, row_base(a, row), row, r, log_probs, entropies, norms);
}

template <class E, int K>
__global__ __launch_bounds__(kFewRows) void few_log_probs_kernel(const ActionRows<E> a, const FewRows f, float* __restrict__ log_probs,
                                                                 float* __restrict__ entropies, float* __restrict__ norms) {
  extern __shared__ __align__(16) float lds[];
  for (int64_t row0 = (int64_t)blockIdx.x * kFewRows; row0 < a.rows; row0 += (int64_t)gridDim.x * kFewRows) {
    const int rows = (int)(a.rows - row0 < kFewRows ? a.rows - row0 : kFewRows);
    const int64_t row = row0 + threadIdx.x;
    const int64_t act = (int)threadIdx.x < rows ? a.actions[row] : 0;
    f.take(a.logits + row0 * a.A, rows * a.A, lds);
    __syncthreads();
    if ((int)threadIdx.x < rows) {
      const float* mine = lds + threadIdx.x * f.pitch;
      FewLogits<K> h;
      h.load(mine, a.A);
      const RowStats r = h.stats(a.c);
      write_row(r, act >= 0 && act < a.A ? mine[act] : NAN, a.c, row, log_probs, entropies, norms);
    }
    __syncthreads();
  }
}

template <class E, int LANES>
__global__ __launch_bounds__(256) void backward_kernel(const ActionRows<E> a, const float* __restrict__ entropies,
                                                       const float* __restrict__ norms, const float* __restrict__ gl,
                                                       const float* __restrict__ ge, E* __restrict__ out) {
  constexpr int PER = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  for (int64_t row = first_row<LANES>(); row < a.rows; row += (int64_t)gridDim.x * PER) {
    const Frame<E> f(row_base(a, row), a.A);
    const float log2s = norms[2 * row + 1];
    const RowGrad g(gl ? gl[row] : 0.f, ge ? ge[row] : 0.f, entropies[row], norms[2 * row], a.c, log2s, a.inv_tau, a.actions[row],
                    log2s == INFINITY);
    write_grad<E, LANES, 0>(f, nullptr, out + row * a.A, g, lane, Part{0, f.nfull, true});
  }
}

template <class E>
int forward(const rlk_action_rows* rows, float* lp, float* ent, float* norms, hipStream_t s) {
  const ActionRows<E> a = action_rows<E>(rows);
  FewRows few;
  if (few_rows(a, nullptr, &few)) {
    int64_t blocks = (a.rows + kFewRows - 1) / kFewRows;
    if (blocks > 2048) blocks = 2048;
    return dispatch_few(a.A, [&](auto k) {
      few_log_probs_kernel<E, decltype(k)::value><<<dim3((unsigned)blocks), dim3(kFewRows), FewRows::bytes(few.pitch), s>>>(
          a, few, lp, ent, norms);
      return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
    });
  }
  constexpr int VEC = Frame<E>::VEC;
  const RowParts parts = plan_parts(a.rows, (a.A + VEC - 1) / VEC, false, rows->workspace, rows->workspace_bytes);
  if (parts.parts > 0) {
    part_stats_kernel<E><<<dim3((unsigned)(a.rows * parts.parts)), dim3(256), 0, s>>>(a, parts, nullptr);
    join_log_probs_kernel<E><<<dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s>>>(a, parts, lp, ent, norms);
    return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
  }
  return dispatch_read((a.A + VEC - 1) / VEC, a.rows, [&](auto lanes, auto nv, int64_t most) {
    constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value, NT = rows_threads<L>();
    int64_t blocks = (a.rows + NT / L - 1) / (NT / L);
    if (blocks > most) blocks = most;
    log_probs_kernel<E, L, NV><<<dim3((unsigned)blocks), dim3(NT), 0, s>>>(a, lp, ent, norms);
    return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
  });
}

template <class E>
int backward(const rlk_action_rows* rows, const float* ent, const float* norms, const float* gl, const float* ge, void* out,
             hipStream_t s) {
  const ActionRows<E> a = action_rows<E>(rows);
  constexpr int VEC = Frame<E>::VEC;
  const int64_t vecs = (a.A + VEC - 1) / VEC;
  auto run = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    int64_t blocks = (a.rows + 256 / L - 1) / (256 / L);
    if (blocks > 8192) blocks = 8192;
    backward_kernel<E, L><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(a, ent, norms, gl, ge, static_cast<E*>(out));
    return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
  };
  if (vecs <= 8) return run(std::integral_constant<int, 4>{});
  if (vecs <= 64) return run(std::integral_constant<int, 16>{});
  return run(std::integral_constant<int, 256>{});
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" {

int rlk_action_log_probs(const rlk_action_rows* rows, float* log_probs, float* entropies, float* norms, void* stream) {
  if (!valid_rows(rows)) return RLK_ERR_INVALID_ARGUMENT;
  if (rows->num_envs * rows->seq_len == 0) return RLK_OK;
  if (!log_probs || !entropies) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return rows->bf16 ? forward<bf16>(rows, log_probs, entropies, norms, s) : forward<float>(rows, log_probs, entropies, norms, s);
}

int rlk_action_log_probs_backward(const rlk_action_rows* rows, const float* entropies, const float* norms,
                                  const float* grad_log_probs, const float* grad_entropies, void* grad_logits, void* stream) {
  if (!valid_rows(rows)) return RLK_ERR_INVALID_ARGUMENT;
  if (rows->num_envs * rows->seq_len == 0) return RLK_OK;
  if (!entropies || !norms || !grad_logits) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return rows->bf16 ? backward<bf16>(rows, entropies, norms, grad_log_probs, grad_entropies, grad_logits, s)
                    : backward<float>(rows, entropies, norms, grad_log_probs, grad_entropies, grad_logits, s);
}

}  // extern "C"
