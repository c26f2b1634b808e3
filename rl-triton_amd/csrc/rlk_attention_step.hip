// rlk_attention_step.hip -- one step of linear attention for every environment (include/rl_triton_policy.h):
//   S' = lambda (1 - done) S + k v^T,  out = scale S'^T q.
// The state is read and written once and is nearly all there is to move: a workgroup per (environment, head),
// each thread a quad of columns, the rows dealt out over the workgroup.  [512,16,128,128]: 191 us, 5.6 TB/s (a large copy 5.2);
// [8,4,64,64]: 3.9 us, of which a launch is the most.
#include "rlk_attention.hpp"

namespace rlk {
namespace {

constexpr int kNT = 256;

// LANES lanes cover a row of the state in quads.  NT: non-temporal accesses to it.
template <class E, int LANES, bool VEC, bool NT>
__global__ __launch_bounds__(kNT) void step_kernel(const Walk<E> w, int heads, int64_t first, const float* __restrict__ decay,
                                                   const float* __restrict__ dones) {
  constexpr int ROWS = kNT / LANES;
  __shared__ float qs[128], ks[128];
  __shared__ float4 part[ROWS][LANES];
  const int64_t eh = first + blockIdx.x, env = eh / heads;
  const int head = (int)(eh - env * heads), tid = threadIdx.x;
  const int lane = tid % LANES, row0 = tid / LANES, j = lane * 4;
  if (tid < w.da) {
    qs[tid] = load_one(w.a.data + env * w.a.env_stride + head * w.a.head_stride + tid);
    ks[tid] = load_one(w.b.data + env * w.b.env_stride + head * w.b.head_stride + tid);
  }
  const float lambda = decay[head];
  const bool cut = lambda == 0.f || (dones != nullptr && dones[env] != 0.f);
  const E* gv = w.c.data + env * w.c.env_stride + head * w.c.head_stride;
  float v[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) v[x] = j + x < w.dc ? load_one(gv + j + x) : 0.f;
  __syncthreads();
  const float* src = w.state + eh * (int64_t)(w.da * w.dc);
  float* dst = w.state_out + eh * (int64_t)(w.da * w.dc);
  float4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = row0; i < w.da; i += ROWS) {
    float4 x{0.f, 0.f, 0.f, 0.f};
    if (j < w.dc) {
      const int at = i * w.dc + j;
      if (!cut) {  // (what a cut state held has no part, NaN included, nor what a decay of 0 leaves)
        if constexpr (VEC) {
          x = load_quad<NT>(src + at);
        } else {
          x.x = src[at];
          if (j + 1 < w.dc) x.y = src[at + 1];
          if (j + 2 < w.dc) x.z = src[at + 2];
          if (j + 3 < w.dc) x.w = src[at + 3];
        }
      }
      const float k = ks[i], q = qs[i];
      x.x = fmaf(lambda, x.x, k * v[0]), x.y = fmaf(lambda, x.y, k * v[1]);
      x.z = fmaf(lambda, x.z, k * v[2]), x.w = fmaf(lambda, x.w, k * v[3]);
      if constexpr (VEC) {
        store_quad<NT>(dst + at, x);
      } else {
        dst[at] = x.x;
        if (j + 1 < w.dc) dst[at + 1] = x.y;
        if (j + 2 < w.dc) dst[at + 2] = x.z;
        if (j + 3 < w.dc) dst[at + 3] = x.w;
      }
      acc.x = fmaf(q, x.x, acc.x), acc.y = fmaf(q, x.y, acc.y), acc.z = fmaf(q, x.z, acc.z), acc.w = fmaf(q, x.w, acc.w);
    }
  }
  part[row0][lane] = acc;
  __syncthreads();
  if (tid < w.dc) {
    float y = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) y += reinterpret_cast<const float*>(&part[r][0])[tid];
    w.y.data[env * w.y.env_stride + head * w.y.head_stride + tid] = from_f32<E>(y * w.scale);
  }
}

template <class E>
int step_impl(const rlk_attention& c, hipStream_t s) {
  Walk<E> w = {};
  w.a = sequence<const E>(c.q), w.b = sequence<const E>(c.k), w.c = sequence<const E>(c.v), w.y = sequence<E>(c.out);
  w.da = (int)c.dim_k, w.dc = (int)c.dim_v, w.state = c.state, w.state_out = c.state_out, w.scale = c.scale;
  const bool vec = c.dim_v % 4 == 0 && ((reinterpret_cast<uintptr_t>(c.state) | reinterpret_cast<uintptr_t>(c.state_out)) & 15u) == 0;
  const int heads = (int)c.heads;
  // A state that the 256 MB of last-level cache cannot keep for the next step goes past the caches (512 MB: 192 us, 206 through
  // them; 256 MB: 99 and 99 to 107); a smaller one is found there again (64 MB: 23.5 us, 26 past them).
  const bool large = c.num_envs * c.heads * c.dim_k * c.dim_v * (int64_t)sizeof(float) >= int64_t{1} << 28;
  const int64_t pairs = c.num_envs * c.heads, most = int64_t{1} << 23;  // (of one launch: 2^31 work-items)
  for (int64_t first = 0; first < pairs; first += most) {
    const dim3 grid((unsigned)(pairs - first < most ? pairs - first : most)), block(kNT);
    auto launch = [&](auto lanes, auto v, auto nt) {
      step_kernel<E, decltype(lanes)::value, decltype(v)::value, decltype(nt)::value><<<grid, block, 0, s>>>(w, heads, first, c.decay, c.dones);
    };
    auto by_size = [&](auto v, auto nt) {
      if (c.dim_v <= 64) launch(std::integral_constant<int, 16>{}, v, nt);
      else launch(std::integral_constant<int, 32>{}, v, nt);
    };
    if (!vec) by_size(std::false_type{}, std::false_type{});
    else if (large) by_size(std::true_type{}, std::true_type{});
    else by_size(std::true_type{}, std::false_type{});
    if (hipGetLastError() != hipSuccess) return RLK_ERR_LAUNCH;
  }
  return RLK_OK;
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" int rlk_linear_attention_step(const rlk_attention* call, void* stream) {
  if (!call || !valid_attention(*call)) return RLK_ERR_INVALID_ARGUMENT;
  if (call->num_envs == 0 || call->heads == 0) return RLK_OK;
  if (!call->state || !call->state_out || call->heads > 0x7fffffff) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return call->bf16 ? step_impl<bf16>(*call, s) : step_impl<float>(*call, s);
}
