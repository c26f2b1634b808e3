// rlk_delta.hip -- the gated delta rule's C entries (include/rl_triton_policy.h): checks, memory and launches of whole sequences, and the
// kernel of one step.
#include "rlk_delta.hpp"

namespace rlk {
namespace delta {
namespace {

// How many environments go into one set of launches: their records (11.5 KB a chunk of a pair, environment and head) or a backward pass's gradients
// of states and z (up to 96 KB) are scratch memory.  As many as 1 GB holds, but at least 512 pairs, so that every CU has some to walk, and at
// least one environment: a backward pass of 512 pairs over 16384 steps asks for 12 GB at 128 + 128 dims, one environment of 16 heads and 2^20 steps for
// 24.  A launch has at most 2^31 work-items.
constexpr size_t kScratch = size_t{1} << 30;
constexpr int64_t kMostChunks = int64_t{1} << 22;
inline int64_t envs_at_once(int64_t envs, int64_t heads, int64_t chunks, size_t chunk_bytes) {
  int64_t n = (int64_t)(kScratch / (chunk_bytes * (size_t)(heads * chunks)));
  const int64_t filling = (512 + heads - 1) / heads, most = kMostChunks / (heads * chunks);
  if (n < filling) n = filling;
  if (n > most) n = most;
  return n < envs ? (n > 1 ? n : 1) : envs;
}
inline int64_t chunks_of(int64_t T) { return (T + C - 1) / C; }
inline size_t state_bytes(int64_t dk, int64_t dv) { return sizeof(float) * pad16((int)dk) * pad16((int)dv); }
inline size_t columns_bytes(int64_t dv) { return sizeof(float) * C * pad16((int)dv); }

bool valid(const rlk_delta_rule& c, bool steps) {
  if (c.num_envs < 0 || c.heads < 0 || c.dim_k < 1 || c.dim_k > 128 || c.dim_v < 1 || c.dim_v > 128) return false;
  if (!std::isfinite(c.scale)) return false;
  if (c.num_envs == 0 || c.heads == 0) return true;
  const uintptr_t low = c.bf16 ? 1u : 3u;
  for (const rlk_sequence* x : {&c.q, &c.k, &c.v, &c.out})
    if (steps && (!x->data || (reinterpret_cast<uintptr_t>(x->data) & low) != 0)) return false;
  return !steps || c.betas != nullptr;
}
// Whether heads and chunks are few enough for the launches of one environment.
bool fits(const rlk_delta_rule& c) { return c.seq_len <= (int64_t{1} << 30) && c.heads <= kMostChunks && c.heads * chunks_of(c.seq_len) <= kMostChunks; }
bool scratch_fits(const void* p, size_t have, size_t need) { return need == 0 || (have >= need && p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15u) == 0); }

template <class E>
Rule<E> rule(const rlk_delta_rule& c) {
  Rule<E> r = {};
  r.q = seq<const E>(c.q), r.k = seq<const E>(c.k), r.v = seq<const E>(c.v), r.y = seq<E>(c.out);
  r.seq_len = c.seq_len, r.chunks = chunks_of(c.seq_len), r.heads = (int)c.heads, r.dk = (int)c.dim_k, r.dv = (int)c.dim_v;
  r.gates = c.log_decays, r.betas = c.betas, r.dones = c.dones, r.state = c.state, r.state_out = c.state_out, r.scale = c.scale;
  return r;
}

// The state after no steps: the one before them.
__global__ __launch_bounds__(256) void same_state_kernel(const float* from, float* to, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from != nullptr ? from[i] : 0.f;
}
int same_state(const rlk_delta_rule& c, const float* from, float* to, hipStream_t s) {
  if (to == nullptr) return RLK_OK;
  const int64_t n = c.num_envs * c.heads * c.dim_k * c.dim_v, units = (n + 255) / 256;
  same_state_kernel<<<dim3((unsigned)(units < 4096 ? units : 4096)), dim3(256), 0, s>>>(from, to, n);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

// What a forward pass leaves for the one back: records, states, corrections.
struct Saved {
  char* base;
  int64_t per_env;  // chunks of an environment
  size_t count, dk, dv;
  Saved(void* p, const rlk_delta_rule& c)
      : base(static_cast<char*>(p)), per_env(c.heads * chunks_of(c.seq_len)), count((size_t)(c.num_envs * per_env)), dk((size_t)c.dim_k), dv((size_t)c.dim_v) {}
  size_t bytes() const { return count * (sizeof(Record) + state_bytes(dk, dv) + columns_bytes(dv)); }
  template <class E>
  void at(Rule<E>& r) const {
    const size_t first = (size_t)(r.first_env * per_env);
    r.records = reinterpret_cast<Record*>(base) + first;
    r.states = reinterpret_cast<float*>(base + count * sizeof(Record) + first * state_bytes(dk, dv));
    r.w = reinterpret_cast<float*>(base + count * (sizeof(Record) + state_bytes(dk, dv)) + first * columns_bytes(dv));
  }
};

template <class E>
int forward(const rlk_delta_rule& c, void* saved, hipStream_t s) {
  Rule<E> r = rule<E>(c);
  const int64_t most = envs_at_once(c.num_envs, c.heads, r.chunks, sizeof(Record));
  for (r.first_env = 0; r.first_env < c.num_envs; r.first_env += most) {
    const int64_t envs = c.num_envs - r.first_env < most ? c.num_envs - r.first_env : most;
    const int64_t pairs = envs * c.heads;
    r.records = static_cast<Record*>(c.workspace);
    float* p = reinterpret_cast<float*>(r.records + (saved != nullptr ? 0 : pairs * r.chunks));
    const Segments plan = plan_segments(pairs, r.chunks);
    r.segs = plan.segs, r.seg_chunks = plan.chunks;
    if (plan.segs > 1) {
      r.wild = reinterpret_cast<int*>(p);
      r.phi = p + (pairs + 3) / 4 * 4;
      r.seg_states = r.phi + (size_t)(pairs * plan.segs) * pad16(r.dk) * pad16(r.dk);
    } else {
      r.wild = nullptr;
    }
    if (saved != nullptr) Saved(saved, c).at(r);
    int st = launch_records(r, envs, s);
    if (st == RLK_OK) st = launch_forward(r, envs, s);
    if (st != RLK_OK) return st;
  }
  return RLK_OK;
}

size_t backward_chunk_bytes(int64_t dk, int64_t dv) { return state_bytes(dk, dv) + columns_bytes(dv); }

template <class E>
int backward(const rlk_delta_rule& c, const rlk_delta_rule_gradients& g, const void* saved, hipStream_t s) {
  Rule<E> r = rule<E>(c);
  r.from_zero = c.state == nullptr;
  r.y = {}, r.state = g.state_out, r.state_out = g.state;
  r.gy = seq<const E>(g.out), r.gq = seq<E>(g.q), r.gk = seq<E>(g.k), r.gv = seq<E>(g.v), r.gg = g.log_decays, r.gb = g.betas;
  const int64_t most = envs_at_once(c.num_envs, c.heads, r.chunks, backward_chunk_bytes(c.dim_k, c.dim_v));
  const bool more = r.gq.data || r.gk.data || r.gg || r.gb;
  for (r.first_env = 0; r.first_env < c.num_envs; r.first_env += most) {
    const int64_t envs = c.num_envs - r.first_env < most ? c.num_envs - r.first_env : most;
    Saved(const_cast<void*>(saved), c).at(r);
    r.z = static_cast<float*>(c.workspace);
    r.dstates = more ? r.z + (size_t)(envs * c.heads * r.chunks) * columns_bytes(c.dim_v) / sizeof(float) : nullptr;
    int st = launch_backward(r, envs, s);
    if (st == RLK_OK && more) st = launch_gradients(r, envs, s);
    if (st != RLK_OK) return st;
  }
  return RLK_OK;
}

// One step: a workgroup per (environment, head) holds the state in registers, a thread a quad of columns of every ROWS-th row; what keys and
// queries read from it is added up over the rows, then the state goes back with the correction.  The state is read and written once and
// is nearly all there is to move: [512] of 16 heads of 128 + 128 198 us, 5.4 TB/s; [8] of 4 heads of 64 + 64 5.5 us, a launch.
template <class E, int LANES, int PER, bool VEC, bool NT>
__global__ __launch_bounds__(256) void step_kernel(const Rule<E> r, int64_t first) {
  constexpr int ROWS = 256 / LANES;
  __shared__ float qs[128], ks[128];
  __shared__ float4 part[2][ROWS][LANES];
  __shared__ float dots[4];
  const int64_t eh = first + blockIdx.x, env = eh / r.heads;
  const int head = (int)(eh - env * r.heads), tid = threadIdx.x, lane = tid % LANES, row0 = tid / LANES, j = lane * 4;
  const float g = r.gates != nullptr ? r.gates[eh] : 0.f, b = r.betas[eh];
  const bool cut = g <= kNoDecay || (r.dones != nullptr && r.dones[env] != 0.f);
  const float a = cut ? 0.f : expf(g);
  const float* src = r.state + eh * r.dk * r.dv;
  float* dst = r.state_out + eh * r.dk * r.dv;
  float4 S[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = row0 + ROWS * i;
    S[i] = float4{0.f, 0.f, 0.f, 0.f};
    if (d < r.dk && j < r.dv && !cut) {  // (what a cut state held has no part, NaN included)
      const float* p = src + d * r.dv + j;
      if constexpr (VEC) {
        S[i] = load_quad<NT>(p);
      } else {
        S[i].x = p[0];
        if (j + 1 < r.dv) S[i].y = p[1];
        if (j + 2 < r.dv) S[i].z = p[2];
        if (j + 3 < r.dv) S[i].w = p[3];
      }
    }
  }
  if (tid < 128) {
    const float q = tid < r.dk ? load_one(r.q.data + env * r.q.env + head * r.q.head + tid) : 0.f;
    const float k = tid < r.dk ? load_one(r.k.data + env * r.k.env + head * r.k.head + tid) : 0.f;
    qs[tid] = q, ks[tid] = k;
    float x = tid < r.dk ? q * k : 0.f;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    if ((tid & 63) == 0) dots[tid >> 6] = x;
  }
  const E* gv = r.v.data + env * r.v.env + head * r.v.head;
  float v[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) v[x] = j + x < r.dv ? load_one(gv + j + x) : 0.f;
  __syncthreads();
  float4 fk{0.f, 0.f, 0.f, 0.f}, fq = fk;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = row0 + ROWS * i;
    if (d < r.dk) {
      S[i].x *= a, S[i].y *= a, S[i].z *= a, S[i].w *= a;
      const float k = ks[d], q = qs[d];
      fk.x = fmaf(k, S[i].x, fk.x), fk.y = fmaf(k, S[i].y, fk.y), fk.z = fmaf(k, S[i].z, fk.z), fk.w = fmaf(k, S[i].w, fk.w);
      fq.x = fmaf(q, S[i].x, fq.x), fq.y = fmaf(q, S[i].y, fq.y), fq.z = fmaf(q, S[i].z, fq.z), fq.w = fmaf(q, S[i].w, fq.w);
    }
  }
  part[0][row0][lane] = fk, part[1][row0][lane] = fq;
  __syncthreads();
  float4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const float4 x = part[0][i][lane];
    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
  }
  const float u[4] = {b * (v[0] - sum.x), b * (v[1] - sum.y), b * (v[2] - sum.z), b * (v[3] - sum.w)};
  if (j < r.dv) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int d = row0 + ROWS * i;
      if (d < r.dk) {
        const float k = ks[d];
        const float4 x{fmaf(k, u[0], S[i].x), fmaf(k, u[1], S[i].y), fmaf(k, u[2], S[i].z), fmaf(k, u[3], S[i].w)};
        float* p = dst + d * r.dv + j;
        if constexpr (VEC) {
          store_quad<NT>(p, x);
        } else {
          p[0] = x.x;
          if (j + 1 < r.dv) p[1] = x.y;
          if (j + 2 < r.dv) p[2] = x.z;
          if (j + 3 < r.dv) p[3] = x.w;
        }
      }
    }
    if (row0 == 0) {
      // q . (S + k u^T) = q . S + (q . k) u
      float4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float4 x = part[1][i][lane];
        y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
      }
      const float qk = dots[0] + dots[1];
      E* p = r.y.data + env * r.y.env + head * r.y.head + j;
      const float out[4] = {fmaf(qk, u[0], y.x) * r.scale, fmaf(qk, u[1], y.y) * r.scale, fmaf(qk, u[2], y.z) * r.scale, fmaf(qk, u[3], y.w) * r.scale};
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (j + x < r.dv) p[x] = from_f32<E>(out[x]);
    }
  }
}

template <class E>
int step(const rlk_delta_rule& c, hipStream_t s) {
  const Rule<E> r = rule<E>(c);
  const bool vec = c.dim_v % 4 == 0 && ((reinterpret_cast<uintptr_t>(c.state) | reinterpret_cast<uintptr_t>(c.state_out)) & 15u) == 0;
  // A state that the last-level cache cannot keep for the next step goes past the caches (as in rlk_attention_step.hip).
  const bool large = c.num_envs * c.heads * c.dim_k * c.dim_v * (int64_t)sizeof(float) >= int64_t{1} << 28;
  const int64_t pairs = c.num_envs * c.heads, most = int64_t{1} << 23;
  for (int64_t first = 0; first < pairs; first += most) {
    const dim3 grid((unsigned)(pairs - first < most ? pairs - first : most)), block(256);
    auto launch = [&](auto lanes, auto per, auto v, auto nt) {
      step_kernel<E, decltype(lanes)::value, decltype(per)::value, decltype(v)::value, decltype(nt)::value><<<grid, block, 0, s>>>(r, first);
    };
    auto by_size = [&](auto v, auto nt) {
      typedef std::integral_constant<int, 16> Sixteen;
      typedef std::integral_constant<int, 32> ThirtyTwo;
      if (c.dim_v <= 64) c.dim_k <= 64 ? launch(Sixteen{}, std::integral_constant<int, 4>{}, v, nt) : launch(Sixteen{}, std::integral_constant<int, 8>{}, v, nt);
      else c.dim_k <= 64 ? launch(ThirtyTwo{}, std::integral_constant<int, 8>{}, v, nt) : launch(ThirtyTwo{}, Sixteen{}, v, nt);
    };
    if (!vec) by_size(std::false_type{}, std::false_type{});
    else if (large) by_size(std::true_type{}, std::true_type{});
    else by_size(std::true_type{}, std::false_type{});
    if (hipGetLastError() != hipSuccess) return RLK_ERR_LAUNCH;
  }
  return RLK_OK;
}

}  // namespace
}  // namespace delta
}  // namespace rlk

using namespace rlk;
using namespace rlk::delta;

extern "C" {

size_t rlk_delta_rule_workspace_bytes(int64_t num_envs, int64_t seq_len, int64_t heads, int64_t dim_k, int64_t dim_v, int pass) {
  const bool backward = pass == RLK_DELTA_BACKWARD;
  if (num_envs <= 0 || seq_len <= 0 || heads <= 0 || dim_k <= 0 || dim_v <= 0 || dim_k > 128 || dim_v > 128 || heads > kMostChunks ||
      seq_len > (int64_t{1} << 30) || heads * chunks_of(seq_len) > kMostChunks)
    return 0;
  const int64_t chunks = chunks_of(seq_len);
  const size_t each = backward ? backward_chunk_bytes(dim_k, dim_v) : sizeof(Record);
  const int64_t envs = envs_at_once(num_envs, heads, chunks, each);
  size_t bytes = pass == RLK_DELTA_FORWARD_SAVED ? 0 : (size_t)(envs * heads * chunks) * each;
  if (!backward) {  // (the last set of environments, the smaller one, may be the one that is cut)
    size_t floats = segment_floats(envs * heads, plan_segments(envs * heads, chunks), (int)dim_k, (int)dim_v);
    if (const int64_t left = num_envs % envs) {
      const size_t last = segment_floats(left * heads, plan_segments(left * heads, chunks), (int)dim_k, (int)dim_v);
      if (last > floats) floats = last;
    }
    bytes += floats * sizeof(float);
  }
  return bytes;
}

size_t rlk_delta_rule_saved_bytes(int64_t num_envs, int64_t seq_len, int64_t heads, int64_t dim_k, int64_t dim_v) {
  if (num_envs <= 0 || seq_len <= 0 || heads <= 0 || dim_k <= 0 || dim_v <= 0 || dim_k > 128 || dim_v > 128) return 0;
  return (size_t)(num_envs * heads * chunks_of(seq_len)) * (sizeof(Record) + state_bytes(dim_k, dim_v) + columns_bytes(dim_v));
}

int rlk_gated_delta_rule(const rlk_delta_rule* call, void* saved, size_t saved_bytes, void* stream) {
  if (!call || call->seq_len < 0 || !valid(*call, call->seq_len != 0)) return RLK_ERR_INVALID_ARGUMENT;
  if (call->num_envs == 0 || call->heads == 0) return RLK_OK;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (call->seq_len == 0) return same_state(*call, call->state, call->state_out, s);
  if (!fits(*call)) return RLK_ERR_INVALID_ARGUMENT;
  if ((saved != nullptr && !scratch_fits(saved, saved_bytes, Saved(saved, *call).bytes())) ||
      !scratch_fits(call->workspace, call->workspace_bytes,
                    rlk_delta_rule_workspace_bytes(call->num_envs, call->seq_len, call->heads, call->dim_k, call->dim_v,
                                                   saved != nullptr ? RLK_DELTA_FORWARD_SAVED : RLK_DELTA_FORWARD)))
    return RLK_ERR_WORKSPACE;
  return call->bf16 ? forward<bf16>(*call, saved, s) : forward<float>(*call, saved, s);
}

int rlk_gated_delta_rule_backward(const rlk_delta_rule* call, const rlk_delta_rule_gradients* grads, const void* saved, size_t saved_bytes,
                                  void* stream) {
  if (!call || !grads || call->seq_len < 0) return RLK_ERR_INVALID_ARGUMENT;
  rlk_delta_rule c = *call;
  c.out = grads->out;  // (the outputs themselves are not read)
  if (!valid(c, c.seq_len != 0)) return RLK_ERR_INVALID_ARGUMENT;
  const uintptr_t low = c.bf16 ? 1u : 3u;
  for (const rlk_sequence* x : {&grads->q, &grads->k, &grads->v})
    if ((reinterpret_cast<uintptr_t>(x->data) & low) != 0) return RLK_ERR_INVALID_ARGUMENT;
  if (c.num_envs == 0 || c.heads == 0) return RLK_OK;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (c.seq_len == 0) return same_state(c, grads->state_out, grads->state, s);
  if (!fits(c)) return RLK_ERR_INVALID_ARGUMENT;
  if (!scratch_fits(saved, saved_bytes, Saved(nullptr, c).bytes()) ||
      !scratch_fits(c.workspace, c.workspace_bytes, rlk_delta_rule_workspace_bytes(c.num_envs, c.seq_len, c.heads, c.dim_k, c.dim_v, RLK_DELTA_BACKWARD)))
    return RLK_ERR_WORKSPACE;
  return c.bf16 ? backward<bf16>(c, *grads, saved, s) : backward<float>(c, *grads, saved, s);
}

int rlk_gated_delta_rule_step(const rlk_delta_rule* call, void* stream) {
  if (!call || !valid(*call, true)) return RLK_ERR_INVALID_ARGUMENT;
  if (call->num_envs == 0 || call->heads == 0) return RLK_OK;
  if (!call->state || !call->state_out || call->heads > 0x7fffffff) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return call->bf16 ? step<bf16>(*call, s) : step<float>(*call, s);
}

}  // extern "C"
