// rlk_head_norms.hip -- queries and keys normed head by head and turned by their positions, in one pass, and back
// (include/rl_triton_policy.h).
//
//   y = x r w, r = 1 / sqrt(mean(x^2) + eps), and pairs (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin), angle = position * base^(-2 i / rotary).
// Back, with g turned back by the same angle: dw = sum over rows of g x r, dx = r (w g - x r^2 mean(x w g)).
//
// Bound by memory: a row is read once and written once.  A group of lanes holds a row, each lane 4 pairs (or 1, where sizes or addresses
// do not allow vectors): elements that are not turned are paired as they come.  A group takes a few heads of a step one after the other, all
// loads first, with the angles formed once.  Angles: position times frequency in turns, in float64, and what is left of the nearest quarter
// turn in float32, so that a position of a million is as exact as the first one.
//
// GPU time, bf16: [1,16384,16+4,128] 42 us (4.0 TB/s; 52 where nothing is in the caches yet), [64,1024,8+8,64] forward 75 us (3.6 TB/s), back 118 us (3.4 TB/s) and 4 for the weights; what
// keeps it from the copy's 4.8 are the angles, some third of the instructions.  One group for queries and keys alike, to share them: 42 -> 59
// and 77 -> 92 us.
#include "rlk_launch.hpp"
#include "rlk_policy.hpp"

namespace rlk {
namespace {

constexpr int kMostDim = 256;
// Heads of a step that a group takes: 4, forward, share their angles; back, where a row is two arrays', 2 of them leave room for more wavefronts
// ([64,1024,8+8,64] bf16: 144 us, 190 with 4).
template <bool BACK>
constexpr int kHeads = BACK ? 2 : 4;
// Back: as many workgroups along the steps, for all blocks of heads together, as are resident at once, 5 a CU: each goes on over the steps until
// all are done, and leaves its sums of the weights' gradients ([64,1024,8+8,64] bf16: 118 us; 130 with 4 a CU, 137 with 8, whose last ones
// run by themselves).
constexpr int kResident = 5;
int64_t back_blocks(int64_t blocks) { return std::max<int64_t>(1, kResident * device_cus() / std::max<int64_t>(1, blocks)); }

struct Frequencies {
  double turns[kMostDim / 2];  // of a position, by pair
};

template <class E>
struct Side {
  const E* x;
  E* y;
  const E* g;  // backward
  int64_t env, step, head, yenv, ystep, yhead, genv, gstep, ghead;
  const float* weight;
  int heads, blocks;  // blocks of heads that a group takes together
};

template <class E>
struct Norms {
  Side<E> side[2];  // queries, keys
  int64_t tokens, steps;
  int64_t stride_envs, stride_steps;  // from a group's token to its next one
  int dim, rotary, blocks;  // blocks: of heads, queries' and keys'
  const int64_t* positions;
  float eps, inv_dim;
  float* partial;  // backward: [back_blocks() at most][blocks of queries + keys][dim]
};

// N consecutive elements of E.
template <class E, int N>
struct Elements {
  float x[N];
  __device__ void load(const E* p) {
    if constexpr (N == 4) {
      const float4 f = load_quad<false>(p);
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
      x[0] = load_one(p);
    }
  }
  __device__ void store(E* p) const {
    if constexpr (N == 4) store_quad<false>(p, float4{x[0], x[1], x[2], x[3]});
    else *p = from_f32<E>(x[0]);
  }
};

// Where a lane's unit of N pairs lies: N firsts and N seconds.  HALVES: pairs are (i, i + rotary / 2); else neighbours, which for N = 4 are
// two quads of elements.
template <int N, bool HALVES>
struct Unit {
  int a, b;      // the first and second run of N elements
  bool there, second;  // second: the second run is there too (the last of an odd number of elements that are not turned has none)
  int pair;      // the first pair's number, or -1: not turned
  __device__ Unit(int slot, int dim, int rotary) {
    const int half = rotary / 2, s = slot * N;
    pair = s < half ? s : -1;
    if (s < half && HALVES) {
      a = s, b = s + half;
    } else {  // neighbours: turned ones, or those behind
      const int e = s < half ? 2 * s : rotary + 2 * (s - half);
      a = e, b = e + N;
    }
    there = a < dim, second = b < dim;
  }
};

template <int N, bool HALVES>
struct Turn {
  float c[N], s[N];
  bool on;
  __device__ void set(const Unit<N, HALVES>& u, const Frequencies& f, const int64_t* position) {
    on = position != nullptr && u.there && u.pair >= 0;
    const double where = on ? (double)*position : 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = 1.f, s[i] = 0.f;
      if (!on) continue;
      // in turns, less whole ones, and of these less quarters: what is left is within an eighth
      const double t = __builtin_amdgcn_fract(where * f.turns[u.pair + i]);
      const double quarters = rint(4.0 * t);
      const float x = (float)((t - 0.25 * quarters) * 6.283185307179586476925), y = x * x;
      // (series up to pi / 4: the first terms left out are below 2^-28)
      float sn = fmaf(y, 1.f / 362880.f, -1.f / 5040.f), cs = fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
      sn = fmaf(sn, y, 1.f / 120.f), cs = fmaf(cs, y, -1.f / 720.f);
      sn = fmaf(sn, y, -1.f / 6.f), cs = fmaf(cs, y, 1.f / 24.f);
      sn = fmaf(sn * y, x, x), cs = fmaf(cs, y, -0.5f);
      cs = fmaf(cs, y, 1.f);
      const int n = (int)quarters;
      const float a = n & 1 ? sn : cs, b = n & 1 ? cs : sn;
      c[i] = (n + 1) & 2 ? -a : a;
      s[i] = n & 2 ? -b : b;
    }
  }
  // pairs of a unit: element i of both runs, or neighbours across the two runs
  __device__ void apply(float (&x)[N], float (&y)[N], bool back) const {
    if (!on) return;
    float v[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = x[i], v[N + i] = y[i];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = HALVES ? i : 2 * i, q = HALVES ? N + i : 2 * i + 1;
      const float a = v[p], b = v[q], sn = back ? -s[i] : s[i];
      v[p] = fmaf(a, c[i], -b * sn), v[q] = fmaf(b, c[i], a * sn);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = v[i], y[i] = v[N + i];
  }
};

template <int G>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int d = 1; d < G; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// G lanes a row, UNITS units of N pairs a lane.
template <class E, int N, int G, int UNITS, bool HALVES, bool BACK>
__global__ __launch_bounds__(256, BACK ? kResident : 4) void norms_kernel(const Norms<E> n, const Frequencies f) {
  const int lane = threadIdx.x & (G - 1), group = threadIdx.x / G;
  constexpr int GROUPS = 256 / G;
  // (the blocks of heads of the same steps run together, as a step's heads lie: [1,16384,16+4,128] 52 us, 55 with all steps of a block first)
  const uint32_t slot = blockIdx.x / (uint32_t)n.blocks, slots = gridDim.x / (uint32_t)n.blocks;
  const int block = (int)(blockIdx.x - slot * (uint32_t)n.blocks);
  const bool keys = block >= n.side[0].blocks;
  const Side<E>& d = n.side[keys];
  const int head0 = (block - (keys ? n.side[0].blocks : 0)) * kHeads<BACK>, heads = d.heads - head0 < kHeads<BACK> ? d.heads - head0 : kHeads<BACK>;
  Elements<E, N> wa[UNITS], wb[UNITS], ga[UNITS], gb[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const Unit<N, HALVES> at(lane + G * u, n.dim, n.rotary);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      wa[u].x[i] = d.weight != nullptr && at.there ? d.weight[at.a + i] : 1.f;
      wb[u].x[i] = d.weight != nullptr && at.second ? d.weight[at.b + i] : 1.f;
      ga[u].x[i] = gb[u].x[i] = 0.f;
    }
  }
  int64_t token = (int64_t)slot * GROUPS + group;
  // (a division in 64 bits is as much work as a row)
  int64_t env = n.tokens >> 32 == 0 ? (int64_t)((uint32_t)token / (uint32_t)n.steps) : token / n.steps, step = token - env * n.steps;
  for (; token < n.tokens; token += (int64_t)slots * GROUPS) {
    const E* px = d.x + env * d.env + step * d.step + head0 * d.head;
    Elements<E, N> xa[kHeads<BACK>][UNITS], xb[kHeads<BACK>][UNITS], ya[BACK ? kHeads<BACK> : 1][UNITS], yb[BACK ? kHeads<BACK> : 1][UNITS];
#pragma unroll
    for (int h = 0; h < kHeads<BACK>; ++h) {
      if (h >= heads) continue;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const Unit<N, HALVES> at(lane + G * u, n.dim, n.rotary);
#pragma unroll
        for (int i = 0; i < N; ++i) xa[h][u].x[i] = xb[h][u].x[i] = 0.f;
        if (at.there) xa[h][u].load(px + h * d.head + at.a);
        if (at.second) xb[h][u].load(px + h * d.head + at.b);
        if constexpr (BACK) {
          const E* pg = d.g + env * d.genv + step * d.gstep + (head0 + h) * d.ghead;
#pragma unroll
          for (int i = 0; i < N; ++i) ya[h][u].x[i] = yb[h][u].x[i] = 0.f;
          if (at.there) ya[h][u].load(pg + at.a);
          if (at.second) yb[h][u].load(pg + at.b);
        }
      }
    }
    Turn<N, HALVES> turn[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
      turn[u].set(Unit<N, HALVES>(lane + G * u, n.dim, n.rotary), f, n.positions != nullptr ? n.positions + token : nullptr);
    E* py = d.y != nullptr ? d.y + env * d.yenv + step * d.ystep + head0 * d.yhead : nullptr;
#pragma unroll
    for (int h = 0; h < kHeads<BACK>; ++h) {
      if (h >= heads) continue;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) sum = fmaf(xa[h][u].x[i], xa[h][u].x[i], fmaf(xb[h][u].x[i], xb[h][u].x[i], sum));
      const float square = fmaf(group_sum<G>(sum), n.inv_dim, n.eps);
      float r = __builtin_amdgcn_rsqf(square);
      r = fmaf(r * fmaf(-square * r, r, 1.f), 0.5f, r);  // (one step to the last bit)
      if (square < 1e-30f || square > 1e30f) {
        // Squares near or past the ends of float32, in all lanes of the group alike: of elements and a root of eps taken times a power of two.
        const float times = square < 1.f ? 0x1p80f : 0x1p-80f;
        sum = 0.f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float a = xa[h][u].x[i] * times, b = xb[h][u].x[i] * times;
            sum = fmaf(a, a, fmaf(b, b, sum));
          }
        r = times / sqrtf(fmaf(group_sum<G>(sum), n.inv_dim, n.eps * times * times));
      }
      if constexpr (!BACK) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const Unit<N, HALVES> at(lane + G * u, n.dim, n.rotary);
          Elements<E, N> a, b;
#pragma unroll
          for (int i = 0; i < N; ++i) a.x[i] = xa[h][u].x[i] * r * wa[u].x[i], b.x[i] = xb[h][u].x[i] * r * wb[u].x[i];
          turn[u].apply(a.x, b.x, false);
          if (at.there) a.store(py + h * d.yhead + at.a);
          if (at.second) b.store(py + h * d.yhead + at.b);
        }
      } else {
        float dot = 0.f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          turn[u].apply(ya[h][u].x, yb[h][u].x, true);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float a = xa[h][u].x[i] * r, b = xb[h][u].x[i] * r;  // unit rows
            xa[h][u].x[i] = a, xb[h][u].x[i] = b;
            ga[u].x[i] = fmaf(ya[h][u].x[i], a, ga[u].x[i]), gb[u].x[i] = fmaf(yb[h][u].x[i], b, gb[u].x[i]);
            ya[h][u].x[i] *= wa[u].x[i], yb[h][u].x[i] *= wb[u].x[i];
            dot = fmaf(ya[h][u].x[i], a, fmaf(yb[h][u].x[i], b, dot));
          }
        }
        const float mean = group_sum<G>(dot) * n.inv_dim;
        if (py != nullptr)
#pragma unroll
          for (int u = 0; u < UNITS; ++u) {
            const Unit<N, HALVES> at(lane + G * u, n.dim, n.rotary);
            Elements<E, N> a, b;
#pragma unroll
            for (int i = 0; i < N; ++i)
              a.x[i] = r * fmaf(-xa[h][u].x[i], mean, ya[h][u].x[i]), b.x[i] = r * fmaf(-xb[h][u].x[i], mean, yb[h][u].x[i]);
            if (at.there) a.store(py + h * d.yhead + at.a);
            if (at.second) b.store(py + h * d.yhead + at.b);
          }
      }
    }
    env += n.stride_envs, step += n.stride_steps;
    if (step >= n.steps) step -= n.steps, ++env;
  }
  if constexpr (BACK) {
    if (n.partial == nullptr) return;
    // the workgroup's sums: a wavefront's groups, then the wavefronts
    __shared__ float sums[4][kMostDim];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const Unit<N, HALVES> at(lane + G * u, n.dim, n.rotary);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float a = ga[u].x[i], b = gb[u].x[i];
#pragma unroll
        for (int d = G; d < 64; d <<= 1) a += __shfl_xor(a, d), b += __shfl_xor(b, d);
        if ((threadIdx.x & 63) < G && at.there) sums[threadIdx.x >> 6][at.a + i] = a;
        if ((threadIdx.x & 63) < G && at.second) sums[threadIdx.x >> 6][at.b + i] = b;
      }
    }
    __syncthreads();
    if ((int)threadIdx.x < n.dim)
      n.partial[(int64_t)blockIdx.x * n.dim + threadIdx.x] =
          (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
  }
}

// The weights' gradients from the workgroups' sums: a workgroup per 4 elements and side, in float64 and a fixed order.  0 where there are no rows.
__global__ __launch_bounds__(256) void weights_kernel(const float* partial, int blocks, int q_blocks, int k_blocks, int dim, float* gq, float* gk) {
  float* out = blockIdx.y ? gk : gq;
  if (out == nullptr) return;
  const int e = blockIdx.x * 4 + threadIdx.x % 4, first = blockIdx.y ? q_blocks : 0, count = blockIdx.y ? k_blocks : q_blocks, all = q_blocks + k_blocks;
  __shared__ double s[256];
  double x = 0.0;
  if (e < dim)
#pragma unroll 4
    for (int i = threadIdx.x / 4; i < blocks * count; i += 64) x += (double)partial[((int64_t)(i / count) * all + first + i % count) * dim + e];
  s[threadIdx.x] = x;
  __syncthreads();
  for (int d = 128; d >= 4; d >>= 1) {
    if ((int)threadIdx.x < d) s[threadIdx.x] += s[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x < 4 && e < dim) out[e] = (float)s[threadIdx.x];
}

template <class E>
bool quads(const void* p, int64_t a, int64_t b, int64_t c) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (4 * sizeof(E)) == 0 && a % 4 == 0 && b % 4 == 0 && c % 4 == 0);
}

// Of the last base and number of elements that a thread has asked for (64 powers take 2 us).
const Frequencies& frequencies(double base, int rotary) {
  static thread_local Frequencies f = {};
  static thread_local double of_base = 0.0;
  static thread_local int of_rotary = -1;
  if (base != of_base || rotary != of_rotary) {
    for (int i = 0; i < rotary / 2; ++i) f.turns[i] = std::pow(base, -2.0 * i / rotary) / 6.283185307179586476925;
    of_base = base, of_rotary = rotary;
  }
  return f;
}

template <class E, bool BACK>
int run(const rlk_head_norms& c, const rlk_sequence* grads, float* const* weight_grads, float* partial, hipStream_t s) {
  Norms<E> n = {};
  const rlk_sequence *x[2] = {&c.q, &c.k}, *y[2] = {&c.q_out, &c.k_out};
  n.tokens = c.num_envs * c.seq_len, n.steps = c.seq_len, n.dim = (int)c.dim, n.positions = c.positions;
  n.rotary = c.positions != nullptr ? (int)c.rotary_dim : 0;
  n.eps = (float)c.eps, n.inv_dim = (float)(1.0 / (double)c.dim), n.partial = partial;
  bool vec = c.dim % 8 == 0 && n.rotary % 8 == 0;
  for (int i = 0; i < 2; ++i) {
    Side<E>& d = n.side[i];
    d.x = static_cast<const E*>(x[i]->data), d.y = static_cast<E*>(const_cast<void*>(y[i]->data));
    d.env = x[i]->env_stride, d.step = x[i]->step_stride, d.head = x[i]->head_stride;
    d.yenv = y[i]->env_stride, d.ystep = y[i]->step_stride, d.yhead = y[i]->head_stride;
    d.weight = i ? c.k_weight : c.q_weight, d.heads = (int)(i ? c.k_heads : c.q_heads);
    if (grads) d.g = static_cast<const E*>(grads[i].data), d.genv = grads[i].env_stride, d.gstep = grads[i].step_stride, d.ghead = grads[i].head_stride;
    if (BACK && d.g == nullptr) d.heads = 0;
    d.blocks = (d.heads + kHeads<BACK> - 1) / kHeads<BACK>;
    if (d.heads > 0) vec = vec && quads<E>(d.x, d.env, d.step, d.head) && quads<E>(d.y, d.yenv, d.ystep, d.yhead) && quads<E>(d.g, d.genv, d.gstep, d.ghead);
  }
  const Frequencies& f = frequencies(c.base, n.rotary);
  const int blocks = n.side[0].blocks + n.side[1].blocks;
  n.blocks = blocks;
  int64_t along = 0;
  auto launch = [&](auto N, auto G, auto U, auto halves) {
    if (n.tokens == 0 || blocks == 0) return;
    constexpr int groups = 256 / decltype(G)::value;
    along = (n.tokens + groups - 1) / groups;
    const int64_t most = BACK ? back_blocks(blocks) : std::max<int64_t>(1, (int64_t{1} << 23) / std::max(1, blocks));
    if (along > most) along = most;
    n.stride_envs = along * groups / n.steps, n.stride_steps = along * groups % n.steps;
    norms_kernel<E, decltype(N)::value, decltype(G)::value, decltype(U)::value, decltype(halves)::value, BACK>
        <<<dim3((unsigned)(along * blocks)), dim3(256), 0, s>>>(n, f);
  };
  auto by_size = [&](auto halves) {
    const auto one = std::integral_constant<int, 1>{};
    const auto two = std::integral_constant<int, 2>{};
    const auto four = std::integral_constant<int, 4>{};
    if (vec) {
      const int units = (int)c.dim / 8;
      if (units <= 4) launch(four, four, one, halves);
      else if (units <= 8) launch(four, std::integral_constant<int, 8>{}, one, halves);
      else if (units <= 16) launch(four, std::integral_constant<int, 16>{}, one, halves);
      else launch(four, std::integral_constant<int, 32>{}, one, halves);
    } else if (c.dim <= 32) {
      launch(one, std::integral_constant<int, 16>{}, one, halves);
    } else if (c.dim <= 128) {
      launch(one, std::integral_constant<int, 64>{}, one, halves);
    } else {
      launch(one, std::integral_constant<int, 64>{}, two, halves);
    }
  };
  if (c.interleaved) by_size(std::false_type{});
  else by_size(std::true_type{});
  if (BACK && weight_grads && partial)
    weights_kernel<<<dim3((unsigned)((c.dim + 3) / 4), 2), dim3(256), 0, s>>>(partial, (int)along, n.side[0].blocks, n.side[1].blocks, (int)c.dim,
                                                                             weight_grads[0], weight_grads[1]);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

bool valid_norms(const rlk_head_norms* c) {
  if (!c || c->num_envs < 0 || c->seq_len < 0 || c->q_heads < 0 || c->k_heads < 0 || c->q_heads > (1 << 16) || c->k_heads > (1 << 16) || c->dim < 1 ||
      c->dim > kMostDim || c->rotary_dim < 0 || c->rotary_dim > c->dim || c->rotary_dim % 2 != 0)
    return false;
  if (!(c->base > 0.0) || !std::isfinite(c->base) || !(c->eps >= 0.0) || !std::isfinite((float)c->eps)) return false;
  const uintptr_t low = c->bf16 ? 1u : 3u;
  for (const rlk_sequence* x : {&c->q, &c->k, &c->q_out, &c->k_out})
    if ((reinterpret_cast<uintptr_t>(x->data) & low) != 0) return false;
  const bool any = c->num_envs > 0 && c->seq_len > 0;
  return !any || ((c->q_heads == 0 || c->q.data) && (c->k_heads == 0 || c->k.data));
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" {

int rlk_query_key_norms(const rlk_head_norms* c, void* stream) {
  if (!valid_norms(c)) return RLK_ERR_INVALID_ARGUMENT;
  if (c->num_envs == 0 || c->seq_len == 0 || c->q_heads + c->k_heads == 0) return RLK_OK;
  if ((c->q_heads > 0 && !c->q_out.data) || (c->k_heads > 0 && !c->k_out.data)) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return c->bf16 ? run<bf16, false>(*c, nullptr, nullptr, nullptr, s) : run<float, false>(*c, nullptr, nullptr, nullptr, s);
}

size_t rlk_head_norms_workspace_bytes(const rlk_head_norms* c) {
  if (!valid_norms(c)) return 0;
  const int64_t blocks = (c->q_heads + kHeads<true> - 1) / kHeads<true> + (c->k_heads + kHeads<true> - 1) / kHeads<true>;
  return sizeof(float) * (size_t)(std::max<int64_t>(kResident * device_cus(), blocks) * c->dim);  // (also of one side alone, whose blocks are fewer)
}

int rlk_query_key_norms_backward(const rlk_head_norms* c, rlk_sequence grad_q, rlk_sequence grad_k, float* q_weight_grad, float* k_weight_grad,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_norms(c)) return RLK_ERR_INVALID_ARGUMENT;
  const uintptr_t low = c->bf16 ? 1u : 3u;
  if (((reinterpret_cast<uintptr_t>(grad_q.data) | reinterpret_cast<uintptr_t>(grad_k.data)) & low) != 0) return RLK_ERR_INVALID_ARGUMENT;
  const bool weights = q_weight_grad || k_weight_grad;
  if (weights && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3u) != 0 || workspace_bytes < rlk_head_norms_workspace_bytes(c)))
    return RLK_ERR_WORKSPACE;
  if (!weights && (c->num_envs == 0 || c->seq_len == 0 || c->q_heads + c->k_heads == 0)) return RLK_OK;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const rlk_sequence grads[2] = {grad_q, grad_k};
  float* const to[2] = {q_weight_grad, k_weight_grad};
  float* partial = weights ? static_cast<float*>(workspace) : nullptr;
  return c->bf16 ? run<bf16, true>(*c, grads, to, partial, s) : run<float, true>(*c, grads, to, partial, s);
}

}  // extern "C"
