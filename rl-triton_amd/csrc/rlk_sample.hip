// rlk_sample.hip -- actions sampled from logits with truncation (include/rl_triton_policy.h).
//
// A weight is exp((x - max) / temperature) as a whole number of 2^-43: computed in float64, and from then on every sum is exact and does not
// depend on its order, so the action is the same however a row is split, and that of the definition in real numbers but for uniform numbers within
// some 1e-13 of a border.  (Sums in float32 would be off by more than a probability of a large vocabulary.)  What the rounding leaves out of
// 2^20 actions is below 2^-24, a float32 uniform number's last bit.
//
// Truncations keep a beginning of the actions in the order (logit falling, number rising): what is kept is told by comparing with its last
// member.  Rows of up to 64 actions: a lane per action compares itself with all others.  Longer rows: a workgroup finds the last member's
// place from a histogram of the distances to the maximum, counts and weights added up in LDS, and in its bucket by bisection.
#include "rlk_launch.hpp"
#include "rlk_policy.hpp"

namespace rlk {
namespace {

constexpr int kBuckets = 2048;
constexpr float kPerNat = 64.f;  // buckets of a 64th: 32 below the largest
constexpr int kList = 4096;

struct Sampling {
  const void* logits;
  int64_t rows, steps, env_stride, step_stride, first;
  int actions;
  const float* uniforms;
  double inv_temperature, top_p, least;  // least: log(min_p)
  int top_k;
  bool by_k, by_p, by_min;
  int64_t* out;
  float* log_probs;
};

typedef unsigned long long u64;

// exp(z) for z <= 0 as a multiple of 2^-43, rounded to nearest.
__device__ __forceinline__ u64 weight(double z) {
  if (!(z > -40.0)) return 0;  // (below half a unit)
  return (u64)__double2ll_rn(exp(z) * 0x1p43);
}
__device__ __forceinline__ double distance(float x, float top, const Sampling& s) {
  return x == top ? 0.0 : ((double)x - (double)top) * s.inv_temperature;  // (of a largest of +inf only its equals have weight)
}
// Actions in their order: a larger number comes first.
__device__ __forceinline__ uint32_t key(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);  // (-0 and 0 are equal)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 order(float x, int i) { return (u64)key(x) << 32 | (uint32_t)~i; }

__device__ __forceinline__ u64 shfl64(u64 x, int lane, int width) { return (u64)__shfl((long long)x, lane, width); }

// The share of `total` that a uniform number stands for, below it.
__device__ __forceinline__ u64 share(float u, u64 total) {
  const double t = (double)fminf(fmaxf(u, 0.f), 1.f) * (double)total;
  const u64 n = (u64)t;
  return n < total ? n : total - 1;
}
__device__ __forceinline__ float log_prob(double z, u64 total) { return (float)(z - log((double)total * 0x1p-43)); }

template <class E>
__device__ __forceinline__ const E* row_of(const Sampling& s, int64_t row) {
  return static_cast<const E*>(s.logits) + row / s.steps * s.env_stride + row % s.steps * s.step_stride;
}

// Rows of up to G actions: a lane per action, 256 / G rows a workgroup.
template <class E, int G>
__global__ __launch_bounds__(256) void few_kernel(const Sampling s) {
  const int lane = threadIdx.x & (G - 1);
  const int64_t row = s.first + (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (row >= s.rows) return;
  const bool there = lane < s.actions;
  const float x = there ? load_one(row_of<E>(s, row) + lane) : -INFINITY;
  float top = x;
  bool bad = x != x;
#pragma unroll
  for (int d = 1; d < G; d <<= 1) {
    const float other = __shfl_xor(top, d);
    bad |= (bool)__shfl_xor((int)bad, d);
    top = fmaxf(top, other);
  }
  if (bad || top == -INFINITY) {
    if (lane == 0) s.out[row] = -1, s.log_probs[row] = bad ? NAN : -INFINITY;
    return;
  }
  const double z = distance(x, top, s);
  const u64 w = there ? weight(z) : 0;
  bool kept = there && x > -INFINITY && (!s.by_min || z >= s.least);
  if (s.by_k || s.by_p) {
    const u64 mine = order(x, lane);
    int rank = 0;
    u64 before = 0, held = w;  // held: what top_k leaves
    for (int j = 0; j < s.actions; ++j) {
      const u64 other = shfl64(mine, j, G), wj = shfl64(w, j, G);
      const bool first = other > mine;
      rank += first;
      before += first ? wj : 0;
    }
    kept = kept && (!s.by_k || rank < s.top_k);
    if (s.by_p) {
      held = there && (!s.by_k || rank < s.top_k) ? w : 0;
#pragma unroll
      for (int d = 1; d < G; d <<= 1) held += (u64)__shfl_xor((long long)held, d);
      kept = kept && (double)before < s.top_p * (double)held;
    }
  }
  u64 sum = kept ? w : 0;
#pragma unroll
  for (int d = 1; d < G; d <<= 1) {
    const u64 b = (u64)__shfl_up((long long)sum, d, G);
    if (lane >= d) sum += b;
  }
  const u64 total = shfl64(sum, G - 1, G), want = share(s.uniforms[row], total);
  const u64 beyond = __ballot(sum > want) >> ((threadIdx.x & 63) & ~(G - 1));
  if (lane == __ffsll((long long)beyond) - 1) s.out[row] = lane, s.log_probs[row] = log_prob(z, total);
}

// ---- longer rows: a workgroup of NT threads a row.
template <int NT>
struct Shared {
  u64 mass[kBuckets];
  uint32_t count[kBuckets];
  u64 list[kList];
  u64 sums[NT / 64], sums2[NT / 64];
  u64 scan[NT / 64 + 1];
  uint32_t listed;
  int found;
};

template <int NT>
__device__ __forceinline__ u64 all_sum(u64 x, u64* s) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += (u64)__shfl_xor((long long)x, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  x = s[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) x += s[i];
  return x;
}

__device__ __forceinline__ int bucket(float x, float top, float scale) {
  const float d = (top - x) * scale;
  return x == top ? 0 : d < (float)(kBuckets - 1) ? (int)d : kBuckets - 1;  // (monotone in x; -inf and what lies far below are in the last)
}

template <class E, int NT>
__global__ __launch_bounds__(NT) void row_kernel(const Sampling s) {
  __shared__ Shared<NT> m;
  const int64_t row = s.first + blockIdx.x;
  const E* p = row_of<E>(s, row);
  const int A = s.actions, tid = threadIdx.x;

  float top = -INFINITY;
  bool bad = false;
  for (int i = tid; i < A; i += NT) {
    const float x = load_one(p + i);
    bad |= x != x;
    top = fmaxf(top, x);
  }
  {
    u64 b = order(top, 0);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const u64 o = (u64)__shfl_xor((long long)b, d);
      b = o > b ? o : b;
    }
    const bool any = __any(bad);
    if ((tid & 63) == 0) m.sums[tid >> 6] = b, m.sums2[tid >> 6] = any;
    __syncthreads();
    for (int i = 0; i < NT / 64; ++i) b = m.sums[i] > b ? m.sums[i] : b, bad |= m.sums2[i] != 0;
    const uint32_t k = (uint32_t)(b >> 32);
    top = __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  }
  if (bad || top == -INFINITY) {
    if (tid == 0) s.out[row] = -1, s.log_probs[row] = bad ? NAN : -INFINITY;
    return;
  }

  u64 border = 0;  // the last that is kept, in order()
  if (s.by_k || s.by_p) {
    const float scale = (float)s.inv_temperature * kPerNat;
    for (int i = tid; i < kBuckets; i += NT) m.mass[i] = 0, m.count[i] = 0;
    __syncthreads();
    for (int i = tid; i < A; i += NT) {
      const float x = load_one(p + i);
      const int b = bucket(x, top, scale);
      if (s.by_k) atomicAdd(&m.count[b], 1u);
      if (s.by_p) atomicAdd(&m.mass[b], weight(distance(x, top, s)));
    }
    __syncthreads();

    // The last member of the shortest beginning that reaches `want`, of counts or weights; `held` becomes its weight.
    auto last_of = [&](bool counts, double want, u64* held) {
      // its bucket, and what lies before it: a wavefront's lanes take 32 buckets each
      __syncthreads();
      if (tid < 64) {
        constexpr int PER = kBuckets / 64;
        u64 x = 0;
        for (int i = 0; i < PER; ++i) x += counts ? (u64)m.count[PER * tid + i] : m.mass[PER * tid + i];
        u64 upto = x;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const u64 b = (u64)__shfl_up((long long)upto, d);
          if (tid >= d) upto += b;
        }
        const u64 reached = __ballot((double)upto >= want);
        const int first = reached != 0 ? __ffsll((long long)reached) - 1 : 63;
        if (tid == first) {
          u64 c = upto - x;
          int b = PER * tid;
          for (; b < PER * tid + PER - 1; ++b) {
            const u64 n = counts ? (u64)m.count[b] : m.mass[b];
            if ((double)(c + n) >= want) break;
            c += n;
          }
          m.found = b, m.scan[0] = c, m.listed = 0;
        }
      }
      __syncthreads();
      const int b = m.found;
      const u64 before = m.scan[0];
      u64 lo = ~0ull, hi = 0;
      for (int i = tid; i < A; i += NT) {
        const float x = load_one(p + i);
        if (bucket(x, top, scale) != b) continue;
        const u64 o = order(x, i);
        lo = o < lo ? o : lo, hi = o > hi ? o : hi;
        const uint32_t at = atomicAdd(&m.listed, 1u);
        if (at < kList) m.list[at] = o;
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        const u64 a = (u64)__shfl_xor((long long)lo, d), c = (u64)__shfl_xor((long long)hi, d);
        lo = a < lo ? a : lo, hi = c > hi ? c : hi;
      }
      __syncthreads();
      if ((tid & 63) == 0) m.sums[tid >> 6] = lo, m.sums2[tid >> 6] = hi;
      __syncthreads();
      for (int i = 0; i < NT / 64; ++i) lo = m.sums[i] < lo ? m.sums[i] : lo, hi = m.sums2[i] > hi ? m.sums2[i] : hi;
      const uint32_t n = m.listed;
      auto value = [&](u64 o) {
        const uint32_t k = (uint32_t)(o >> 32);
        return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
      };
      auto from = [&](u64 least, bool weights) {  // the count or weight of the bucket's members from `least` on
        u64 x = 0;
        if (n <= kList) {
          for (uint32_t i = tid; i < n; i += NT)
            if (m.list[i] >= least) x += weights ? weight(distance(value(m.list[i]), top, s)) : 1;
        } else {
          for (int i = tid; i < A; i += NT) {
            const float y = load_one(p + i);
            if (bucket(y, top, scale) == b && order(y, i) >= least) x += weights ? weight(distance(y, top, s)) : 1;
          }
        }
        return all_sum<NT>(x, m.sums);
      };
      // the largest o in [lo, hi] from which on there is enough (all of the bucket, if it never is)
      while (lo < hi) {
        const u64 mid = lo + (hi - lo) / 2 + ((hi - lo) & 1);
        if ((double)(before + from(mid, !counts)) >= want) lo = mid;
        else hi = mid - 1;
      }
      if (held != nullptr) {
        // what the buckets before hold
        u64 x = 0;
        for (int i = tid; i < b; i += NT) x += m.mass[i];
        x = all_sum<NT>(x, m.sums);
        *held = x + from(lo, true);
      }
      return lo;
    };
    u64 held = 0;
    if (s.by_k && s.top_k < A) border = last_of(true, (double)s.top_k, s.by_p ? &held : nullptr);
    else if (s.by_p) {
      for (int i = tid; i < kBuckets; i += NT) held += m.mass[i];
      held = all_sum<NT>(held, m.sums);
    }
    if (s.by_p) {
      const u64 other = last_of(false, s.top_p * (double)held, nullptr);
      border = other > border ? other : border;
    }
  }

  // Of the kept ones in the order of their numbers: NT at a time, their weights added up.
  auto kept_weight = [&](int i, double* z) -> u64 {
    if (i >= A) return 0;
    const float x = load_one(p + i);
    *z = distance(x, top, s);
    return order(x, i) >= border && (!s.by_min || *z >= s.least) ? weight(*z) : 0;
  };
  u64 total = 0;
  double z = 0.0;
  for (int i = tid; i < A; i += NT) total += kept_weight(i, &z);
  total = all_sum<NT>(total, m.sums);
  const u64 want = share(s.uniforms[row], total);
  u64 before = 0;
  for (int i0 = 0; i0 < A; i0 += NT) {
    const u64 w = kept_weight(i0 + tid, &z);
    u64 sum = w;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const u64 b = (u64)__shfl_up((long long)sum, d);
      if ((tid & 63) >= d) sum += b;
    }
    __syncthreads();
    if ((tid & 63) == 63) m.sums[tid >> 6] = sum;
    __syncthreads();
    u64 base = before;
    for (int i = 0; i < NT / 64; ++i) {
      if (i < tid >> 6) base += m.sums[i];
      before += m.sums[i];
    }
    if (base + sum > want && base + sum - w <= want) s.out[row] = i0 + tid, s.log_probs[row] = log_prob(z, total);
    if (before > want) break;
  }
}

template <class E>
int launch(Sampling s, hipStream_t stream) {
  const int64_t rows = s.rows;
  const int G = s.actions <= 16 ? 16 : s.actions <= 32 ? 32 : 64;
  const int64_t most = int64_t{1} << 21;  // workgroups of a launch
  if (s.actions <= 64) {
    const int64_t per = 256 / G;
    for (s.first = 0; s.first < rows; s.first += most * per) {
      const int64_t units = (rows - s.first + per - 1) / per;
      const dim3 grid((unsigned)(units < most ? units : most));
      if (G == 16) few_kernel<E, 16><<<grid, dim3(256), 0, stream>>>(s);
      else if (G == 32) few_kernel<E, 32><<<grid, dim3(256), 0, stream>>>(s);
      else few_kernel<E, 64><<<grid, dim3(256), 0, stream>>>(s);
    }
  } else {
    for (s.first = 0; s.first < rows; s.first += most) {
      const dim3 grid((unsigned)(rows - s.first < most ? rows - s.first : most));
      if (s.actions <= 4096) row_kernel<E, 256><<<grid, dim3(256), 0, stream>>>(s);
      else row_kernel<E, 1024><<<grid, dim3(1024), 0, stream>>>(s);
    }
  }
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" int rlk_sample_actions(const rlk_sampling* c, void* stream) {
  if (!c || c->num_envs < 0 || c->seq_len < 0 || c->num_actions < 1 || c->num_actions > RLK_MOST_SAMPLED_ACTIONS || c->top_k < 0)
    return RLK_ERR_INVALID_ARGUMENT;
  if (!(c->temperature >= RLK_LEAST_TEMPERATURE && c->temperature <= RLK_LARGEST_TEMPERATURE) || !(c->top_p > 0.0 && c->top_p <= 1.0) ||
      !(c->min_p >= 0.0 && c->min_p <= 1.0))
    return RLK_ERR_INVALID_ARGUMENT;
  if (c->num_envs == 0 || c->seq_len == 0) return RLK_OK;
  if (!c->logits || !c->uniforms || !c->actions || !c->log_probs || (reinterpret_cast<uintptr_t>(c->logits) & (c->bf16 ? 1u : 3u)) != 0)
    return RLK_ERR_INVALID_ARGUMENT;
  Sampling s = {};
  s.logits = c->logits, s.rows = c->num_envs * c->seq_len, s.steps = c->seq_len, s.env_stride = c->env_stride, s.step_stride = c->step_stride;
  s.actions = (int)c->num_actions, s.uniforms = c->uniforms, s.inv_temperature = 1.0 / c->temperature;
  s.by_k = c->top_k > 0 && c->top_k < c->num_actions, s.top_k = s.by_k ? (int)c->top_k : s.actions;
  s.by_p = c->top_p < 1.0, s.top_p = c->top_p;
  s.by_min = c->min_p > 0.0, s.least = s.by_min ? std::log(c->min_p) : 0.0;
  s.out = c->actions, s.log_probs = c->log_probs;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return c->bf16 ? launch<bf16>(s, st) : launch<float>(s, st);
}
