// rlk_sample.hip -- actions sampled from logits with truncation (include/rl_triton_policy.h).
//
// A weight is exp((x - max) / temperature) as a whole number of 2^-43: computed in float64, and from then on every sum is exact and does not
// depend on its order, so the action is the same however a row is split, and that of the definition in real numbers but for uniform numbers as near
// to a border as the weights' roundings add up to: 2^-44 each, some 1e-13 of a few actions, 1e-11 of a vocabulary's and at most 2^-24 of 2^20, a
// float32 uniform number's last bit.  (Sums in float32 would be off by more than a probability of a large vocabulary.)
//
// Truncations keep a beginning of the actions in the order (logit falling, number rising): what is kept is told by comparing with its last
// member.  Rows of up to 64 actions: a lane per action compares itself with all others.  Longer rows, a workgroup each: of a small top_k
// it lists the candidates and compares them as above; else it finds the last member's place from a histogram of the distances
// to the maximum, counts and weights added up in LDS, and in its bucket by comparison or bisection.
//
// GPU time: [256] of 18 3.8 us, a launch.  [64] of 131072 bf16, top-k 50 with top-p and min-p, 21 us: a workgroup a row, whose two reads are
// some 9 of them (a row of 4096 takes 12), the rest waits for maxima, candidates and their sums.  [512] of 50001 float32, top-p, 92 us: 25.6
// million exponentials in float64 for the histogram and once more for the action's place, and three reads, of which the caches serve two.
// Rows cut into slices with lists of their own, a second launch to join them: 2 to 10 us more up to 131072 actions, half the time only from 2^20
// on.  Sorting the candidates in place of comparing all: 5 us more for 50, from 4 more to 12 less for 256.
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
// (rows of few actions; Weights is for longer ones)
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

// ---- longer rows: a workgroup of NT threads a row.  Thread t has the vectors of 16 bytes t, t + NT, ..., which are read again for every pass: a
// row held in registers is code for each of its elements in each pass, ten times what the instruction cache holds.
constexpr int kTable = 64;
constexpr int kShort = 512;  // lists that are ranked by comparing all with all
template <int NT>
struct Shared {
  static constexpr int WAVES = NT / 64;
  u64 mass[kBuckets];
  uint32_t count[kBuckets];
  u64 list[kList];
  u64 weights[kShort];
  double table[kTable];
  u64 sums[WAVES], sums2[WAVES];
  u64 before, border;
  uint32_t listed;
  int bucket;
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

// How many 64ths of a nat x lies below the largest, held to the buckets there are: 0 for its equals (inf - inf and 0 inf too), the last for
// -inf and what lies far below; monotone in x.
__device__ __forceinline__ float depth(float x, float top, float scale) {
  return fminf(fmaxf((top - x) * scale, 0.f), (float)(kBuckets - 1));
}
__device__ __forceinline__ int bucket(float x, float top, float scale) { return (int)depth(x, top, scale); }
__device__ __forceinline__ float value_of(u64 order) {
  const uint32_t k = (uint32_t)(order >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// What a row's weights are formed with: `unit` turns a difference of logits into 64ths of an octave.
struct Weights {
  const double* table;  // 2^(43 + i / 64)
  double top, unit;
  // The distance of x below the largest, in 64ths of an octave: 0 for its equals (inf - inf too), at least what still rounds to no weight.
  __device__ __forceinline__ double steps(float x) const { return fmax(fmin(((double)x - top) * unit, 0.0), -3693.0); }
  // exp as weight() gives it: 2^(n / 64) from the table, what is left by its series (the first term left out is below 2^-44), rounded to a whole
  // number by what float64 holds beside 2^52.
  __device__ __forceinline__ u64 of_steps(double t) const {
    constexpr double U = 0.69314718055994530942 / 64.0;
    const double n = rint(t), f = t - n;
    const int k = (int)n;
    double e = fma(f, U * U * U * U / 24.0, U * U * U / 6.0);
    e = fma(e, f, U * U / 2.0);
    e = fma(e, f, U);
    e = fma(e, f, 1.0);
    const double r = ldexp(e * table[k & (kTable - 1)], k >> 6);
    return (u64)(__double_as_longlong(r + 0x1p52) & 0xfffffffffffffll);
  }
  __device__ __forceinline__ u64 operator()(float x) const { return of_steps(steps(x)); }
};

template <class E>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(E);
  typedef uint32_t By2 __attribute__((ext_vector_type(4), aligned(2)));  // (an access need not be aligned to its size)
  typedef uint32_t By4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef typename std::conditional<sizeof(E) == 2, By2, By4>::type Words_;
  u32x4 w;
  __device__ __forceinline__ void load(const E* row, int first) { w = *reinterpret_cast<const Words_*>(row + first); }
  __device__ __forceinline__ void load_some(const E* row, int first, int count) {  // -inf behind the row's end
    if (first + N <= count) return load(row, first);
    const uint32_t none = sizeof(E) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = none;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (first + i >= count) continue;
      if constexpr (sizeof(E) == 4) w[i] = __float_as_uint(load_one(row + first + i));
      else w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | (uint32_t)(row + first + i)->bits << 16 : (w[i / 2] & 0xffff0000u) | (row + first + i)->bits;
    }
  }
  __device__ __forceinline__ float get(int i) const { return Words<E>::get(w[i / Words<E>::kPerWord], i % Words<E>::kPerWord); }
};

// Two elements at a time: the compiler would work on a whole vector's side by side, in twice the registers.
__device__ __forceinline__ void apart(int e) {
  if (e & 1) __builtin_amdgcn_sched_barrier(0);
}

template <class E, int NT>
__global__ __launch_bounds__(NT, NT >= 512 ? 4 : 2) void row_kernel(const Sampling s) {
  typedef Shared<NT> M;
  constexpr int N = Vec<E>::N, WAVES = NT / 64;
  __shared__ M m;
  u64* const part = m.list;  // [trip][wavefront], once the list has had its use
  static_assert(RLK_MOST_SAMPLED_ACTIONS / 4 / 64 <= kList);
  const int64_t row = s.first + blockIdx.x;
  const E* p = row_of<E>(s, row);
  const int A = s.actions, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int trips = (A + NT * N - 1) / (NT * N);

  // Goes over the row, the next U vectors on their way: f(vector, its first action, trip).
  const int whole = A / (NT * N);  // trips in which all threads have whole vectors
  auto each = [&](auto ahead, auto f) {
    constexpr int U = decltype(ahead)::value;
    Vec<E> next[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (i < whole) next[i].load(p, (i * NT + tid) * N);
#pragma unroll 1
    for (int c = 0; c < whole; c += U) {
      Vec<E> x[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        x[i] = next[i];
        if (c + U + i < whole) next[i].load(p, ((c + U + i) * NT + tid) * N);
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (c + i < whole) f(x[i], ((c + i) * NT + tid) * N, c + i);
    }
    if (whole < trips) {
      Vec<E> x;
      x.load_some(p, (whole * NT + tid) * N, A);
      f(x, (whole * NT + tid) * N, whole);
    }
  };
  const std::integral_constant<int, 4> light{};  // (passes of a few instructions an element)
  const std::integral_constant<int, 2> heavy{};
  // The same, one element after the other: for passes that are made seldom.
  auto each_again = [&](auto f) {
    for (int c = 0; c < trips; ++c) {
#pragma unroll 1
      for (int e = 0; e < N; ++e) {
        const int i = (c * NT + tid) * N + e;
        if (i < A) f(load_one(p + i), i);
      }
    }
  };

  for (int i = tid; i < kBuckets; i += NT) m.mass[i] = 0, m.count[i] = 0;
  if (tid < kTable) m.table[tid] = exp2((double)tid / kTable) * 0x1p43;
  if (tid == 0) m.listed = 0;
  float top = -INFINITY, first_of = -INFINITY;
  bool bad = false;
  each(light, [&](const Vec<E>& x, int, int) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float y = x.get(e);
      bad |= y != y;
      top = fmaxf(top, y);
    }
  });
  first_of = top;  // of this thread's
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  {
    const bool any = __any(bad);
    if (lane == 0) m.sums[wave] = __float_as_uint(top), m.sums2[wave] = any;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) top = fmaxf(top, __uint_as_float((uint32_t)m.sums[i])), bad |= m.sums2[i] != 0;
  }
  if (bad || top == -INFINITY) {
    if (tid == 0) s.out[row] = -1, s.log_probs[row] = bad ? NAN : -INFINITY;
    return;
  }
  const float scale = (float)s.inv_temperature * kPerNat;
  const Weights weights{m.table, (double)top, s.inv_temperature * (64.0 * 1.4426950408889634074)};
  auto take = [&](int action, float x, u64 total) { s.out[row] = action, s.log_probs[row] = log_prob(distance(x, top, s), total); };

  // The bucket in which the counts or weights, added up from the first bucket on, reach `want`, and what lies before it.  `all`: their sum.
  auto find_bucket = [&](bool counts, double want, u64* all) {
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
      if (all != nullptr && tid == 63) m.border = upto;
      if (all == nullptr) {
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
          m.bucket = b, m.before = c, m.listed = 0;
        }
      }
    }
    __syncthreads();
    if (all != nullptr) *all = m.border;
  };

  u64 border = 0;  // the last that is kept, in order()
  if (s.by_k && s.top_k <= 256) {
    // As many of the threads' largest as top_k asks for are at least the border: what is before or in their last one's bucket are candidates.
    if (first_of > -INFINITY) atomicAdd(&m.count[bucket(first_of, top, scale)], 1u);
    find_bucket(true, (double)s.top_k, nullptr);
    const int last = m.bucket;
    const float reach = (float)(last + 1);  // (the last bucket's depths are its number)
    each(light, [&](const Vec<E>& x, int first, int) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < N; ++e) any |= depth(x.get(e), top, scale) < reach;
      if (!any) return;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float y = x.get(e);
        if (!(depth(y, top, scale) < reach) || y == -INFINITY) continue;
        const uint32_t at = atomicAdd(&m.listed, 1u);
        if (at < kShort) m.list[at] = order(y, first + e);
      }
    });
    __syncthreads();
    const int n = (int)m.listed;
    if (n <= kShort) {
      // (comparisons by eights: one after the other each would wait for the LDS)
      constexpr int PER = (kShort + NT - 1) / NT;
      const int padded = (n + 7) & ~7;
      u64 mine[PER], w[PER], before[PER];
      int rank[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int at = tid + NT * i;
        mine[i] = at < n ? m.list[at] : 0;
        w[i] = at < n ? weights(value_of(mine[i])) : 0;
        if (at < n) m.weights[at] = w[i];
        else if (at < padded) m.list[at] = m.weights[at] = 0;
        before[i] = 0, rank[i] = 0;
      }
      __syncthreads();
      if (wave * 64 < n)
        for (int j0 = 0; j0 < padded; j0 += 8) {
          u64 other[8], wj[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) other[j] = m.list[j0 + j], wj[j] = m.weights[j0 + j];
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const bool first = other[j] > mine[i];
              rank[i] += first;
              before[i] += first ? wj[j] : 0;
            }
        }
      u64 left = 0;  // what top_k leaves
#pragma unroll
      for (int i = 0; i < PER; ++i) left += tid + NT * i < n && rank[i] < s.top_k ? w[i] : 0;
      left = all_sum<NT>(left, m.sums);
      u64 total = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int at = tid + NT * i;
        const bool kept = at < n && rank[i] < s.top_k && (!s.by_p || (double)before[i] < s.top_p * (double)left) &&
                          (!s.by_min || distance(value_of(mine[i]), top, s) >= s.least);
        w[i] = kept ? w[i] : 0;
        if (at < n) m.weights[at] = w[i];
        total += w[i];
      }
      total = all_sum<NT>(total, m.sums);
      const u64 want = share(s.uniforms[row], total);
      __syncthreads();
      u64 upto[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) upto[i] = 0;
      if (wave * 64 < n)
        for (int j0 = 0; j0 < padded; j0 += 8) {
          uint32_t other[8];  // (~action: an earlier one has a larger number)
          u64 wj[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) other[j] = (uint32_t)m.list[j0 + j], wj[j] = m.weights[j0 + j];
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < PER; ++i) upto[i] += other[j] >= (uint32_t)mine[i] ? wj[j] : 0;
        }
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (w[i] != 0 && upto[i] > want && upto[i] - w[i] <= want) take((int)~(uint32_t)mine[i], value_of(mine[i]), total);
      return;
    }
    for (int i = tid; i < kBuckets; i += NT) m.count[i] = 0;
    __syncthreads();
  }

  if (s.by_k || s.by_p) {
    if (s.by_k)
      each(light, [&](const Vec<E>& x, int, int) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (x.get(e) > -INFINITY) atomicAdd(&m.count[bucket(x.get(e), top, scale)], 1u);
      });
    if (s.by_p)
      each(heavy, [&](const Vec<E>& x, int, int) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          atomicAdd(&m.mass[bucket(x.get(e), top, scale)], weights(x.get(e)));
          apart(e);
        }
      });

    // The last member of the shortest beginning that reaches `want`: of counts, then of weights.
    for (int round = s.by_k ? 0 : 1; round < (s.by_p ? 2 : 1); ++round) {
      const bool counts = round == 0;
      double want = (double)s.top_k;
      if (!counts) {
        u64 left = 0;  // what top_k leaves
        if (s.by_k) {
          each(heavy, [&](const Vec<E>& x, int first, int) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
              left += order(x.get(e), first + e) >= border ? weights(x.get(e)) : 0;
              apart(e);
            }
          });
          left = all_sum<NT>(left, m.sums);
        } else {
          find_bucket(false, 0.0, &left);
        }
        want = s.top_p * (double)left;
      }
      find_bucket(counts, want, nullptr);
      const int b = m.bucket;
      const u64 before = m.before;
      u64 lo = ~0ull, hi = 0;
      each(light, [&](const Vec<E>& x, int first, int) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float d = depth(x.get(e), top, scale);
          any |= d >= (float)b && d < (float)(b + 1);
        }
        if (!any) return;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float y = x.get(e);
          if (bucket(y, top, scale) != b || first + e >= A) continue;
          const u64 o = order(y, first + e);
          lo = o < lo ? o : lo, hi = o > hi ? o : hi;
          const uint32_t at = atomicAdd(&m.listed, 1u);
          if (at < kList) m.list[at] = o;
        }
      });
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        const u64 a = (u64)__shfl_xor((long long)lo, d), c = (u64)__shfl_xor((long long)hi, d);
        lo = a < lo ? a : lo, hi = c > hi ? c : hi;
      }
      if (lane == 0) m.sums[wave] = lo, m.sums2[wave] = hi;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WAVES; ++i) lo = m.sums[i] < lo ? m.sums[i] : lo, hi = m.sums2[i] > hi ? m.sums2[i] : hi;
      const uint32_t n = m.listed;
      if (n <= kShort) {
        // each compares itself with all
        const uint32_t padded = (n + 7) & ~7u;
        if (tid == 0) m.border = lo;  // (all of the bucket, if it never is enough)
        for (uint32_t i = tid; i < padded; i += NT) {
          if (i >= n) m.list[i] = 0;
          m.weights[i] = i >= n ? 0 : counts ? 1 : weights(value_of(m.list[i]));
        }
        __syncthreads();
        for (uint32_t i = tid; i < n; i += NT) {
          const u64 mine = m.list[i];
          u64 sum = before;
          for (uint32_t j0 = 0; j0 < padded; j0 += 8) {
            u64 other[8], wj[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) other[j] = m.list[j0 + j], wj[j] = m.weights[j0 + j];
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += other[j] > mine ? wj[j] : 0;
          }
          if ((double)sum < want && (double)(sum + m.weights[i]) >= want) m.border = mine;
        }
        __syncthreads();
        lo = m.border;
      } else {
        // the largest order in [lo, hi] from which on there is enough
        while (lo < hi) {
          const u64 mid = lo + (hi - lo) / 2 + ((hi - lo) & 1);
          u64 x = 0;
          if (n <= kList) {
            for (uint32_t i = tid; i < n; i += NT)
              if (m.list[i] >= mid) x += counts ? 1 : weights(value_of(m.list[i]));
          } else {
            each_again([&](float y, int i) {
              if (bucket(y, top, scale) == b && order(y, i) >= mid) x += counts ? 1 : weights(y);
            });
          }
          if ((double)(before + all_sum<NT>(x, m.sums)) >= want) lo = mid;
          else hi = mid - 1;
        }
      }
      border = lo > border ? lo : border;
    }
  }

  // Of the kept ones in the order of their numbers: the weights of a wavefront's vectors of a trip, of these the one up to which there is enough, and in
  // it the action.
  __syncthreads();
  const float border_value = border != 0 ? value_of(border) : -INFINITY;
  const int border_action = border != 0 ? (int)~(uint32_t)border : A;
  const double least = s.least * (64.0 * 1.4426950408889634074);
  auto kept_weight = [&](float x, int i) -> u64 {
    if (!(x > border_value || (x == border_value && i <= border_action))) return 0;
    const double t = weights.steps(x);
    return !s.by_min || t >= least ? weights.of_steps(t) : 0;
  };
  each(heavy, [&](const Vec<E>& x, int first, int c) {
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      sum += kept_weight(x.get(e), first + e);
      apart(e);
    }
    if (__any(sum != 0)) {
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) sum += (u64)__shfl_xor((long long)sum, d);
    }
    if (lane == 0) part[c * WAVES + wave] = sum;
  });
  __syncthreads();
  const int parts = trips * WAVES;
  u64 total = 0;
  for (int i = tid; i < parts; i += NT) total += part[i];
  total = all_sum<NT>(total, m.sums);
  const u64 want = share(s.uniforms[row], total);
  if (wave != 0) return;
  u64 before = 0;
  int at = 0;
  for (int i0 = 0;; i0 += 64) {  // (ends: `want` is below the total)
    const u64 x = i0 + lane < parts ? part[i0 + lane] : 0;
    u64 upto = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const u64 b = (u64)__shfl_up((long long)upto, d);
      if (lane >= d) upto += b;
    }
    const u64 beyond = __ballot(before + upto > want);
    if (beyond != 0 || i0 + 64 >= parts) {
      const int l = beyond != 0 ? __ffsll((long long)beyond) - 1 : 63;
      before += shfl64(upto - x, l, 64);
      at = i0 + l;
      break;
    }
    before += shfl64(upto, 63, 64);
  }
  const int first = (at / WAVES * NT + at % WAVES * 64 + lane) * N;
  Vec<E> x;
  x.load_some(p, first, A);
  u64 sum = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) sum += kept_weight(x.get(e), first + e);
  u64 upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 b = (u64)__shfl_up((long long)upto, d);
    if (lane >= d) upto += b;
  }
  before += upto - sum;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const u64 w = kept_weight(x.get(e), first + e);
    if (w != 0 && before <= want && before + w > want) take(first + e, x.get(e), total);
    before += w;
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
      // A row to a CU: by 1024 threads ([64] of 131072, top-k: 26 us against 33 by 512; by now 21).  More: two workgroups of 512 a CU, one of which works while the
      // other waits (top-p, [512] of 50001: 105 us, 127 by 1024).
      if (s.actions <= 4096) row_kernel<E, 256><<<grid, dim3(256), 0, stream>>>(s);
      else if (rows <= device_cus()) row_kernel<E, 1024><<<grid, dim3(1024), 0, stream>>>(s);
      else row_kernel<E, 512><<<grid, dim3(512), 0, stream>>>(s);
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
