// rlk_action_rows.hpp -- rows of logits: softmax statistics in one read, and the gradient written from the
// registers that still hold the row.
//
// For a row x and temperature tau, with c = log2(e) / tau, m = max x and y_j = (x_j - m) c:
//   s = sum 2^y,  u = sum 2^y y,  log p_j = ln2 (y_j - log2 s),  H = ln2 (log2 s - u / s)
// and for upstream gradients g of log p_a and h of H
//   dx_j = (g ([j = a] - p_j) - h p_j (log p_j + H)) / tau.
// x - m is formed before the product: the largest logit's y is then 0 (one fma, x c - (m c rounded), leaves a residue
// there, and log-probabilities above 0), and a row whose logits are all the type's lowest value is uniform and
// not NaN.  Logits of -inf have no part (p = 0, nothing in u); a row of them alone has log p = -inf,
// H = 0 and a zero gradient.  NaN and +inf make the row's outputs NaN through s.
#pragma once
#include "rlk_policy.hpp"

namespace rlk {

template <class E>
struct ActionRows {
  const E* logits;
  const int64_t* actions;
  int64_t rows, seq_len, env_stride, step_stride;
  int A;
  float c, inv_tau;
};

template <class E>
__device__ __forceinline__ const E* row_base(const ActionRows<E>& a, int64_t row) {
  if (a.env_stride == a.seq_len * a.step_stride) return a.logits + row * a.step_stride;
  const int64_t e = row / a.seq_len;
  return a.logits + e * a.env_stride + (row - e * a.seq_len) * a.step_stride;
}

// The row as the lanes of a group hold it: `nfull` vectors of 16 bytes at 16-byte boundaries from element
// `head` on, lane l holding vectors l, l + LANES, ...; the at most 2 (VEC - 1) elements before and after
// them are held one by one.
template <class E>
struct Frame {
  static constexpr int VEC = 16 / (int)sizeof(E);
  const E* base;
  int A, head, nfull;
  __device__ Frame(const E* row, int A_) : base(row), A(A_) {
    const int off = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(E)) & (VEC - 1));
    head = (VEC - off) & (VEC - 1);
    if (head > A) head = A;
    nfull = (A - head) / VEC;
  }
  // the element that edge slot `i` (0 .. 2 VEC - 1) stands for, or -1
  __device__ int edge(int i) const {
    if (i < VEC) return i < head ? i : -1;
    const int j = head + nfull * VEC + (i - VEC);
    return j < A ? j : -1;
  }
};

__device__ __forceinline__ u32x4 load_words(const void* p) {
  return __builtin_nontemporal_load(static_cast<const u32x4*>(p));
}
__device__ __forceinline__ void store_words(void* p, u32x4 w) {
  __builtin_nontemporal_store(w, static_cast<u32x4*>(p));
}

// The k-th vector of a lane of LANES from `first`, a row's first whole vector: the same address for the wavefront plus a
// 32-bit offset for the lane (as one offset, formed in 64 bits for every k, they filled 32 registers of a held row).
template <int LANES, class T>
__device__ __forceinline__ T* vector_at(T* first, int k, int lane) {
  typedef std::conditional_t<std::is_const_v<T>, const char, char> Byte;
  return reinterpret_cast<T*>(reinterpret_cast<Byte*>(first) + (int64_t)k * (LANES * 16) + (uint32_t)(lane * 16));
}

// The row that a group of LANES threads works on: one for a whole wavefront, and known to be.
template <int LANES>
__device__ __forceinline__ int64_t first_row() {
  constexpr int PER = LANES > 256 ? 1 : 256 / LANES;
  int group = threadIdx.x / LANES;
  if constexpr (LANES >= 64) group = __builtin_amdgcn_readfirstlane(group);
  return (int64_t)blockIdx.x * PER + group;
}

template <class E>
__device__ __forceinline__ void unpack(u32x4 w, float (&x)[16 / sizeof(E)]) {
  constexpr int P = Words<E>::kPerWord;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < P; ++k) x[i * P + k] = Words<E>::get(w[i], k);
}
template <class E>
__device__ __forceinline__ u32x4 pack(const float (&x)[16 / sizeof(E)]) {
  constexpr int P = Words<E>::kPerWord;
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = Words<E>::put(x[i * P], x[i * P + P - 1]);
  return w;
}

// Sums and maxima over the LANES lanes that hold a row: lanes of a wavefront, or the whole workgroup
// (s: LANES / 64 floats, used alternately by two reductions).
template <int LANES>
__device__ __forceinline__ float group_max(float x, float* s) {
#pragma unroll
  for (int d = (LANES < 64 ? LANES : 64) / 2; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    x = s[0];
#pragma unroll
    for (int i = 1; i < LANES / 64; ++i) x = fmaxf(x, s[i]);
  }
  return x;
}
template <int LANES>
__device__ __forceinline__ void group_sum2(float& a, float& b, float* s) {
#pragma unroll
  for (int d = (LANES < 64 ? LANES : 64) / 2; d > 0; d >>= 1) a += __shfl_xor(a, d), b += __shfl_xor(b, d);
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a, s[LANES / 64 + (threadIdx.x >> 6)] = b;
    __syncthreads();
    a = s[0], b = s[LANES / 64];
#pragma unroll
    for (int i = 1; i < LANES / 64; ++i) a += s[i], b += s[LANES / 64 + i];
  }
}

constexpr float kDeep = -1024.f;  // 2^kDeep is 0: below it y only has to be finite where it multiplies 2^y

__device__ __forceinline__ void softmax_add(float y, float& s, float& u) {
  const float e = __builtin_amdgcn_exp2f(y);
  s += e;
  u = fmaf(e, fmaxf(y, kDeep), u);  // (y = -inf: e = 0 counts as 0)
}

constexpr float kLn2 = 0.69314718055994531f;

struct RowStats {
  float m, s, u;  // of a row without any finite logit: m = 0, s = u = 0
  __device__ bool empty() const { return s == 0.f; }
  __device__ float log2s() const { return empty() ? 0.f : __log2f(s); }
  // of an action whose logit is x
  __device__ float log_prob(float x, float c) const { return empty() && x == x ? -INFINITY : ((x - m) * c - log2s()) * kLn2; }
  __device__ float entropy() const { return empty() ? 0.f : (log2s() - u / s) * kLn2; }
};

// What the writer of a gradient needs: p = 2^(y - log2 s), dx = p (a1 + b1 (y - log2 s)), plus g at the action.
struct RowGrad {
  float m, c, log2s, a1, b1, at;
  int action;
  bool zero;
  __device__ RowGrad(float g, float h, float entropy, float m_, float c_, float log2s_, float inv_tau, int64_t a, bool empty)
      : m(m_), c(c_), log2s(log2s_), a1((-g - h * entropy) * inv_tau), b1(-h * kLn2 * inv_tau), at(g * inv_tau),
        action(a >= 0 && a < (int64_t{1} << 30) ? (int)a : -1), zero(empty) {}
  // but for what the taken action adds, `at`
  __device__ __forceinline__ float operator()(float x) const {
    const float y = fmaf(x - m, c, -log2s);
    return __builtin_amdgcn_exp2f(y) * fmaf(b1, fmaxf(y, kDeep), a1);
  }
  __device__ __forceinline__ float operator()(float x, int j) const { return (*this)(x) + (j == action ? at : 0.f); }
};

// Keeps the work on one held vector from being mixed with the next one's: where most registers hold the row the
// mixture's do not fit any more.
template <int NV>
__device__ __forceinline__ void apart() {
  if constexpr (NV >= 8) __builtin_amdgcn_sched_barrier(0);
}

template <class E, int LANES, int NV>
struct RowHolder {
  static constexpr int VEC = Frame<E>::VEC;
  static constexpr int EDGES = (2 * VEC + LANES - 1) / LANES;
  u32x4 v[NV];
  float edge[EDGES];

  __device__ __forceinline__ void load(const Frame<E>& f, int lane) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (lane + LANES * k < f.nfull) v[k] = load_words(vector_at<LANES>(f.base + f.head, k, lane));
    }
#pragma unroll
    for (int k = 0; k < EDGES; ++k) {
      const int j = lane + LANES * k < 2 * VEC ? f.edge(lane + LANES * k) : -1;
      edge[k] = j >= 0 ? load_one(f.base + j) : -INFINITY;
    }
  }
  __device__ __forceinline__ RowStats stats(const Frame<E>& f, int lane, float c, float* lds) const {
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < EDGES; ++k) m = fmaxf(m, edge[k]);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (lane + LANES * k < f.nfull) {
        float x[VEC];
        unpack<E>(v[k], x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) m = fmaxf(m, x[i]);
      }
    RowStats r{group_max<LANES>(m, lds), 0.f, 0.f};
    if (r.m == -INFINITY) r.m = 0.f;
#pragma unroll
    for (int k = 0; k < EDGES; ++k) softmax_add((edge[k] - r.m) * c, r.s, r.u);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (lane + LANES * k < f.nfull) {
        float x[VEC];
        unpack<E>(v[k], x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) softmax_add((x[i] - r.m) * c, r.s, r.u);
        apart<NV>();
      }
    group_sum2<LANES>(r.s, r.u, lds + LANES / 64 + 1);
    return r;
  }
};

// A part of a row: its whole vectors v0 .. v1 - 1 and, `edges`, the elements around all of them.
struct Part {
  int v0, v1;
  bool edges;
};

// Writes the gradient of a row, `held` (NV > 0), or of a part of it that is read again.
template <class E, int LANES, int NV>
__device__ __forceinline__ void write_grad(const Frame<E>& f, const RowHolder<E, LANES, NV>* held, E* out, const RowGrad& g,
                                           int lane, const Part& part) {
  constexpr int VEC = Frame<E>::VEC;
  // the output has the input's place in its 16 bytes unless the logits' rows are strided
  const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(f.base)) & 15u) == 0;
  auto vec = [&](u32x4 w, int r) {
    E* to = vector_at<LANES>(out + f.head + part.v0 * VEC, r, lane);
    const int j0 = f.head + (part.v0 + lane + LANES * r) * VEC;
    float x[VEC];
    unpack<E>(w, x);
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = g.zero ? 0.f : g(x[k]);
    if ((uint32_t)(g.action - j0) < (uint32_t)VEC && !g.zero) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] += j0 + k == g.action ? g.at : 0.f;
    }
    if (same) {
      store_words(to, pack<E>(x));
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) to[k] = from_f32<E>(x[k]);
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (lane + LANES * k < f.nfull) {
        vec(held->v[k], k);
        apart<NV>();
      }
  } else {
#pragma unroll 4
    for (int k = 0; part.v0 + lane + LANES * k < part.v1; ++k)
      vec(load_words(vector_at<LANES>(f.base + f.head + part.v0 * VEC, k, lane)), k);
  }
  if (!part.edges) return;
  for (int i = lane; i < 2 * VEC; i += LANES) {
    const int j = f.edge(i);
    if (j >= 0) out[j] = from_f32<E>(g.zero ? 0.f : g(load_one(f.base + j), j));
  }
}

template <class E, int LANES>
__device__ __forceinline__ void write_zeros(E* out, int A, int lane, int part = 0, int parts = 1) {
  const Frame<E> f(out, A);
  for (int i = lane + LANES * part; i < f.nfull; i += LANES * parts) store_words(out + f.head + (int64_t)i * Frame<E>::VEC, u32x4{0, 0, 0, 0});
  if (part > 0) return;
  for (int i = lane; i < 2 * Frame<E>::VEC; i += LANES) {
    const int j = f.edge(i);
    if (j >= 0) out[j] = from_f32<E>(0.f);
  }
}

// Statistics of a row too long to hold, or of a part of it: read once, with a running maximum per lane.
template <class E, int LANES>
__device__ __forceinline__ RowStats streamed_stats(const Frame<E>& f, int lane, float c, float* lds, const Part& part) {
  constexpr int VEC = Frame<E>::VEC;
  float m = -INFINITY, s = 0.f, u = 0.f;
  auto rebase = [&](float to) {  // sums about `to` in place of m
    if (m == to) return;
    if (m != -INFINITY) {  // (else they are 0, or NaN from a NaN)
      const float d = fmaxf((m - to) * c, kDeep), f2 = __builtin_amdgcn_exp2f(d);  // (finite: d s where f2 is 0)
      u = f2 * fmaf(d, s, u);
      s = f2 * s;
    }
    m = to;
  };
  for (int i = lane; part.edges && i < 2 * VEC; i += LANES) {
    const int j = f.edge(i);
    const float x = j >= 0 ? load_one(f.base + j) : -INFINITY;
    if (x != -INFINITY) {
      rebase(fmaxf(m, x));
      softmax_add((x - m) * c, s, u);
    }
  }
#pragma unroll 4
  for (int r = 0; part.v0 + lane + LANES * r < part.v1; ++r) {
    float x[VEC];
    unpack<E>(load_words(vector_at<LANES>(f.base + f.head + part.v0 * VEC, r, lane)), x);
    float t = x[0];
    bool nan = x[0] != x[0];
#pragma unroll
    for (int k = 1; k < VEC; ++k) t = fmaxf(t, x[k]), nan |= x[k] != x[k];
    if (nan) {
      s = NAN;
    } else if (t != -INFINITY) {
      rebase(fmaxf(m, t));
#pragma unroll
      for (int k = 0; k < VEC; ++k) softmax_add((x[k] - m) * c, s, u);
    }
  }
  float top = group_max<LANES>(m, lds);
  if (top != -INFINITY) rebase(top);
  else top = 0.f;
  group_sum2<LANES>(s, u, lds + LANES / 64 + 1);
  return RowStats{top, s, u};
}

// ---------------------------------------------------------------------------------------
// Few rows, and long: each is shared by `parts` workgroups.  A first launch writes the parts' statistics, the second joins
// a row's (a wavefront, in the parts' order) and goes on from there.
// ---------------------------------------------------------------------------------------
struct RowParts {
  int parts;     // 0: rows are not shared
  int per;       // vectors of a part
  float* stats;  // [row, part, 3]: largest logit (-inf: none), s, u
  __device__ Part part(int i, int nfull) const {
    const int v0 = i * per < nfull ? i * per : nfull;
    return {v0, v0 + per < nfull ? v0 + per : nfull, i == 0};
  }
};
constexpr int kMaxShares = 1024, kMaxParts = 64;
static_assert(RLK_ROWS_WORKSPACE_BYTES == sizeof(float) * 3 * kMaxShares, "the workspace of shared rows");

// Shared where a workgroup each would leave most of the GPU idle for longer than a second launch takes (us, alone -> shared).
// Only read: from 12288 vectors (float32: 16 rows of 131072 25.5 -> 11.8, 160 28.2 -> 23.4, 64 of 50001 12.3 -> 11.9; but 10 of 33776
// 8.0 -> 11.4).  Read and written: up to 64 rows from 4096 vectors (bfloat16: 10 of 33776 17.1 -> 13.4, 64 of 50001 19.9 -> 16.8, 16 of
// 131072 32.7 -> 14.7; but 200 of 32768 16.2 -> 24.3, 32 of 8192 9.4 -> 13.9), and up to 256 that are too long to be held (float32: 160 of
// 131072 103 -> 60).
inline RowParts plan_parts(int64_t rows, int64_t vecs, bool written, void* workspace, size_t bytes) {
  RowParts p{0, 0, static_cast<float*>(workspace)};
  if (workspace == nullptr || bytes < sizeof(float) * 3 * kMaxShares || rows < 1 || rows > 256) return p;
  if (written ? vecs < 4096 || (rows > 64 && vecs <= 16384) : vecs < 12288) return p;
  int64_t n = kMaxShares / rows;
  if (n > kMaxParts) n = kMaxParts;
  if (n > vecs / 512) n = vecs / 512;
  p.parts = (int)n, p.per = (int)((vecs + n - 1) / n);
  return p;
}

template <class E>
__global__ __launch_bounds__(256) void part_stats_kernel(const ActionRows<E> a, const RowParts p, const float* __restrict__ mask) {
  __shared__ float lds[3 * 4 + 2];
  const int part = blockIdx.x % p.parts;
  const int64_t row = blockIdx.x / p.parts;
  if (mask != nullptr && mask[row] == 0.f) return;
  const Frame<E> f(row_base(a, row), a.A);
  const RowStats r = streamed_stats<E, 256>(f, threadIdx.x, a.c, lds, p.part(part, f.nfull));
  if (threadIdx.x == 0) {
    float* to = p.stats + 3 * (int64_t)blockIdx.x;
    to[0] = r.s == 0.f ? -INFINITY : r.m, to[1] = r.s, to[2] = r.u;
  }
}

// The row's statistics, in every lane of a wavefront.
__device__ __forceinline__ RowStats join_parts(const RowParts& p, int64_t row, float c) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, s = 0.f, u = 0.f;
  if (lane < p.parts) {
    const float* from = p.stats + 3 * (row * p.parts + lane);
    m = from[0], s = from[1], u = from[2];
  }
  float top = group_max<64>(m, nullptr);
  if (top == -INFINITY) top = 0.f;
  const float d = fmaxf((m - top) * c, kDeep), f = __builtin_amdgcn_exp2f(d);
  u = f * fmaf(d, s, u), s = f * s;
  group_sum2<64>(s, u, nullptr);
  return RowStats{top, s, u};
}

// ---------------------------------------------------------------------------------------
// Few actions, rows one after the other in memory: a thread per row.  A workgroup takes 256 rows in 16-byte
// accesses through LDS, which holds them as they are in memory: a lane reads its row in the widest words that divide it (4,
// 8 or 16 bytes), whose places in a wavefront's rows lie in different banks; for rows of a multiple of 32 bytes 16
// more keep them apart.  No lane is idle past the row's end, nothing is reduced over lanes, and what a
// step computes beside its logits it computes once.
// ---------------------------------------------------------------------------------------
constexpr int kFewActions = 32, kFewRows = 256;

struct FewRows {
  int A, pitch;    // pitch: A, or A + 4 for a multiple of 8
  uint32_t magic;  // ceil(2^32 / A): i / A = umulhi(i, magic) for i < 2^13 (A > 1)
  bool quads;      // the arrays are aligned to 4 elements
  static constexpr size_t bytes(int pitch) { return (size_t)pitch * kFewRows * sizeof(float); }
  // where element i of the rows lies
  __device__ int place(int i) const { return pitch == A ? i : i + 4 * (int)__umulhi((uint32_t)i, magic); }

  // LDS <- `count` elements at `src`
  template <class E>
  __device__ void take(const E* src, int count, float* lds) const {
    const int whole = quads ? count / 4 : 0;
    for (int q = threadIdx.x; q < whole; q += kFewRows) *reinterpret_cast<float4*>(lds + place(4 * q)) = load_quad<true>(src + 4 * q);
    for (int i = 4 * whole + threadIdx.x; i < count; i += kFewRows) lds[place(i)] = load_one(src + i);
  }
  template <class E>
  __device__ void put(E* dst, int count, const float* lds) const {
    const int whole = quads ? count / 4 : 0;
    for (int q = threadIdx.x; q < whole; q += kFewRows) store_quad<true>(dst + 4 * q, *reinterpret_cast<const float4*>(lds + place(4 * q)));
    for (int i = 4 * whole + threadIdx.x; i < count; i += kFewRows) dst[i] = from_f32<E>(lds[place(i)]);
  }
};

// A thread's row: K >= A logits, -inf beyond A.
template <int K>
struct FewLogits {
  float x[K];
  // f(first element, vector type) for each of the widest words that divide the row, K of 4 at the most
  template <class F>
  __device__ __forceinline__ static void words(int A, F f) {
    if ((A & 3) == 0) {
#pragma unroll
      for (int j = 0; j < K; j += 4) f(j, float4{});
    } else if ((A & 1) == 0) {
#pragma unroll
      for (int j = 0; j < K; j += 2)
        if (j < K - 2) f(j, float2{});
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (j < K - 3 || j < A) f(j, 0.f);
    }
  }
  __device__ __forceinline__ void load(const float* row, int A) {
#pragma unroll
    for (int j = K - 3; j < K; ++j) x[j] = -INFINITY;
    words(A, [&](int j, auto word) {
      word = *reinterpret_cast<const decltype(word)*>(row + j);
      const float* e = reinterpret_cast<const float*>(&word);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(word) / 4); ++i) x[j + i] = e[i];
    });
  }
  __device__ __forceinline__ void store(float* row, int A) const {
    words(A, [&](int j, auto word) {
      float* e = reinterpret_cast<float*>(&word);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(word) / 4); ++i) e[i] = x[j + i];
      *reinterpret_cast<decltype(word)*>(row + j) = word;
    });
  }
  __device__ __forceinline__ RowStats stats(float c) const {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < K; ++j) m = fmaxf(m, x[j]);
    RowStats r{m == -INFINITY ? 0.f : m, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < K; ++j) softmax_add((x[j] - r.m) * c, r.s, r.u);
    return r;
  }
};

// Calls f(integral constant K) with the multiple of 4 that holds A.
template <class F>
int dispatch_few(int A, F f) {
  switch ((A + 3) / 4) {
    case 1: return f(std::integral_constant<int, 4>{});
    case 2: return f(std::integral_constant<int, 8>{});
    case 3: return f(std::integral_constant<int, 12>{});
    case 4: return f(std::integral_constant<int, 16>{});
    case 5: return f(std::integral_constant<int, 20>{});
    case 6: return f(std::integral_constant<int, 24>{});
    case 7: return f(std::integral_constant<int, 28>{});
    default: return f(std::integral_constant<int, 32>{});
  }
}

template <class E>
bool few_rows(const ActionRows<E>& a, const void* out, FewRows* f) {
  if (a.A > kFewActions || a.step_stride != a.A || a.env_stride != a.seq_len * a.step_stride) return false;
  const uintptr_t low = (reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(out)) & (4 * sizeof(E) - 1);
  *f = {a.A, a.A % 8 == 0 ? a.A + 4 : a.A, (uint32_t)(((uint64_t{1} << 32) + (uint32_t)a.A - 1) / (uint32_t)a.A), low == 0};
  return true;
}

template <int LANES>
constexpr int rows_threads() { return LANES > 256 ? LANES : 256; }

// Calls f(integral constants LANES, NV, most workgroups) for `rows` rows of `vecs` 16-byte vectors.
//
// Rows of up to 256 vectors are held by as few lanes as hold them in four vectors each (two in the shortest): whole
// wavefronts' lanes are busy and what is computed once a row is repeated in few lanes (float32, 84 MB read: 40 actions 25.7 us with 8 lanes,
// 37.6 with 16; 128: 13.8 with 8, 17.2 with 16; 511: 14.3 with 32, 17.8 with 64).  Longer ones:
//  - only read (log-probabilities): streamed (NV = 0), a workgroup per row, many small workgroups so that one loads while
//    another reduces; wider ones where there are too few rows for that.  16384 rows of 32768 bfloat16: 256 lanes 183 us,
//    512 199, 1024 233, held by 1024 lanes 284; a round of 256 rows of 65536: 9.3 us with 1024 lanes, 13 with 512, 22 with 256.
//  - read and written (losses): held, in the fewest lanes whose registers leave room for a second workgroup per CU
//    (4096 vectors: 512 lanes 313 us, 256 lanes 351, 1024 lanes 380; 1000 vectors: 256 lanes 355, 512 420, 1024 727); rows of
//    more than 256 KB are read twice.
template <class F>
int dispatch_short(int64_t vecs, F f) {
  using std::integral_constant;
  if (vecs <= 8) return f(integral_constant<int, 4>{}, integral_constant<int, 2>{}, 2048);
  if (vecs <= 16) return f(integral_constant<int, 8>{}, integral_constant<int, 2>{}, 2048);
  if (vecs <= 32) return f(integral_constant<int, 8>{}, integral_constant<int, 4>{}, 2048);
  if (vecs <= 64) return f(integral_constant<int, 16>{}, integral_constant<int, 4>{}, 2048);
  if (vecs <= 128) return f(integral_constant<int, 32>{}, integral_constant<int, 4>{}, 2048);
  if (vecs <= 256) return f(integral_constant<int, 64>{}, integral_constant<int, 4>{}, 2048);
  return f(integral_constant<int, 256>{}, integral_constant<int, 2>{}, 2048);
}
template <class F>
int dispatch_read(int64_t vecs, int64_t rows, F f) {
  using std::integral_constant;
  if (vecs <= 512) return dispatch_short(vecs, f);
  const int64_t many = int64_t{1} << 22;
  if (rows < 512) return f(integral_constant<int, 1024>{}, integral_constant<int, 0>{}, many);
  if (rows < 1024) return f(integral_constant<int, 512>{}, integral_constant<int, 0>{}, many);
  return f(integral_constant<int, 256>{}, integral_constant<int, 0>{}, many);
}
template <class F>
int dispatch_update(int64_t vecs, F f) {
  using std::integral_constant;
  if (vecs <= 512) return dispatch_short(vecs, f);
  if (vecs <= 1024) return f(integral_constant<int, 256>{}, integral_constant<int, 4>{}, 2048);
  if (vecs <= 2048) return f(integral_constant<int, 256>{}, integral_constant<int, 8>{}, 2048);
  if (vecs <= 4096) return f(integral_constant<int, 512>{}, integral_constant<int, 8>{}, 2048);
  if (vecs <= 8192) return f(integral_constant<int, 1024>{}, integral_constant<int, 8>{}, 1024);
  if (vecs <= 16384) return f(integral_constant<int, 1024>{}, integral_constant<int, 16>{}, 1024);
  return f(integral_constant<int, 512>{}, integral_constant<int, 0>{}, 2048);
}

inline bool valid_rows(const rlk_action_rows* r) {
  if (!r || r->num_envs < 0 || r->seq_len < 0 || r->num_actions < 1 || r->num_actions > (int64_t{1} << 30)) return false;
  if (!(r->temperature >= RLK_LEAST_TEMPERATURE && r->temperature <= RLK_LARGEST_TEMPERATURE)) return false;
  return r->num_envs * r->seq_len == 0 || (r->logits && r->actions && (reinterpret_cast<uintptr_t>(r->logits) & (r->bf16 ? 1u : 3u)) == 0);
}

template <class E>
ActionRows<E> action_rows(const rlk_action_rows* r) {
  const double inv = 1.0 / r->temperature;
  return {static_cast<const E*>(r->logits), r->actions, r->num_envs * r->seq_len, r->seq_len, r->env_stride, r->step_stride,
          (int)r->num_actions, (float)(1.4426950408889634 * inv), (float)inv};
}

}  // namespace rlk
