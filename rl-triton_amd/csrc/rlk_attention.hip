// rlk_attention.hip -- linear attention with a decay for each head and episode ends, whole sequences
// (include/rl_triton_policy.h).
//
// One kernel computes, in walk order s = 0 .. T-1 (from the last step to the first where `reverse`),
//   S_s = lambda (1 - cut_s) S_{s-1} + b_s c_s^T,   y_s = scale S_s^T a_s
// with (a, b, c) = (q, k, v) for the outputs, and for the gradients of an upstream dy: (dy, v, k) forward for
// dq, and in reverse (v, dy, q) for dk and (k, q, dy) for dv.
//
// Chunks of C = 64 steps (one per lane of a wavefront: a chunk's cuts are one ballot).  With U the state that
// enters the chunk, already decayed by its first step, row i of the chunk and
// same(j, i) = no cut in (j, i]:
//   y_i = scale (lambda^i [no cut in [0, i]] U^T a_i + sum_{j <= i} lambda^{i-j} same(j, i) (a_i . b_j) c_j)
//   U'  = lambda^L [no cut in the chunk] U + sum_j lambda^{L-j} same(j, L-1) b_j c_j^T
// Every factor is a power with an exponent >= 0 (no quotient of powers, which would leave float's range).
//
// A workgroup of 4 wavefronts walks the chunks of its (environment, head, segment); wavefront w owns a quarter of
// the columns of c.  Its part of U stays in the accumulators of the matrix instructions for the whole walk: the
// accumulator layout (4 consecutive rows of a column per lane) is also an operand layout once the inner index is
// taken in that order, so U feeds U^T a without a trip through LDS.
#include "rlk_attention.hpp"

namespace rlk {
namespace {

constexpr int C = 64;       // steps per chunk
constexpr int kNT = 256;    // 4 wavefronts

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 8 consecutive (in the inner index) elements of an operand row: the unit of a matrix instruction's operands.
template <class E>
struct Frag;
template <>
struct Frag<bf16> {
  bf16x8 x;
  __device__ static Frag load(const bf16* p) { return {*reinterpret_cast<const bf16x8*>(p)}; }
  __device__ static Frag load2(const bf16* p, const bf16* q) {
    union { u32x2 h[2]; bf16x8 v; } u;
    u.h[0] = *reinterpret_cast<const u32x2*>(p), u.h[1] = *reinterpret_cast<const u32x2*>(q);
    return {u.v};
  }
  __device__ static Frag from(f32x4 a, f32x4 b) {
    union { uint32_t w[4]; bf16x8 v; } u;
    u.w[0] = pack_bf16x2(a[0], a[1]), u.w[1] = pack_bf16x2(a[2], a[3]);
    u.w[2] = pack_bf16x2(b[0], b[1]), u.w[3] = pack_bf16x2(b[2], b[3]);
    return {u.v};
  }
};
template <>
struct Frag<float> {
  f32x4 lo, hi;
  __device__ static Frag load(const float* p) { return load2(p, p + 4); }
  __device__ static Frag load2(const float* p, const float* q) {
    return {*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(q)};
  }
  __device__ static Frag from(f32x4 a, f32x4 b) { return {a, b}; }
};

// acc[m][n] += sum over 32 inner indices: lane l holds row/column l % 16 and inner indices of its quarter l / 16
// (8 of them; which 8 is the same for both operands, so their order does not matter).  The result's lane l holds
// column l % 16, rows 4 (l / 16) + 0..3.
__device__ __forceinline__ f32x4 mma(const Frag<bf16>& a, const Frag<bf16>& b, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.x, b.x, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Frag<float>& a, const Frag<float>& b, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[i], b.lo[i], acc, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[i], b.hi[i], acc, 0, 0, 0);
  return acc;
}

// 4 consecutive elements.
template <class E>
struct Quad;
template <>
struct Quad<bf16> {
  u32x2 w;
  __device__ float get(int i) const { return Words<bf16>::get(w[i >> 1], i & 1); }
  __device__ static Quad of(float a, float b, float c, float d) { return {{pack_bf16x2(a, b), pack_bf16x2(c, d)}}; }
  __device__ static Quad load(const bf16* p) { return {*reinterpret_cast<const u32x2*>(p)}; }
  __device__ void store(bf16* p) const { *reinterpret_cast<u32x2*>(p) = w; }
};
template <>
struct Quad<float> {
  f32x4 w;
  __device__ float get(int i) const { return w[i]; }
  __device__ static Quad of(float a, float b, float c, float d) { return {{a, b, c, d}}; }
  __device__ static Quad load(const float* p) { return {*reinterpret_cast<const f32x4*>(p)}; }
  __device__ void store(float* p) const { *reinterpret_cast<f32x4*>(p) = w; }
};

// x^n for n >= 0 from log2 x (x = 0: 1, 0, 0, ...).
__device__ __forceinline__ float power(float log2x, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(log2x * (float)n); }

template <class E, int D>
struct Tiles {
  static constexpr int PAD = 16 / (int)sizeof(E);
  E a[C][D + PAD];    // rows of a chunk
  E b[C][D + PAD];
  E bt[D][C + PAD];   // b transposed
  E ct[D][C + PAD];   // c transposed
  E p[C][C + PAD];    // (a_i . b_j) lambda^{i-j} same(j, i)
};

// One array's part of a chunk, held by a thread: R rows of 4 columns.
template <class E, int D>
struct Part {
  static constexpr int GROUPS = D / 4, R = C * GROUPS / kNT;
  Quad<E> x[R];
};

template <class E, int D, bool VEC>
__device__ __forceinline__ void fetch(Part<E, D>& part, const E* base, int64_t step_stride, int dim, int64_t first, int count,
                                      int64_t T, bool reverse) {
  constexpr int R = Part<E, D>::R;
  const int col = (threadIdx.x % Part<E, D>::GROUPS) * 4, row0 = (threadIdx.x / Part<E, D>::GROUPS) * R;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = row0 + r;
    part.x[r] = Quad<E>::of(0.f, 0.f, 0.f, 0.f);
    if (i < count && col < dim) {
      const int64_t t = reverse ? T - 1 - (first + i) : first + i;
      const E* p = base + t * step_stride + col;
      if constexpr (VEC) {
        part.x[r] = Quad<E>::load(p);
      } else {
        part.x[r] = Quad<E>::of(load_one(p), col + 1 < dim ? load_one(p + 1) : 0.f, col + 2 < dim ? load_one(p + 2) : 0.f,
                                col + 3 < dim ? load_one(p + 3) : 0.f);
      }
    }
  }
}

// Puts the R x 4 part down as 4 rows of R consecutive elements.
template <class E, int D>
__device__ __forceinline__ void put_transposed(const Part<E, D>& part, E (*dst)[C + Tiles<E, D>::PAD]) {
  constexpr int R = Part<E, D>::R;
  const int col = (threadIdx.x % Part<E, D>::GROUPS) * 4, row0 = (threadIdx.x / Part<E, D>::GROUPS) * R;
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int r = 0; r < R; r += 4)
      Quad<E>::of(part.x[r].get(x), part.x[r + 1].get(x), part.x[r + 2].get(x), part.x[r + 3].get(x)).store(&dst[col + x][row0 + r]);
}

// acc += a (w * c) for an operand row c and weights w of its inner indices.  The weighted bfloat16 operand is
// taken as the sum of two bfloat16 numbers (the product's upper 8 bits and the next 8): the state is a float32
// result and sums over all steps, and one rounding of every term to 8 bits would be 2^-9 of it.
template <class E>
struct Weighted;
template <>
struct Weighted<float> {
  Frag<float> x;
  __device__ Weighted(const Frag<float>& c, const float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.lo[i] = c.lo[i] * w[i], x.hi[i] = c.hi[i] * w[4 + i];
  }
  __device__ f32x4 mma_with(const Frag<float>& a, f32x4 acc) const { return mma(a, x, acc); }
};
template <>
struct Weighted<bf16> {
  Frag<bf16> hi, lo;
  __device__ Weighted(const Frag<bf16>& c, const float (&w)[8]) {
    union { bf16x8 v; uint32_t u[4]; } in{c.x}, h, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = Words<bf16>::get(in.u[i], 0) * w[2 * i], b = Words<bf16>::get(in.u[i], 1) * w[2 * i + 1];
      h.u[i] = pack_bf16x2(a, b);
      l.u[i] = pack_bf16x2(a - Words<bf16>::get(h.u[i], 0), b - Words<bf16>::get(h.u[i], 1));
    }
    hi.x = h.v, lo.x = l.v;
  }
  __device__ f32x4 mma_with(const Frag<bf16>& a, f32x4 acc) const { return mma(a, hi, mma(a, lo, acc)); }
};

// The walk over a segment.  STATE: only the state at its end, from zero, for the segments after it.
template <class E, int D, bool VEC, bool STATE>
__global__ __launch_bounds__(kNT) void walk_kernel(const Walks<E> walks) {
  __shared__ __align__(16) Tiles<E, D> tiles;
  constexpr int MT = D / 16, NT = D / 64;  // tiles of 16: rows of the state; this wavefront's columns
  const Walk<E>& w = walks.w[blockIdx.z];
  const int head = blockIdx.x % walks.heads, seg = blockIdx.y;
  const int64_t env = blockIdx.x / walks.heads, T = walks.seq_len;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, l4 = lane >> 4;
  const int n0 = wave * (D / 4);  // this wavefront's columns
  const int64_t first = (int64_t)seg * walks.seg_len, last = first + walks.seg_len < T ? first + walks.seg_len : T;
  const float lambda = walks.decay[head], lg = __log2f(lambda);
  const float* dones = walks.dones ? walks.dones + env * T : nullptr;
  const E* ga = w.a.data + env * w.a.env_stride + head * w.a.head_stride;
  const E* gb = w.b.data + env * w.b.env_stride + head * w.b.head_stride;
  const E* gc = w.c.data + env * w.c.env_stride + head * w.c.head_stride;
  const bool reverse = w.reverse;

  // U[da][dc]: lane holds column n0 + 16 n + l16, rows 16 m + 4 l4 + 0..3
  f32x4 U[MT][NT];
  const int64_t eh = env * walks.heads + head;
  if (!STATE && seg > 0) {
    const float* p = w.seg_states + (eh * walks.segs + seg) * (int64_t)(w.da * w.dc);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * m + 4 * l4 + r, j = n0 + 16 * n + l16;
          U[m][n][r] = i < w.da && j < w.dc ? p[i * w.dc + j] : 0.f;
        }
  } else {
    const float f = reverse ? w.state_scale : w.state_scale * lambda;
    const float* p = STATE || w.state == nullptr ? nullptr : w.state + eh * (int64_t)(w.da * w.dc);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * m + 4 * l4 + r, j = n0 + 16 * n + l16;
          U[m][n][r] = p != nullptr && i < w.da && j < w.dc ? p[w.transposed ? j * w.da + i : i * w.dc + j] * f : 0.f;
        }
  }

  // lambda^{i-j}, j <= i, of this lane's elements of p (computed transposed: row j, column i): i = 16 wave + l16
  f32x4 among[4];
#pragma unroll
  for (int jt = 0; jt < 4; ++jt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * wave + l16 - (16 * jt + 4 * l4 + r);
      among[jt][r] = d < 0 ? 0.f : power(lg, d);
    }
  float back[4];  // lambda^i of the output rows i = 16 t + l16
#pragma unroll
  for (int t = 0; t < 4; ++t) back[t] = power(lg, 16 * t + l16);

  Part<E, D> pa, pb, pc;
  uint64_t cuts, next_cuts = 0;
  auto fetch_all = [&](int64_t s0) {
    const int count = (int)(last - s0 < C ? last - s0 : C);
    if (!STATE) fetch<E, D, VEC>(pa, ga, w.a.step_stride, w.da, s0, count, T, reverse);
    fetch<E, D, VEC>(pb, gb, w.b.step_stride, w.da, s0, count, T, reverse);
    fetch<E, D, VEC>(pc, gc, w.c.step_stride, w.dc, s0, count, T, reverse);
    bool cut = false;
    if (dones != nullptr && lane < count) {
      const int64_t s = s0 + lane;
      if (reverse) cut = dones[T - 1 - s] != 0.f;
      else cut = s > 0 && dones[s - 1] != 0.f;
    }
    next_cuts = __ballot(cut);
  };
  fetch_all(first);

  bool crossed = false;  // a cut anywhere in the segment
  for (int64_t s0 = first; s0 < last; s0 += C) {
    const int L = (int)(last - s0 < C ? last - s0 : C);
    cuts = next_cuts;
    crossed |= cuts != 0;
    // the state that leaves the sequence forward is the one after the last step, not decayed by another
    const bool end = !reverse && s0 + C >= T;
    const int reach = end ? L - 1 : L;
    __syncthreads();  // the chunk before has been read
    {
      constexpr int R = Part<E, D>::R;
      const int col = (tid % Part<E, D>::GROUPS) * 4, row0 = (tid / Part<E, D>::GROUPS) * R;
      if constexpr (!STATE) {
#pragma unroll
        for (int r = 0; r < R; ++r) pa.x[r].store(&tiles.a[row0 + r][col]), pb.x[r].store(&tiles.b[row0 + r][col]);
      }
      put_transposed<E, D>(pc, tiles.ct);
      put_transposed<E, D>(pb, tiles.bt);
    }
    __syncthreads();
    if (s0 + C < last) fetch_all(s0 + C);  // in flight while this chunk is worked on

    if constexpr (!STATE) {
      // p^T: rows j, columns i = 16 wave + l16
      f32x4 pt[4];
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) pt[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
        const Frag<E> fa = Frag<E>::load(&tiles.a[16 * wave + l16][32 * kk + 8 * l4]);
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
          if (jt <= wave) pt[jt] = mma(Frag<E>::load(&tiles.b[16 * jt + l16][32 * kk + 8 * l4]), fa, pt[jt]);
      }
      const int i = 16 * wave + l16;
      // cuts before or at step i: two steps belong together when these numbers are the same
      const int ep_i = __popcll(cuts & ((uint64_t)2 << i) - 1);
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * jt + 4 * l4 + r;
          const bool same = cuts == 0 || __popcll(cuts & ((uint64_t)2 << j) - 1) == ep_i;
          x[r] = j <= i && same ? pt[jt][r] * among[jt][r] : 0.f;
        }
        Quad<E>::of(x[0], x[1], x[2], x[3]).store(&tiles.p[i][16 * jt + 4 * l4]);
      }
      __syncthreads();

      // y^T: rows = this wavefront's columns of c, columns i = 16 t + l16
      f32x4 y[4][NT];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) y[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
        Frag<E> fu[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) fu[n] = Frag<E>::from(U[2 * kk][n], U[2 * kk + 1][n]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const E* row = &tiles.a[16 * t + l16][32 * kk + 4 * l4];
          const Frag<E> fa = Frag<E>::load2(row, row + 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) y[t][n] = mma(fu[n], fa, y[t][n]);
        }
      }
      const int until = cuts == 0 ? C : __ffsll((long long)cuts) - 1;  // the first step that the state does not reach
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float f = 16 * t + l16 < until ? back[t] : 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) y[t][n][r] = f == 0.f ? 0.f : y[t][n][r] * f;
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        Frag<E> fc[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) fc[n] = Frag<E>::load(&tiles.ct[n0 + 16 * n + l16][32 * kk + 8 * l4]);
#pragma unroll
        for (int t = 2 * kk; t < 4; ++t) {  // (rows before the steps 32 kk + 0..31 have none of them)
          const Frag<E> fp = Frag<E>::load(&tiles.p[16 * t + l16][32 * kk + 8 * l4]);
#pragma unroll
          for (int n = 0; n < NT; ++n) y[t][n] = mma(fc[n], fp, y[t][n]);
        }
      }
      E* gy = w.y.data + env * w.y.env_stride + head * w.y.head_stride;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int row = 16 * t + l16;
        if (row < L) {
          const int64_t at = reverse ? T - 1 - (s0 + row) : s0 + row;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int j = n0 + 16 * n + 4 * l4;
            E* p = gy + at * w.y.step_stride + j;
            const f32x4 v = y[t][n] * w.scale;
            if (VEC) {
              if (j < w.dc) Quad<E>::of(v[0], v[1], v[2], v[3]).store(p);
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (j + r < w.dc) p[r] = from_f32<E>(v[r]);
            }
          }
        }
      }
    }

    // U' = lambda^reach U + sum over steps from the last cut on of lambda^{reach-j} b_j c_j^T
    const float keep = cuts == 0 ? power(lg, reach) : 0.f;
    const int from = cuts == 0 ? 0 : 63 - __clzll((long long)cuts);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) U[m][n][r] = keep == 0.f ? 0.f : U[m][n][r] * keep;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      float f[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int j = 32 * kk + 8 * l4 + x;
        f[x] = j >= from && j < L ? power(lg, reach - j) : 0.f;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const Weighted<E> fc(Frag<E>::load(&tiles.ct[n0 + 16 * n + l16][32 * kk + 8 * l4]), f);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          U[m][n] = fc.mma_with(Frag<E>::load(&tiles.bt[16 * m + l16][32 * kk + 8 * l4]), U[m][n]);
      }
    }
  }

  float* out = nullptr;
  float f = 1.f;
  if (STATE) {
    out = w.seg_states + (eh * walks.segs + seg + 1) * (int64_t)(w.da * w.dc);
    if (tid == 0) w.seg_keep[eh * walks.segs + seg + 1] = crossed ? 0.f : power(lg, (int)(last - first));
  } else if (last == T && w.state_out != nullptr) {
    out = w.state_out + eh * (int64_t)(w.da * w.dc);
    f = !reverse && dones != nullptr && dones[T - 1] != 0.f ? 0.f : w.state_out_scale;
  }
  if (out != nullptr)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * m + 4 * l4 + r, j = n0 + 16 * n + l16;
          if (i < w.da && j < w.dc) out[i * w.dc + j] = f == 0.f ? 0.f : U[m][n][r] * f;
        }
}

// The states that enter the segments: in place, from what each segment added and how much of what enters it leaves.
template <class E>
__global__ __launch_bounds__(kNT) void join_kernel(const Walks<E> walks) {
  const Walk<E>& w = walks.w[blockIdx.z];
  const int n = w.da * w.dc;
  const int64_t eh = blockIdx.x;
  const int i = blockIdx.y * kNT + threadIdx.x;
  if (i >= n) return;
  float u = 0.f;
  if (w.state != nullptr) {
    const int64_t at = w.transposed ? (int64_t)(i % w.dc) * w.da + i / w.dc : i;
    u = w.state[eh * n + at] * (w.reverse ? w.state_scale : w.state_scale * walks.decay[eh % walks.heads]);
  }
  for (int s = 1; s < walks.segs; ++s) {
    float* p = w.seg_states + (eh * walks.segs + s) * (int64_t)n + i;
    const float keep = w.seg_keep[eh * walks.segs + s];
    u = keep == 0.f ? *p : fmaf(u, keep, *p);
    *p = u;
  }
}

template <class E, int D, bool VEC>
int launch_walks(const Walks<E>& k, int count, hipStream_t s) {
  const dim3 grid((unsigned)(k.num_envs * k.heads), (unsigned)k.segs, (unsigned)count);
  if (k.segs > 1) {
    dim3 g = grid;
    g.y = (unsigned)k.segs - 1;
    walk_kernel<E, D, VEC, true><<<g, dim3(kNT), 0, s>>>(k);
    if (hipGetLastError() != hipSuccess) return RLK_ERR_LAUNCH;
    int most = 0;
    for (int i = 0; i < count; ++i) most = most < k.w[i].da * k.w[i].dc ? k.w[i].da * k.w[i].dc : most;
    join_kernel<E><<<dim3(grid.x, (unsigned)(most + kNT - 1) / kNT, (unsigned)count), dim3(kNT), 0, s>>>(k);
    if (hipGetLastError() != hipSuccess) return RLK_ERR_LAUNCH;
  }
  walk_kernel<E, D, VEC, false><<<grid, dim3(kNT), 0, s>>>(k);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

template <class E>
bool quads(const Sequence<E>& x, int dim) {
  return dim % 4 == 0 && (reinterpret_cast<uintptr_t>(x.data) % (4 * sizeof(E))) == 0 && x.env_stride % 4 == 0 &&
         x.step_stride % 4 == 0 && x.head_stride % 4 == 0;
}

template <class E>
int walk_impl(const rlk_attention* c, int count, hipStream_t s) {
  Walks<E> k = {};
  k.num_envs = c->num_envs, k.seq_len = c->seq_len, k.heads = (int)c->heads, k.decay = c->decay, k.dones = c->dones;
  const SegmentPlan plan = plan_segments(c->num_envs * c->heads, c->seq_len);
  k.segs = plan.segs, k.seg_len = plan.seg_len;
  bool vec = true, small = true;
  char* ws = static_cast<char*>(c->workspace);
  size_t left = c->workspace_bytes;
  for (int i = 0; i < count; ++i) {
    const rlk_attention& q = c[i];
    Walk<E>& w = k.w[i];
    w.a = sequence<const E>(q.q), w.b = sequence<const E>(q.k), w.c = sequence<const E>(q.v), w.y = sequence<E>(q.out);
    w.da = (int)q.dim_k, w.dc = (int)q.dim_v;
    w.state = q.state, w.transposed = q.state_transposed, w.state_out = q.state_out;
    w.scale = q.scale, w.state_scale = q.state_scale, w.state_out_scale = q.state_out_scale, w.reverse = q.reverse;
    vec = vec && quads(w.a, w.da) && quads(w.b, w.da) && quads(w.c, w.dc) && quads(w.y, w.dc);
    small = small && w.da <= 64 && w.dc <= 64;
    if (k.segs > 1) {
      const size_t states = (size_t)k.num_envs * k.heads * k.segs * w.da * w.dc, keeps = (size_t)k.num_envs * k.heads * k.segs;
      if ((states + keeps) * sizeof(float) > left || ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 3u) != 0)
        return RLK_ERR_WORKSPACE;
      w.seg_states = reinterpret_cast<float*>(ws), w.seg_keep = w.seg_states + states;
      ws += (states + keeps) * sizeof(float), left -= (states + keeps) * sizeof(float);
    }
  }
  if (small) return vec ? launch_walks<E, 64, true>(k, count, s) : launch_walks<E, 64, false>(k, count, s);
  return vec ? launch_walks<E, 128, true>(k, count, s) : launch_walks<E, 128, false>(k, count, s);
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" {

size_t rlk_attention_workspace_bytes(int64_t num_envs, int64_t seq_len, int64_t heads, int64_t dim_k, int64_t dim_v) {
  if (num_envs <= 0 || seq_len <= 0 || heads <= 0 || dim_k <= 0 || dim_v <= 0) return 0;
  const SegmentPlan plan = plan_segments(num_envs * heads, seq_len);
  return plan.segs <= 1 ? 0 : (size_t)num_envs * heads * plan.segs * (dim_k * dim_v + 1) * sizeof(float);
}

int rlk_linear_attention(const rlk_attention* calls, int count, void* stream) {
  if (!calls || count < 1 || count > 3) return RLK_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < count; ++i) {
    const rlk_attention& c = calls[i];
    if (!valid_attention(c) || c.seq_len < 0 || c.num_envs != calls->num_envs || c.seq_len != calls->seq_len ||
        c.heads != calls->heads || c.decay != calls->decay || c.dones != calls->dones || c.bf16 != calls->bf16)
      return RLK_ERR_INVALID_ARGUMENT;
  }
  if (calls->num_envs == 0 || calls->heads == 0 || calls->seq_len == 0) return RLK_OK;
  if (calls->num_envs * calls->heads > kMaxGrid || calls->seq_len > (int64_t{1} << 30)) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return calls->bf16 ? walk_impl<bf16>(calls, count, s) : walk_impl<float>(calls, count, s);
}

}  // extern "C"
