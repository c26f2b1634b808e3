// rlk_delta.hpp -- the gated delta rule (include/rl_triton_policy.h): its mathematics by chunks of steps, and what its kernels share.
//
//   S_t = a_t S_{t-1} + k_t u_t^T,   u_t = b_t (v_t - a_t S_{t-1}^T k_t),   y_t = scale S_t^T q_t,
// with a_t = exp(g_t), 0 where an episode begins.  In a chunk of C = 64 steps, S the state before it and
//   D_ij = a_{j+1} .. a_i (i >= j; 0 where an episode begins in between),  back_i = a_0 .. a_i,  into_j = D_{C-1,j},  keep = back_{C-1},
// e_i = v_i - back_i S^T k_i is what a step would correct if none of the chunk came before it, and with L_ij = D_ij k_i . k_j (i > j) the steps'
// corrections w (u = b w) solve w = e - L (b w).  M = (1 + L b)^-1 L = L (1 + b L)^-1 depends on keys and gates only, and
//   w = e - M (b e),   y_i = scale (back_i S^T q_i + sum_{j <= i} D_ij (q_i . k_j) u_j),   S' = keep S + sum_j into_j k_j u_j^T.
// The same M serves the way back: with P_ij = scale D_ij q_i . k_j, G the outputs' gradients and R that of S',
//   du = P^T G + into k R,   z = du - M^T (b du),   dv = b z,   dS = keep R + sum_i scale back_i q_i G_i^T - back_i k_i dv_i^T
// (z is the gradient of u once the later steps' corrections have had their part; that of b is z . w).
//
// So a launch with a wavefront per (environment, head, chunk) forms the records (M, the products of gates), and a walk over the chunks
// keeps 16 columns of the state per wavefront in the accumulators of the matrix instructions, with three products after each other in a chunk.
//
// Numbers: every factor that is not one of the call's bfloat16 arrays is taken as three bfloat16 numbers, 8 bits each, which is the whole
// float; of the products of two such the ones below 2^-24 are left out.  float32 arrays are split in the same way: six bfloat16 products in
// place of one float32 product at a sixteenth of the rate.  So states, w, z, gradients and outputs are float32 results; a bfloat16 one is rounded once.
// (Outputs from factors of two numbers, 2^-16 off, were the neighbour of the rounded one in some 0.5% of cases, for 2 to 3% of a forward pass's time.)
#pragma once
#include "rlk_launch.hpp"
#include "rlk_policy.hpp"

namespace rlk {
namespace delta {

constexpr int C = 64;
constexpr float kNoDecay = -104.f;  // gates below: exp is 0 in float32, and nothing of the state stays

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class E>
constexpr int kParts = sizeof(E) == 2 ? 1 : 3;

// A record of a chunk, written by records_kernel.  M's tiles (ti, tj), tj <= ti, at ti (ti + 1) / 2 + tj, row-major; D_ij = exp((ghi_i -
// ghi_j) + (glo_i - glo_j)), the upper ones multiples of 2^-10, so that their difference is exact.
struct Record {
  float tiles[10][256];
  float ghi[C], glo[C], back[C], into[C], beta[C];
  float keep;
  uint32_t cuts[2];  // steps that begin an episode, or that keep nothing
  uint32_t wild;     // something is not finite: the chunk is walked step by step
};
static_assert(sizeof(Record) % 16 == 0);

template <class E>
struct Seq {
  E* data;
  int64_t env, step, head;
};
template <class E>
Seq<E> seq(const rlk_sequence& x) {
  return {static_cast<E*>(const_cast<void*>(x.data)), x.env_stride, x.step_stride, x.head_stride};
}

// Dims padded to whole tiles, as the workspace's arrays are laid out.
__host__ __device__ inline int pad16(int d) { return (d + 15) / 16 * 16; }

template <class E>
struct Rule {
  Seq<const E> q, k, v;
  Seq<E> y;
  Seq<const E> gy;          // backward: the outputs' gradients ...
  Seq<E> gq, gk, gv;        // ... and the inputs'
  int64_t seq_len, chunks;  // of a sequence
  int64_t first_env;        // of this launch
  int heads, dk, dv;
  const float *gates, *betas, *dones;  // [env, step, head], [env, step]
  const float* state;
  float* state_out;
  float scale;
  Record* records;  // [pair of this launch, chunk]
  // training, [pair, chunk]: states before the chunk [pad16(dk), pad16(dv)] and w [C, pad16(dv)]; backward: gradients of the states after
  // it, and z.  NULL: not kept.
  float *states, *w, *dstates, *z;
  float *gg, *gb;  // gradients of gates and betas
  // Sequences cut into segments of seg_chunks chunks, where there are few pairs.  A segment turns the state S that enters it into phi S + n:
  // [pair, segment] phi [pad16(dk), pad16(dk)], and in seg_states [pair, segment, pad16(dk), pad16(dv)] n of the segment before, then the state
  // that enters.  wild: [pair], a segment that can only be walked from the state itself, or one that a state enters that
  // is not finite; such a pair is walked by one workgroup.
  int segs;
  int64_t seg_chunks;
  float *phi, *seg_states;
  int* wild;
  bool from_zero;  // the sequences begin without a state: the first gate has nothing to act on, and no gradient
};

// ---- operands of the matrix instruction 16x16x32: lane l holds row (or column) l % 16 and 8 inner indices of its quarter l / 16; the result's
// lane holds column l % 16, rows 4 (l / 16) + 0..3.  Inner indices are taken as 4 quarter + 0..3 and 16 + 4 quarter + 0..3 of 32, the order in
// which two results lie in a lane, so results are operands as they are.
template <int N>
struct Op {
  bf16x8 p[N];
};

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }

// acc + a b, without the products of parts below 2^-8(UPTO + 1) of it; the small ones first.
template <int UPTO, int NA, int NB>
__device__ __forceinline__ f32x4 mul(const Op<NA>& a, const Op<NB>& b, f32x4 acc) {
#pragma unroll
  for (int s = UPTO; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) acc = mma(a.p[i], b.p[s - i], acc);
  return acc;
}

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ uint32_t uppers(float x, float y) { return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u); }
__device__ __forceinline__ u32x2 upper_quad(f32x4 x) { return {uppers(x[0], x[1]), uppers(x[2], x[3])}; }
__device__ __forceinline__ f32x4 rest(f32x4 x) { return f32x4{x[0] - upper(x[0]), x[1] - upper(x[1]), x[2] - upper(x[2]), x[3] - upper(x[3])}; }

// Two quads of numbers, split.
template <int N>
__device__ __forceinline__ Op<N> split(f32x4 a, f32x4 b) {
  Op<N> o;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    union { u32x2 h[2]; bf16x8 v; } u;
    u.h[0] = upper_quad(a), u.h[1] = upper_quad(b);
    o.p[i] = u.v;
    if (i + 1 < N) a = rest(a), b = rest(b);
  }
  return o;
}

// A number that the compiler takes for a new one: places that are formed from it are formed where they are used, not once before a loop and
// held in registers for all of it.
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The same for a stride, which all lanes have: multiples of it are formed again by the scalar unit, and not held in more scalar registers than there are.
__device__ __forceinline__ int64_t opaque_stride(int64_t x) {
  asm volatile("" : "+s"(x));
  return x;
}

// ---- tiles in LDS: parts of bfloat16, row by row.
template <class E, int D>
struct Tile {
  static constexpr int N = kParts<E>, ROW = 2 * D + 16, PART = C * ROW, BYTES = N * PART;
  static constexpr __host__ __device__ int row(int i) { return i * ROW; }
};
// A lower triangular matrix of a chunk's steps, of N parts: rows 0 .. 31 have 32 columns, the others 64.
template <int N_>
struct Tri {
  static constexpr int N = N_, PART = 32 * 80 + 32 * 144, BYTES = N * PART;
  static constexpr __host__ __device__ int row(int i) { return i < 32 ? i * 80 : 32 * 80 + (i - 32) * 144; }
};

__device__ __forceinline__ u32x2 read_across(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}
// A lane's places in tiles, formed once.  Opaque, or the compiler would fold tiles' places into an address of its own for every access
// and hold them all.
struct Places {
  int l16, l4;     // (of the operand: row l16, quarter l4)
  int quarter;     // in a row: 8 bytes of it
  int across_row, across_col;  // read across: 4 rows of 16 columns, a lane 4 of them
  __device__ Places() {
    const int lane = threadIdx.x & 63;
    l16 = lane & 15, l4 = lane >> 4;
    quarter = 8 * l4, across_row = 4 * l4 + (l16 >> 2), across_col = 8 * (l16 & 3);
  }
};
template <class T>
struct At {
  static constexpr int FIRST = T::row(1), SECOND = T::row(33) - T::row(32);  // bytes from row to row of the first 32 and of the others
  static constexpr bool ONE = FIRST == SECOND;
  int row[2], col[2];
  __device__ At() {
    const Places p;
    row[0] = opaque(p.l16 * FIRST + p.quarter), col[0] = opaque(p.across_row * FIRST + p.across_col);
    row[1] = ONE ? row[0] : opaque(p.l16 * SECOND + p.quarter), col[1] = ONE ? col[0] : opaque(p.across_row * SECOND + p.across_col);
  }
  // The operand whose rows are the tile's rows 16 t .., inner indices its columns 32 kk ..
  __device__ __forceinline__ Op<T::N> rows(const char* tile, int t, int kk) const {
    Op<T::N> o;
#pragma unroll
    for (int i = 0; i < T::N; ++i) {
      const char* p = tile + (ONE || t < 2 ? row[0] : row[1]) + (i * T::PART + T::row(16 * t) + 64 * kk);
      union { u32x2 h[2]; bf16x8 v; } u;
      u.h[0] = *reinterpret_cast<const u32x2*>(p), u.h[1] = *reinterpret_cast<const u32x2*>(p + 32);
      o.p[i] = u.v;
    }
    return o;
  }
  // ... whose rows are the tile's columns 16 t .., inner indices its rows 32 kk ..: read across by the LDS itself.
  __device__ __forceinline__ Op<T::N> columns(const char* tile, int t, int kk) const {
    Op<T::N> o;
#pragma unroll
    for (int i = 0; i < T::N; ++i) {
      const char* p = tile + (ONE || kk == 0 ? col[0] : col[1]) + (i * T::PART + T::row(32 * kk) + 32 * t);
      union { u32x2 h[2]; bf16x8 v; } u;
      u.h[0] = read_across(p), u.h[1] = read_across(p + 16 * (kk ? SECOND : FIRST));
      o.p[i] = u.v;
    }
    return o;
  }
};
// The number at a tile's row and column.
template <class T>
__device__ __forceinline__ float number_at(const char* tile, int i, int d) {
  float x = 0.f;
#pragma unroll
  for (int n = T::N - 1; n >= 0; --n) x += __uint_as_float((uint32_t) * reinterpret_cast<const uint16_t*>(tile + n * T::PART + T::row(i) + 2 * d) << 16);
  return x;
}

// ... and 4 of them from a place on.
template <class T>
__device__ __forceinline__ f32x4 parts_at(const char* place) {
  f32x4 x;
#pragma unroll
  for (int n = T::N - 1; n >= 0; --n) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(place + n * T::PART);
    const f32x4 y{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
    x = n == T::N - 1 ? y : x + y;
  }
  return x;
}
template <class T>
__device__ __forceinline__ f32x4 numbers_at(const char* tile, int i, int d) { return parts_at<T>(tile + T::row(i) + 2 * d); }

// 4 consecutive elements as they are stored.
template <class E>
struct Four;
template <>
struct Four<bf16> {
  u32x2 w;
  __device__ void put(char* p, int) const { *reinterpret_cast<u32x2*>(p) = w; }
  __device__ void clear() { w = u32x2{0, 0}; }
  __device__ void set(int i, bf16 x) { w[i >> 1] = i & 1 ? (w[i >> 1] & 0xffffu) | (uint32_t)x.bits << 16 : (w[i >> 1] & 0xffff0000u) | x.bits; }
  __device__ f32x4 floats() const {
    return f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
  }
};
template <>
struct Four<float> {
  f32x4 w;
  __device__ void put(char* p, int part) const {
    *reinterpret_cast<u32x2*>(p) = upper_quad(w);
    const f32x4 r = rest(w);
    *reinterpret_cast<u32x2*>(p + part) = upper_quad(r);
    *reinterpret_cast<u32x2*>(p + 2 * part) = upper_quad(rest(r));
  }
  __device__ void clear() { w = zero4(); }
  __device__ void set(int i, float x) { w[i] = x; }
  __device__ f32x4 floats() const { return w; }
};
// The 4 elements from column `col` of a row on, of `dim`.  What lies beyond is read from a place that exists and cleared when it is used: a
// choice made here would wait for the load.
template <class E, bool VEC>
__device__ __forceinline__ Four<E> four(const E* row, int col, int dim) {
  Four<E> x;
  if constexpr (VEC) {
    x = *reinterpret_cast<const Four<E>*>(row + (col < dim ? col : 0));
  } else {
    x.clear();
#pragma unroll
    for (int i = 0; i < 4; ++i) x.set(i, row[col + i < dim ? col + i : 0]);
  }
  return x;
}
template <class E, bool VEC>
__device__ __forceinline__ void clip(Four<E>& x, int col, int dim, bool row) {
  if (!row || col >= dim) x.clear();
  if constexpr (!VEC) {
    const E zero = from_f32<E>(0.f);
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (col + i >= dim) x.set(i, zero);
  }
}

// A chunk's rows of an array on their way to a tile: NT threads, each 4 elements of 64 * D / 4 / NT rows.
template <class E, int D, int NT, bool VEC>
struct Rows {
  static constexpr int PER = C * D / 4 / NT, GROUPS = D / 4;
  static constexpr int APART = NT / GROUPS;  // rows from one of a thread's to the next
  Four<E> x[PER];
  __device__ __forceinline__ void fetch(const E* first, int64_t stride, int dim, int count) {
    const int64_t step = opaque_stride(stride);
    const int tid = opaque(threadIdx.x), r0 = tid / GROUPS, col = tid % GROUPS * 4;
    if (count == C) {
      const E* p = first + r0 * step;
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = four<E, VEC>(p + i * APART * step, col, dim);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int r = r0 + APART * i;
        x[i] = four<E, VEC>(first + (r < count ? r : count - 1) * step, col, dim);
      }
    }
  }
  // rows [from, to) as they are, the others 0
  __device__ __forceinline__ void put(char* tile, int dim, int from, int to) const {
    const int tid = opaque(threadIdx.x), r0 = tid / GROUPS, col = tid % GROUPS * 4;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = r0 + APART * i;
      Four<E> y = x[i];
      clip<E, VEC>(y, col, dim, r >= from && r < to);
      y.put(tile + Tile<E, D>::row(r) + col * 2, Tile<E, D>::PART);
    }
  }
};

// After matrix products that branches lead around: a result may not be read within the next instructions, and the compiler does not follow
// every way to them.
__device__ __forceinline__ void settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 9");
  __builtin_amdgcn_sched_barrier(0);
}

// Between a wavefront's writes to LDS and its reads of what other lanes wrote (the LDS takes a wavefront's accesses in their order; this keeps
// the compiler to it).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Loads of operands are kept from moving up over this: held too early they fill the registers.
__device__ __forceinline__ void apart() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// Launches of the parts (host), for the pairs of `envs` environments from rule.first_env on.
template <class E>
int launch_records(const Rule<E>& r, int64_t envs, hipStream_t s);
template <class E>
int launch_forward(const Rule<E>& r, int64_t envs, hipStream_t s);  // (with its segments)
template <class E>
int launch_backward(const Rule<E>& r, int64_t envs, hipStream_t s);
template <class E>
int launch_gradients(const Rule<E>& r, int64_t envs, hipStream_t s);

// Segments: none where the pairs fill the GPU by themselves; else for one workgroup a CU ([1,16384,16,128+128] bf16: 465 us; 535 for two, more
// to join and no faster walks; 2490 in one piece), of at least 8 chunks, and no fewer than 4 (cutting costs two more walks without outputs,
// which that many segments make up for).
struct Segments {
  int segs;
  int64_t chunks;
};
inline Segments plan_segments(int64_t pairs, int64_t chunks) {
  int64_t segs = device_cus() / pairs;
  if (segs > chunks / 8) segs = chunks / 8;
  if (segs < 4) return {1, chunks};
  const int64_t per = (chunks + segs - 1) / segs;
  return {(int)((chunks + per - 1) / per), per};
}
// Scratch memory of the segments, in floats.
inline size_t segment_floats(int64_t pairs, const Segments& s, int dk, int dv) {
  if (s.segs <= 1) return 0;
  return (size_t)((pairs + 3) / 4 * 4) + (size_t)(pairs * s.segs) * pad16(dk) * (pad16(dk) + pad16(dv));
}

// Whether an array's rows can be read 4 elements at a time.
template <class E>
bool fours(const Seq<E>& x, int dim) {
  return x.data == nullptr || (dim % 4 == 0 && reinterpret_cast<uintptr_t>(x.data) % (4 * sizeof(E)) == 0 && x.env % 4 == 0 && x.step % 4 == 0 &&
                               x.head % 4 == 0);
}

}  // namespace delta
}  // namespace rlk
