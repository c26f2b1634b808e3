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
// A workgroup walks the chunks of its (environment, head, segment) with a wavefront for every 16 columns of c (4
// wavefronts for dims of up to 64, 8 for up to 128).  A wavefront's part of U stays in the accumulators of the matrix instructions for the whole walk: the
// accumulator layout (4 consecutive rows of a column per lane) is also an operand layout once the inner index is
// taken in that order, so U feeds U^T a without a trip through LDS.
//
// Measured (us; floors are bytes at the 5.2 TB/s of a large copy): bfloat16 [64,1024,8,64] 79 forward (floor 52) and 196 for
// the three walks back (90 with each array read once); float32 172 and 468 (103, 181).  [1,16384,16,128], a row of
// segments: states 43, join 8.1, walks 88 (52 for all).  [37,333,4,40 and 72] float32: 59 and 111 (23 for both; the
// useful products alone 13), on 148 of 256 CUs forward, each with the wavefronts' fifth tile of columns on one SIMD.
// Neither HBM nor the matrix units are the bound in bfloat16: the vector units are busy for 46% of the time (a chunk costs a
// wavefront some 490 instructions, two fifths of them splits: the weights' into three numbers, the state's and p's into two; without
// the latter two it took 75 and 185), matrix products for 20%, and
// the rest is waits for LDS and the two barriers of a chunk, with two wavefronts a SIMD to cover them.  In
// float32 matrix products (16x16x4, a sixteenth of bfloat16's rate) take 34% of [37,333,4,40 and 72], over the SIMDs.
#include "rlk_attention.hpp"

namespace rlk {
namespace {

constexpr int C = 64;       // steps per chunk

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Two floats as bfloat16, rounded to nearest even as the instruction does it (a NaN keeps its own bits).
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, bf16x2_t));
}

// 8 consecutive (in the inner index) elements of an operand row: the unit of a matrix instruction's operands.
template <class E>
struct Frag;
template <>
struct Frag<bf16> {
  bf16x8 x;
  __device__ static Frag load(const char* p) { return {*reinterpret_cast<const bf16x8*>(p)}; }
  __device__ static Frag load2(const char* p, const char* q) {
    union { u32x2 h[2]; bf16x8 v; } u;
    u.h[0] = *reinterpret_cast<const u32x2*>(p), u.h[1] = *reinterpret_cast<const u32x2*>(q);
    return {u.v};
  }
  __device__ static Frag from(f32x4 a, f32x4 b) {
    union { uint32_t w[4]; bf16x8 v; } u;
    u.w[0] = bf16_pair(a[0], a[1]), u.w[1] = bf16_pair(a[2], a[3]);
    u.w[2] = bf16_pair(b[0], b[1]), u.w[3] = bf16_pair(b[2], b[3]);
    return {u.v};
  }
};
template <>
struct Frag<float> {
  f32x4 lo, hi;
  __device__ static Frag load(const char* p) { return load2(p, p + 16); }
  __device__ static Frag load2(const char* p, const char* q) {
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

// The first 16 of the inner indices only, where the operands' `lo` hold those.
__device__ __forceinline__ f32x4 mma_half(const Frag<float>& a, const Frag<float>& b, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[i], b.lo[i], acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ f32x4 mma_half(const Frag<bf16>& a, const Frag<bf16>& b, f32x4 acc) { return mma(a, b, acc); }

// 4 consecutive elements.
template <class E>
struct Quad;
template <>
struct Quad<bf16> {
  u32x2 w;
  __device__ static Quad of(f32x4 x) { return {{bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3])}}; }
  __device__ static Quad bits(bf16 a, bf16 b, bf16 c, bf16 d) {
    return {{(uint32_t)a.bits | (uint32_t)b.bits << 16, (uint32_t)c.bits | (uint32_t)d.bits << 16}};
  }
  __device__ static Quad load(const bf16* p) { return {*reinterpret_cast<const u32x2*>(p)}; }
  __device__ void store(bf16* p) const { *reinterpret_cast<u32x2*>(p) = w; }
  __device__ void clear() { w = u32x2{0, 0}; }
  // sum + each element's square
  __device__ float squares(float sum) const {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const pair x = __builtin_bit_cast(pair, (uint32_t)w[0]), y = __builtin_bit_cast(pair, (uint32_t)w[1]);
    return __builtin_amdgcn_fdot2_f32_bf16(y, y, __builtin_amdgcn_fdot2_f32_bf16(x, x, sum, false), false);
  }
  // element x of four quads
  template <int X>
  __device__ static Quad across(const Quad& a, const Quad& b, const Quad& c, const Quad& d) {
    constexpr uint32_t sel = X & 1 ? 0x07060302u : 0x05040100u;
    return {{__builtin_amdgcn_perm(b.w[X >> 1], a.w[X >> 1], sel), __builtin_amdgcn_perm(d.w[X >> 1], c.w[X >> 1], sel)}};
  }
};
template <>
struct Quad<float> {
  f32x4 w;
  __device__ static Quad of(f32x4 x) { return {x}; }
  __device__ static Quad bits(float a, float b, float c, float d) { return {{a, b, c, d}}; }
  __device__ static Quad load(const float* p) { return {*reinterpret_cast<const f32x4*>(p)}; }
  __device__ void store(float* p) const { *reinterpret_cast<f32x4*>(p) = w; }
  __device__ void clear() { w = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ float squares(float sum) const { return fmaf(w[3], w[3], fmaf(w[2], w[2], fmaf(w[1], w[1], fmaf(w[0], w[0], sum)))); }
  template <int X>
  __device__ static Quad across(const Quad& a, const Quad& b, const Quad& c, const Quad& d) {
    return {{a.w[X], b.w[X], c.w[X], d.w[X]}};
  }
};

// After matrix products that branches lead around: a copy of a result, which such a way reaches within a few instructions, was
// emitted without the wait that it needs, and read the sums of before (states wrong in two rows of four).  So the wait
// stands here, in the way of everything.
__device__ __forceinline__ void settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 9");
  __builtin_amdgcn_sched_barrier(0);
}

// x^n for n >= 0 from log2 x (x = 0: 1, 0, 0, ...).
__device__ __forceinline__ float power(float log2x, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(log2x * (float)n); }

// A chunk in LDS, in bytes.  Accesses are a lane's offset, formed once, plus a constant: the offsets are made opaque, or the
// compiler would fold the tiles' places (past the 64 KB that an instruction's own offset reaches) into an address of its own
// for every access and hold them all.
template <class E, int D>
struct Lds {
  static constexpr int S = (int)sizeof(E), PAD = 16;
  static constexpr int ROW = D * S + PAD, PROW = C * S + PAD, TROW = C * S;
  static constexpr int BT = 0, CT = D * TROW;                // b and c transposed, at transposed(d, j)
  static constexpr int A = 2 * D * TROW, B = A + C * ROW;    // rows of a and b
  static constexpr int CHUNK = B + C * ROW;
  // Two chunks where they fit (160 KB a CU; two workgroups of it for bfloat16 dims of up to 64): the next one is put down
  // while this one is worked on.  float32 dims of up to 64 have one, and two workgroups a CU (training [64,1024,8,64] 645 us;
  // two chunks and one workgroup 818).
  // p, (a_i . b_j) lambda^{i-j} same(j, i).  bfloat16: as two numbers, the upper ones first, without the columns past the diagonal's
  // tiles (rows 0 .. 31 have 32 columns, the others 64) and without padding: the 16-byte units of a row are exchanged with
  // its number, so that a column of 16 rows' units lies in all banks.
  static constexpr bool PARTS = S == 2;
  static constexpr int P_PART = 32 * 32 * S + 32 * C * S;
  static constexpr int P_BYTES = PARTS ? 2 * P_PART : C * PROW;
  static constexpr bool OVER = S == 4 && D == 64;            // p in the place of b's rows, which are read for nothing else
  static constexpr int CHUNKS = !OVER && 2 * CHUNK + P_BYTES <= 160 * 1024 ? 2 : 1;
  static constexpr int P = OVER ? B : CHUNKS * CHUNK;
  static constexpr int BYTES = CHUNKS * CHUNK + (OVER ? 0 : P_BYTES);
  static_assert(D == 128 || 2 * BYTES <= 160 * 1024, "two workgroups a CU");
  // whether wavefront w has put down an inf, a NaN or a value near the type's largest: in the padding of a's first rows
  __device__ static constexpr int taint(int w) { return A + (w >> 2) * ROW + D * S + (w & 3) * 4; }
  // where the upper numbers of p's row i, columns j .. j + 3 lie (bfloat16)
  __device__ static int part(int i, int j) {
    const int unit = j * S / 16;
    return P + (i < 32 ? i * 64 + (unit ^ ((i >> 2) & 3)) * 16 : 2048 + (i - 32) * 128 + (unit ^ ((i >> 1) & 7)) * 16) + j * S % 16;
  }
  // Where a transposed tile holds row d, column j.  The 16-byte units of a row are exchanged with d's low bits: a write has
  // lanes at every fourth row, a read at consecutive ones, and f takes all 8 values over either set, so both spread over
  // all banks (with padded rows the writes met in an eighth of them: 20 of 75 us of a [64,1024,8,64] call).
  __device__ static int transposed(int d, int j) {
    const int f = (d & 7) ^ ((d >> 3) & 3);
    return d * TROW + (((j * S / 16) ^ f) * 16) + j * S % 16;
  }
};
__device__ __forceinline__ int opaque(int x) {
  asm("" : "+v"(x));
  return x;
}

// One array's part of a chunk, held by a thread: R rows of 4 columns.
template <class E, int D>
struct Part {
  static constexpr int GROUPS = D / 4, R = C * GROUPS / (4 * D);
  static_assert(R == 4, "a square of 4 x 4 elements per thread");
  Quad<E> x[R];
  const E* p;     // the first row's place
  int64_t step;   // from a walk's step to the next, in elements
  bool columns;   // this thread's columns exist

  __device__ __forceinline__ void start(const E* base, int64_t stride, int dim, int64_t first, int64_t T, bool reverse) {
    const int col = (threadIdx.x % GROUPS) * 4, row0 = (threadIdx.x / GROUPS) * R;
    columns = col < dim;
    step = reverse ? -stride : stride;
    p = base + (reverse ? T - 1 : 0) * stride + (first + row0) * step + (columns ? col : 0);
  }
  // Loads the next chunk's rows, of which `count` exist; rows beyond are loaded from the last one and cleared
  // when the part is put down.  No branch on a lane's own position: the loads leave together.
  template <bool VEC>
  __device__ __forceinline__ Quad<E> quad(const E* q, int dim) const {
    if constexpr (VEC) return Quad<E>::load(q);
    const int left = dim - (threadIdx.x % GROUPS) * 4 - 1;  // the last column's offset, if these exist
    return Quad<E>::bits(q[0], q[columns && left > 0 ? 1 : 0], q[columns && left > 1 ? 2 : 0], q[columns && left > 2 ? 3 : 0]);
  }
  template <bool VEC>
  __device__ __forceinline__ void fetch(int dim) {
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = quad<VEC>(p + r * step, dim);
    p += C * step;
  }
  template <bool VEC>
  __device__ __forceinline__ void fetch_some(int dim, int count) {
    const int row0 = (threadIdx.x / GROUPS) * R;
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = quad<VEC>(p + ((row0 + r < count ? row0 + r : count - 1) - row0) * step, dim);
  }
  // Clears what lies beyond the chunk's rows or the array's columns.
  template <bool VEC>
  __device__ __forceinline__ void clip(int dim, int count) {
    const int col = (threadIdx.x % GROUPS) * 4, row0 = (threadIdx.x / GROUPS) * R;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!columns || row0 + r >= count) x[r].clear();
      if constexpr (!VEC) {
        const E zero = from_f32<E>(0.f);
        const E* e = reinterpret_cast<const E*>(&x[r]);
        x[r] = Quad<E>::bits(e[0], col + 1 < dim ? e[1] : zero, col + 2 < dim ? e[2] : zero, col + 3 < dim ? e[3] : zero);
      }
    }
  }
  __device__ __forceinline__ float squares(float sum) const {
#pragma unroll
    for (int r = 0; r < R; ++r) sum = x[r].squares(sum);
    return sum;
  }
  // to `at` and three rows on
  __device__ __forceinline__ void put(char* at) const {
#pragma unroll
    for (int r = 0; r < R; ++r) x[r].store(reinterpret_cast<E*>(at + r * Lds<E, D>::ROW));
  }
  // as 4 rows of 4 consecutive elements
  __device__ __forceinline__ void put_transposed(char* tile, const int (&at)[4]) const {
    Quad<E>::template across<0>(x[0], x[1], x[2], x[3]).store(reinterpret_cast<E*>(tile + at[0]));
    Quad<E>::template across<1>(x[0], x[1], x[2], x[3]).store(reinterpret_cast<E*>(tile + at[1]));
    Quad<E>::template across<2>(x[0], x[1], x[2], x[3]).store(reinterpret_cast<E*>(tile + at[2]));
    Quad<E>::template across<3>(x[0], x[1], x[2], x[3]).store(reinterpret_cast<E*>(tile + at[3]));
  }
};

// A number's upper 16 bits, as a float and for two as bfloat16.
__device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ uint32_t uppers(float x, float y) { return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u); }

// acc += a (w * c) for an operand row c and weights w of its inner indices.  The weighted bfloat16 operand is taken as the sum
// of three bfloat16 numbers, the product's upper, middle and lower 8 bits: the state is a float32 result and sums over
// all steps (with one rounding of a term to 8 bits it would be off by 2^-9 of itself, with two numbers by 2.5e-6; three are
// the float32 product).
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
  Frag<bf16> hi, mid, lo;
  __device__ Weighted(const Frag<bf16>& c, const float (&w)[8]) {
    union { bf16x8 v; uint32_t u[4]; } in{c.x}, h, m, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = Words<bf16>::get(in.u[i], 0) * w[2 * i], b = Words<bf16>::get(in.u[i], 1) * w[2 * i + 1];
      h.u[i] = uppers(a, b);
      a -= upper(a), b -= upper(b);
      m.u[i] = uppers(a, b);
      a -= upper(a), b -= upper(b);
      l.u[i] = uppers(a, b);
    }
    hi.x = h.v, mid.x = m.v, lo.x = l.v;
  }
  __device__ f32x4 mma_with(const Frag<bf16>& a, f32x4 acc) const { return mma(a, hi, mma(a, mid, mma(a, lo, acc))); }
};

// A factor that is not one of the call's arrays, for products with one that is: the state where outputs are read from it, and p.
// float32: itself.  bfloat16: the sum of two bfloat16 numbers, the upper 8 bits and the next 8 rounded, 2^-15 off at the most.
// (As one number, 2^-8 off, outputs had half as much error again as their own rounding gives them.)  ANY: not only finite
// numbers; an infinity's rest, inf - inf, is then a number that makes no difference to it.
template <class E>
struct Factor;
template <>
struct Factor<float> {
  Frag<float> x;
  template <bool ANY>
  __device__ static Factor from(f32x4 a, f32x4 b) { return {Frag<float>::from(a, b)}; }
  // acc[t] += this * rows[t]
  template <int N>
  __device__ void times(const Frag<float> (&rows)[N], f32x4* acc, bool half) const {
#pragma unroll
    for (int t = 0; t < N; ++t) acc[t] = half ? mma_half(x, rows[t], acc[t]) : mma(x, rows[t], acc[t]);
  }
};
__device__ __forceinline__ u32x2 upper_quad(f32x4 x) { return {uppers(x[0], x[1]), uppers(x[2], x[3])}; }
template <bool ANY>
__device__ __forceinline__ u32x2 rest_quad(f32x4 x) {
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = x[i] - upper(x[i]);
    if constexpr (ANY) r[i] = fminf(r[i], 0x1p126f);  // (of a NaN and a number the number)
  }
  return {bf16_pair(r[0], r[1]), bf16_pair(r[2], r[3])};
}
template <>
struct Factor<bf16> {
  Frag<bf16> hi, lo;
  template <bool ANY>
  __device__ static Factor from(f32x4 a, f32x4 b) {
    union { u32x2 h[2]; bf16x8 v; } h, l;
    h.h[0] = upper_quad(a), h.h[1] = upper_quad(b);
    l.h[0] = rest_quad<ANY>(a), l.h[1] = rest_quad<ANY>(b);
    return {{h.v}, {l.v}};
  }
  template <int N>
  __device__ void times(const Frag<bf16> (&rows)[N], f32x4* acc, bool) const {
#pragma unroll
    for (int t = 0; t < N; ++t) acc[t] = mma(lo, rows[t], acc[t]);
#pragma unroll
    for (int t = 0; t < N; ++t) acc[t] = mma(hi, rows[t], acc[t]);
  }
};

// Which walk of which environment and head a workgroup takes.  Workgroups go round the 8 XCDs, so the walks over the same
// arrays (a backward pass's three) are 8 apart: on one XCD, one after the other, where they find what the others
// have read in its L2.
struct Place {
  int walk, head;
  int64_t env;
  bool there;
  template <class W>
  __device__ explicit Place(const W& walks) {
    const uint32_t x = blockIdx.x, count = (uint32_t)walks.count;
    const uint32_t eh = x / (8 * count) * 8 + x % 8;
    walk = (int)(x / 8 % count);
    head = (int)(eh % (uint32_t)walks.heads);
    env = eh / (uint32_t)walks.heads;
    there = env < walks.num_envs;
    env += walks.first_env;
  }
};

// The walk over a segment.  STATE: only the state at its end, from zero, for the segments after it.
//
// Wavefront w owns the columns 16 w .. 16 w + 15 of c.  Everything a whole chunk without a cut needs of the
// decay is in registers before the walk, and such chunks run through code without a question about them.
// FORM 2: dims of exactly D; 1: dims are multiples of 4, tiles of the padded dims that hold nothing are skipped;
// 0: any dims and alignment, element by element.
template <class E, int D, int FORM, bool STATE>
__global__ __launch_bounds__(4 * D, 2) void walk_kernel(const Walks<E> walks) {
  typedef Lds<E, D> M;
  __shared__ __align__(16) char lds[M::BYTES];
  constexpr int MT = D / 16, KK = D / 32;
  constexpr int SHARE = D / 64, TILES = 4 / SHARE;  // wavefronts that share 16 rows of p; tiles of p a wavefront at most
  const Place place(walks);
  if (!place.there) return;
  const Walk<E>& w = walks.w[place.walk];
  const int head = place.head, seg = blockIdx.y;
  const int64_t env = place.env, T = walks.seq_len;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, l4 = lane >> 4;
  constexpr bool VEC = FORM > 0, FULL = FORM == 2;
  const int da = FULL ? D : w.da, dc = FULL ? D : w.dc;
  const int64_t first = (int64_t)seg * walks.seg_len, last = first + walks.seg_len < T ? first + walks.seg_len : T;
  const float lambda = walks.decay[head], lg = __log2f(lambda);
  const float* dones = walks.dones ? walks.dones + env * T : nullptr;
  const bool reverse = w.reverse;
  // of the squares of a thread's values: below it each is below 2^60, 2^60 / scale, and no product of two rows overflows, scaled or not
  const float limit = fabsf(w.scale) > 1.f ? 0x1p120f / w.scale / w.scale : 0x1p120f;

  Part<E, D> pa, pb, pc;
  if constexpr (!STATE) pa.start(w.a.data + env * w.a.env_stride + head * w.a.head_stride, w.a.step_stride, da, first, T, reverse);
  pb.start(w.b.data + env * w.b.env_stride + head * w.b.head_stride, w.b.step_stride, da, first, T, reverse);
  pc.start(w.c.data + env * w.c.env_stride + head * w.c.head_stride, w.c.step_stride, dc, first, T, reverse);
  float done = 0.f;  // of this lane's step of the next chunk: looked at when the chunk's other loads are (a ballot
                     // when it is loaded would wait for all of them)
  auto fetch_all = [&](int64_t s0) {
    if (last - s0 >= C) {
      if constexpr (!STATE) pa.template fetch<VEC>(da);
      pb.template fetch<VEC>(da);
      pc.template fetch<VEC>(dc);
    } else {
      const int count = (int)(last - s0);
      if constexpr (!STATE) pa.template fetch_some<VEC>(da, count);
      pb.template fetch_some<VEC>(da, count);
      pc.template fetch_some<VEC>(dc, count);
    }
    if (dones != nullptr) {
      const int64_t s = s0 + lane < last ? s0 + lane : last - 1;
      done = dones[reverse ? T - 1 - s : s > 0 ? s - 1 : 0];
    }
  };
  fetch_all(first);

  // U[da][dc]: lane holds column 16 wave + l16, rows 16 m + 4 l4 + 0..3
  f32x4 U[MT];
  const int64_t eh = env * walks.heads + head;
  {
    const float* p = nullptr;
    float f = 1.f;
    bool across = false;
    if (!STATE) {
      if (seg > 0) {
        p = w.seg_states + (eh * walks.segs + seg) * (int64_t)(da * dc);
      } else if (w.state != nullptr) {
        p = w.state + eh * (int64_t)(da * dc);
        f = reverse ? w.state_scale : w.state_scale * lambda;
        across = w.transposed;
      }
    }
    const int j = 16 * wave + l16, jc = j < dc ? j : 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      U[m] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (p != nullptr && 16 * m < da)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * m + 4 * l4 + r, ic = i < da ? i : 0;
          U[m][r] = p[across ? jc * da + ic : ic * dc + jc];
        }
    }
    if (p != nullptr)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) U[m][r] = 16 * m + 4 * l4 + r < da && j < dc && f != 0.f ? U[m][r] * f : 0.f;
  }

  // This wavefront's part of p: rows i = 16 ti + l16, tiles of columns jt = wave % SHARE + SHARE u.  Computed
  // transposed, so that a lane holds 4 consecutive j; scale lambda^{i-j} of its elements, 0 for j > i.
  const int ti = wave / SHARE;
  f32x4 among[STATE ? 1 : TILES];
  float back[4];  // scale lambda^i of the output rows i = 16 t + l16
  if constexpr (!STATE) {
#pragma unroll
    for (int u = 0; u < TILES; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * ti + l16 - (16 * (wave % SHARE + SHARE * u) + 4 * l4 + r);
        among[u][r] = d < 0 ? 0.f : power(lg, d) * w.scale;
      }
#pragma unroll
    for (int t = 0; t < 4; ++t) back[t] = power(lg, 16 * t + l16) * w.scale;
  }
  float onward[2];  // lambda^{C-j} of the steps j = 32 kk + 8 l4 + 7; the 7 before are lambda times the next
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) onward[kk] = power(lg, C - (32 * kk + 8 * l4 + 7));
  const float whole = power(lg, C);

  E* gy = nullptr;
  int64_t ystep = 0;
  if constexpr (!STATE) {
    ystep = reverse ? -w.y.step_stride : w.y.step_stride;
    gy = w.y.data + env * w.y.env_stride + head * w.y.head_stride + (reverse ? T - 1 : 0) * w.y.step_stride + (first + l16) * ystep +
         16 * wave + 4 * l4;
  }

  // this lane's places in LDS
  constexpr bool HALVES = sizeof(E) == 4;  // an operand of 8 elements is two 16-byte units; else the two chunk halves differ
  const int col = (threadIdx.x % Part<E, D>::GROUPS) * 4, row0 = (threadIdx.x / Part<E, D>::GROUPS) * 4;
  const int at_row = opaque(M::A + row0 * M::ROW + col * M::S);
  const int at_col[4] = {opaque(M::transposed(col, row0)), opaque(M::transposed(col + 1, row0)), opaque(M::transposed(col + 2, row0)),
                         opaque(M::transposed(col + 3, row0))};
  constexpr int PER = HALVES ? 4 : 8;  // consecutive inner indices of a lane, of rows
  const int at_a = opaque(M::A + (16 * ti + l16) * M::ROW + PER * l4 * M::S);
  const int at_b = opaque(M::B + (16 * (wave % SHARE) + l16) * M::ROW + PER * l4 * M::S);
  const int at_a2 = opaque(M::A + l16 * M::ROW + 4 * l4 * M::S);
  const int at_p_put = opaque(M::PARTS ? M::part(16 * ti + l16, 16 * (wave % SHARE) + 4 * l4)
                                       : M::P + (16 * ti + l16) * M::PROW + (16 * (wave % SHARE) + 4 * l4) * M::S);
  const int at_p = opaque(M::PARTS ? M::part(l16, 8 * l4) : M::P + l16 * M::PROW + 8 * l4 * M::S);
  const int at_p2[2] = {M::PARTS ? opaque(M::part(32 + l16, 8 * l4)) : 0, M::PARTS ? opaque(M::part(32 + l16, 32 + 8 * l4)) : 0};
  const int step2 = HALVES ? 4 : 32;
  const int at_bt[2][2] = {{opaque(M::transposed(l16, 8 * l4)), opaque(M::transposed(l16, 8 * l4 + step2))},
                           {opaque(M::transposed(16 + l16, 8 * l4)), opaque(M::transposed(16 + l16, 8 * l4 + step2))}};
  const int at_ct[2] = {opaque(M::CT + M::transposed(16 * wave + l16, 8 * l4)), opaque(M::CT + M::transposed(16 * wave + l16, 8 * l4 + step2))};
  // 8 elements of a transposed tile from column 32 kk on, `more` bytes further
  auto load_t = [&](const char* tile, const int (&at)[2], int kk, int more) {
    if constexpr (HALVES) return Frag<E>::load2(tile + at[0] + 32 * kk * M::S + more, tile + at[1] + 32 * kk * M::S + more);
    else return Frag<E>::load(tile + at[kk] + more);
  };

  auto load_row = [](const char* p) {
    if constexpr (HALVES) return Frag<E>::load2(p, p + 16 * M::S);
    else return Frag<E>::load(p);
  };

  bool crossed = false;  // a cut anywhere in the segment
  // a state of this wavefront's that is not finite, in bfloat16: its chunks are none of the plain ones
  bool wild = false;
  auto look = [&] {
    if constexpr (!STATE && M::PARTS) {
      float sum = 0.f;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum = fmaf(0.f, U[m][r], sum);
      wild = __any(sum != 0.f);
    }
  };
  look();
  // Puts the fetched chunk of the steps from s0 on down and has the one after it fetched; its cuts come back.
  auto put_down = [&](int64_t s0, int buffer) {
    const int L = (int)(last - s0 < C ? last - s0 : C);
    const uint64_t found = __ballot(lane < L && done != 0.f && (reverse || s0 + lane > 0));
    if (!FULL || L < C) {
      if constexpr (!STATE) pa.template clip<VEC>(da, L);
      pb.template clip<VEC>(da, L);
      pc.template clip<VEC>(dc, L);
    }
    char* to = lds + buffer;
    float sum = pc.squares(pb.squares(0.f));
    if constexpr (!STATE) sum = pa.squares(sum);
    const bool tainted = __any(!(sum < limit));
    if (lane == 0) *reinterpret_cast<int*>(to + M::taint(wave)) = tainted;
    if constexpr (!STATE) {
      pa.put(to + at_row);
      pb.put(to + at_row + (M::B - M::A));
    }
    pb.put_transposed(to, at_col);
    pc.put_transposed(to + M::CT, at_col);
    if (s0 + C < last) fetch_all(s0 + C);
    return found;
  };

  // One chunk, unless it is tainted.  PLAIN: whole, without a cut, from a finite state, and not the one that a state leaves the
  // sequence with.  (Wavefronts may go through different forms of a chunk: both have the same barriers.)
  auto chunk = [&](auto plain, int64_t s0, int L, uint64_t cuts, bool end, const char* tile) {
    constexpr bool PLAIN = decltype(plain)::value;
    int4 mark = *reinterpret_cast<const int4*>(tile + M::taint(0));
    if constexpr (D == 128) {
      const int4 more = *reinterpret_cast<const int4*>(tile + M::taint(4));
      mark.x |= more.x | more.y | more.z | more.w;
    }
    // operands that take more registers: loads of more than the next two are kept from moving up
    auto apart = [] {
      if constexpr (sizeof(E) == 4 || D == 128) __builtin_amdgcn_sched_barrier(0);
    };
    // The lane's place again, for what only other chunks need: as a new value to the compiler, which would else compute
    // all of it once before the walk and hold it in a hundred registers.
    int v16 = l16, v4 = l4;
    if constexpr (!PLAIN) asm volatile("" : "+v"(v16), "+v"(v4));
    if constexpr (!STATE) {
      int begin = 0;  // of row i's episode: the last cut at or before it
      if (!PLAIN && cuts != 0) {
        const uint64_t before = cuts & (((uint64_t)2 << (16 * ti + v16)) - 1);
        begin = before != 0 ? 63 - __clzll((long long)before) : 0;
      }
      f32x4 pts[TILES];
#pragma unroll
      for (int u = 0; u < TILES; ++u) pts[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (!FULL && 32 * kk >= da) continue;
        const bool half = !FULL && da - 32 * kk <= 16;
        const Frag<E> fa = load_row(tile + at_a + 32 * kk * M::S);
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
          // (tiles past the diagonal too, whose `among` is 0: the wavefront with the last rows has none, the others would wait for it)
          const Frag<E> fb = load_row(tile + at_b + 16 * SHARE * u * M::ROW + 32 * kk * M::S);
          pts[u] = half ? mma_half(fb, fa, pts[u]) : mma(fb, fa, pts[u]);
        }
      }
      if constexpr (!FULL) settle();
      if constexpr (M::OVER) __syncthreads();
#pragma unroll
      for (int u = 0; u < TILES; ++u) {
        const int jt = wave % SHARE + SHARE * u;
        f32x4 pt = pts[u];
        pt *= among[u];
        if (!PLAIN && cuts != 0) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * jt + 4 * v4 + r < begin) pt[r] = 0.f;
        }
        if constexpr (M::PARTS) {
          // (the units' exchange is of the address's bits 4 to 6)
          if (ti < 2 && SHARE * u >= 2) continue;  // past the diagonal's tiles
          char* p = lds + (at_p_put ^ (16 * SHARE * u * M::S));
          *reinterpret_cast<u32x2*>(p) = upper_quad(pt);
          *reinterpret_cast<u32x2*>(p + M::P_PART) = rest_quad<false>(pt);
        } else {
          Quad<E>::of(pt).store(reinterpret_cast<E*>(lds + at_p_put + 16 * SHARE * u * M::S));
        }
      }
      __syncthreads();
    }
    if (__builtin_amdgcn_readfirstlane(mark.x | mark.y | mark.z | mark.w) != 0) return false;

    Frag<E> fc[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) fc[kk] = load_t(tile, at_ct, kk, 0);
    const bool mine = FULL || 16 * wave < dc;  // else this wavefront only helps with p

    if (!STATE && mine) {
      // y^T: rows = this wavefront's columns of c, columns i = 16 t + l16
      f32x4 y[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) y[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if (!FULL && 32 * kk >= da) continue;
        const bool half = !FULL && da - 32 * kk <= 16;
        const Factor<E> fu = Factor<E>::template from<!PLAIN>(U[2 * kk], U[2 * kk + 1]);
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
          const char *row = tile + at_a2 + 16 * t * M::ROW + 32 * kk * M::S, *next = row + 16 * M::ROW;
          const Frag<E> fr[2] = {Frag<E>::load2(row, row + 16 * M::S), Frag<E>::load2(next, next + 16 * M::S)};
          fu.times(fr, y + t, half);
          apart();
        }
      }
      if constexpr (!FULL) settle();
      // the first step that the state does not reach
      const int until = PLAIN || cuts == 0 ? C : __ffsll((long long)cuts) - 1;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        y[t] *= back[t];
        if (!PLAIN && 16 * t + v16 >= until) y[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int t = 2 * kk; t < 4; ++t) {  // (rows before the steps 32 kk + 0..31 have none of them)
          if constexpr (M::PARTS) {
            const char* p = lds + (t < 2 ? at_p + 1024 * t : at_p2[kk] + 2048 * (t - 2));
            y[t] = mma(fc[kk], Frag<E>::load(p), mma(fc[kk], Frag<E>::load(p + M::P_PART), y[t]));
          } else {
            y[t] = mma(fc[kk], Frag<E>::load(lds + at_p + 16 * t * M::PROW + 32 * kk * M::S), y[t]);
          }
          if (t & 1) apart();
        }
      const int j = 16 * wave + 4 * l4;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        E* p = gy + (16 * t) * ystep;
        const Quad<E> v = Quad<E>::of(y[t]);
        if (VEC) {
          if ((PLAIN || 16 * t + v16 < L) && (FULL || j < dc)) v.store(p);
        } else if (PLAIN || 16 * t + v16 < L) {
          const E* e = reinterpret_cast<const E*>(&v);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (j + r < dc) p[r] = e[r];
        }
      }
      gy += C * ystep;
    }

    // U' = lambda^reach U + sum over steps from the last cut on of lambda^{reach-j} b_j c_j^T.  The state that
    // leaves the sequence forward is the one after its last step, not decayed by another.
    if (mine) {
      const int reach = !PLAIN && end ? L - 1 : L, from = PLAIN || cuts == 0 ? 0 : 63 - __clzll((long long)cuts);
      const float keep = PLAIN ? whole : power(lg, reach);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        U[m] *= keep;
        if (!PLAIN && cuts != 0) U[m] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        float f[8];
        f[7] = onward[kk];
#pragma unroll
        for (int x = 6; x >= 0; --x) f[x] = f[x + 1] * lambda;
        if constexpr (!PLAIN) {
          const int j = 32 * kk + 8 * v4;
          if (reach != C) {
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = j + x < L ? power(lg, reach - j - x) : 0.f;
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] = j + x >= from ? f[x] : 0.f;
        }
        const Weighted<E> wc(fc[kk], f);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (FULL || 16 * m < da) U[m] = wc.mma_with(load_t(tile, at_bt[m & 1], kk, 16 * (m & ~1) * M::TROW), U[m]);
          if (m & 1) apart();
        }
      }
      settle();
    }
    return true;
  };

  // A chunk that holds an inf, a NaN or values whose products overflow, step by step: as products of matrices it would put
  // them (0 inf = NaN) where the recurrence does not, in steps before them and past an episode's end.  bfloat16 [1,16384,16,128]: 129 us
  // without such a chunk, 2526 with one in every chunk; looking for them costs 3% ([64,1024,8,64] training 264 -> 269).
  auto careful = [&](int64_t s0, int L, uint64_t cuts, bool end, const char* tile) {
    int v16 = l16, v4 = l4;
    for (int i = 0; i < L; ++i) {
      asm volatile("" : "+v"(v16), "+v"(v4));  // (as in `chunk`)
      const int j = 16 * wave + v16;
      const float c = load_one(reinterpret_cast<const E*>(tile + M::CT + M::transposed(j, i)));
      const float keep = i == 0 ? 1.f : lambda;
      const bool cut = (cuts >> i) & 1;
      float sum = 0.f;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = 16 * m + 4 * v4 + r;
          const float b = load_one(reinterpret_cast<const E*>(tile + M::BT + M::transposed(d, i)));
          // (a padded row stays 0: times an inf its zeros would be NaN, and in the sum over all rows)
          U[m][r] = FULL || d < da ? fmaf(b, c, cut || keep == 0.f ? 0.f : U[m][r] * keep) : 0.f;
          if constexpr (!STATE) sum = fmaf(load_one(reinterpret_cast<const E*>(tile + M::A + i * M::ROW + d * M::S)), U[m][r], sum);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (!STATE) {
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (v4 == 0 && j < dc) gy[(i - v16) * ystep + v16] = from_f32<E>(sum * w.scale);
      }
    }
    if constexpr (!STATE) gy += C * ystep;
    if (!end)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) U[m][r] = lambda == 0.f ? 0.f : U[m][r] * lambda;
    look();
  };

  int buffer = 0;
  uint64_t cuts = put_down(first, 0);
  __syncthreads();
  for (int64_t s0 = first; s0 < last; s0 += C) {
    const int L = (int)(last - s0 < C ? last - s0 : C);
    const bool end = !reverse && s0 + C >= T;
    crossed |= cuts != 0;
    if (wild) look();  // (an episode's end may have come)
    const bool whole_chunk = L == C && cuts == 0 && !end && !wild;
    if (!(whole_chunk ? chunk(std::true_type{}, s0, L, cuts, end, lds + buffer) : chunk(std::false_type{}, s0, L, cuts, end, lds + buffer)))
      careful(s0, L, cuts, end, lds + buffer);
    if (s0 + C >= last) break;
    if constexpr (M::CHUNKS == 2) buffer ^= M::CHUNK;
    else __syncthreads();  // the chunk has been read
    cuts = put_down(s0 + C, buffer);
    __syncthreads();
  }

  float* out = nullptr;
  float f = 1.f;
  if (STATE) {
    out = w.seg_states + (eh * walks.segs + seg + 1) * (int64_t)(da * dc);
    if (threadIdx.x == 0) w.seg_keep[eh * walks.segs + seg + 1] = crossed || lambda == 0.f ? -1.f : power(lg, (int)(last - first));
  } else if (last == T && w.state_out != nullptr) {
    out = w.state_out + eh * (int64_t)(da * dc);
    f = !reverse && dones != nullptr && dones[T - 1] != 0.f ? 0.f : w.state_out_scale;
  }
  if (out != nullptr)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * m + 4 * l4 + r, j = 16 * wave + l16;
        if (i < da && j < dc) out[i * dc + j] = f == 0.f ? 0.f : U[m][r] * f;
      }
}

// The states that enter the segments: in place, from what each segment added and how much of what enters it leaves.  The chain is
// one multiply-add a segment: what it waits for are the loads, so 16 are on their way at once.
template <class E>
__global__ __launch_bounds__(256) void join_kernel(const Walks<E> walks) {
  const Walk<E>& w = walks.w[blockIdx.z];
  const int n = w.da * w.dc;
  const int64_t eh = walks.first_env * walks.heads + blockIdx.x;
  const int i = blockIdx.y * 256 + threadIdx.x;
  if (i >= n) return;
  float u = 0.f;
  if (w.state != nullptr) {
    const int64_t at = w.transposed ? (int64_t)(i % w.dc) * w.da + i / w.dc : i;
    const float f = w.reverse ? w.state_scale : w.state_scale * walks.decay[eh % walks.heads];
    u = f == 0.f ? 0.f : w.state[eh * n + at] * f;  // (a decay of 0 leaves nothing of it, NaN included)
  }
  constexpr int AHEAD = 16;
  float* p = w.seg_states + eh * walks.segs * (int64_t)n + i;
  const float* keeps = w.seg_keep + eh * walks.segs;
  for (int s0 = 1; s0 < walks.segs; s0 += AHEAD) {
    float x[AHEAD], keep[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int s = s0 + k < walks.segs ? s0 + k : s0;  // (one that is there, for those past the last)
      x[k] = p[(int64_t)s * n], keep[k] = keeps[s];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (s0 + k >= walks.segs) break;
      u = keep[k] < 0.f ? x[k] : fmaf(u, keep[k], x[k]);  // (no part of u, NaN included, passes an episode's end; one too small to see leaves a NaN)
      p[(int64_t)(s0 + k) * n] = u;
    }
  }
}

// The state that leaves a sequence of no steps: the one that enters it.
__global__ __launch_bounds__(256) void no_steps_state_kernel(const float* state, float* state_out, int64_t pairs, int da, int dc, bool transposed,
                                                             float scale) {
  const int64_t n = (int64_t)da * dc, step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < pairs * n; at += step) {
    const int64_t eh = at / n;
    const int i = (int)(at - eh * n);
    state_out[at] = state == nullptr ? 0.f : state[transposed ? eh * n + (int64_t)(i % dc) * da + i / dc : at] * scale;
  }
}

int no_steps(const rlk_attention& c, hipStream_t s) {
  if (!c.state_out) return RLK_OK;
  const int64_t pairs = c.num_envs * c.heads, units = (pairs * c.dim_k * c.dim_v + 255) / 256;
  no_steps_state_kernel<<<dim3((unsigned)(units < 4096 ? units : 4096)), dim3(256), 0, s>>>(
      c.state, c.state_out, pairs, (int)c.dim_k, (int)c.dim_v, c.state_transposed != 0, c.state_scale * c.state_out_scale);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}

template <class E, int D, int FORM>
int launch_walks(Walks<E> k, int count, hipStream_t s) {
  const int64_t envs = k.num_envs, most = kMaxPairs / k.heads;
  for (k.first_env = 0; k.first_env < envs; k.first_env += most) {
    k.num_envs = envs - k.first_env < most ? envs - k.first_env : most;
    const unsigned rows = (unsigned)(k.num_envs * k.heads);
    const dim3 grid((rows + 7) / 8 * 8 * (unsigned)count, (unsigned)k.segs);
    if (k.segs > 1) {
      walk_kernel<E, D, FORM, true><<<dim3(grid.x, grid.y - 1), dim3(4 * D), 0, s>>>(k);
      int most_state = 0;
      for (int i = 0; i < count; ++i) most_state = most_state < k.w[i].da * k.w[i].dc ? k.w[i].da * k.w[i].dc : most_state;
      join_kernel<E><<<dim3(rows, (unsigned)(most_state + 255) / 256, (unsigned)count), dim3(256), 0, s>>>(k);
    }
    walk_kernel<E, D, FORM, false><<<grid, dim3(4 * D), 0, s>>>(k);
    if (hipGetLastError() != hipSuccess) return RLK_ERR_LAUNCH;
  }
  return RLK_OK;
}

template <class E>
bool quads(const Sequence<E>& x, int dim) {
  return dim % 4 == 0 && (reinterpret_cast<uintptr_t>(x.data) % (4 * sizeof(E))) == 0 && x.env_stride % 4 == 0 &&
         x.step_stride % 4 == 0 && x.head_stride % 4 == 0;
}

template <class E>
int walk_impl(const rlk_attention* c, int count, hipStream_t s) {
  Walks<E> k = {};
  k.count = count, k.num_envs = c->num_envs, k.seq_len = c->seq_len, k.heads = (int)c->heads, k.decay = c->decay, k.dones = c->dones;
  const SegmentPlan plan = plan_segments(c->num_envs * c->heads, c->seq_len, c->dim_k <= 64 && c->dim_v <= 64);
  k.segs = plan.segs, k.seg_len = plan.seg_len;
  bool vec = true, small = true;
  int full = 0;  // the one size that all dims have, or -1
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
    full = w.da == w.dc && (full == 0 || full == w.da) ? w.da : -1;
    if (k.segs > 1) {
      const size_t states = (size_t)k.num_envs * k.heads * k.segs * w.da * w.dc, keeps = (size_t)k.num_envs * k.heads * k.segs;
      if ((states + keeps) * sizeof(float) > left || ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 3u) != 0)
        return RLK_ERR_WORKSPACE;
      w.seg_states = reinterpret_cast<float*>(ws), w.seg_keep = w.seg_states + states;
      ws += (states + keeps) * sizeof(float), left -= (states + keeps) * sizeof(float);
    }
  }
  if (small) {
    if (vec && full == 64) return launch_walks<E, 64, 2>(k, count, s);
    return vec ? launch_walks<E, 64, 1>(k, count, s) : launch_walks<E, 64, 0>(k, count, s);
  }
  if (vec && full == 128) return launch_walks<E, 128, 2>(k, count, s);
  return vec ? launch_walks<E, 128, 1>(k, count, s) : launch_walks<E, 128, 0>(k, count, s);
}

}  // namespace
}  // namespace rlk

using namespace rlk;

extern "C" {

size_t rlk_attention_workspace_bytes(int64_t num_envs, int64_t seq_len, int64_t heads, int64_t dim_k, int64_t dim_v) {
  if (num_envs <= 0 || seq_len <= 0 || heads <= 0 || dim_k <= 0 || dim_v <= 0) return 0;
  const SegmentPlan plan = plan_segments(num_envs * heads, seq_len, dim_k <= 64 && dim_v <= 64);
  return plan.segs <= 1 ? 0 : (size_t)num_envs * heads * plan.segs * (dim_k * dim_v + 1) * sizeof(float);
}

int rlk_linear_attention(const rlk_attention* calls, int count, void* stream) {
  if (!calls || count < 1 || count > 3) return RLK_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < count; ++i) {
    const rlk_attention& c = calls[i];
    if (!valid_attention(c, c.seq_len != 0) || c.seq_len < 0 || c.num_envs != calls->num_envs || c.seq_len != calls->seq_len ||
        c.heads != calls->heads || c.decay != calls->decay || c.dones != calls->dones || c.bf16 != calls->bf16)
      return RLK_ERR_INVALID_ARGUMENT;
  }
  if (calls->num_envs == 0 || calls->heads == 0) return RLK_OK;
  if (calls->heads > kMaxPairs || calls->seq_len > (int64_t{1} << 30)) return RLK_ERR_INVALID_ARGUMENT;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (calls->seq_len == 0) {
    int st = RLK_OK;
    for (int i = 0; i < count && st == RLK_OK; ++i) st = no_steps(calls[i], s);
    return st;
  }
  return calls->bf16 ? walk_impl<bf16>(calls, count, s) : walk_impl<float>(calls, count, s);
}

}  // extern "C"
