// rlk_delta_walk.hip -- the gated delta rule over whole sequences: the walk over the chunks, forward and back (rlk_delta.hpp).
//
// A workgroup walks the chunks of its (environment, head), a wavefront per 16 columns of the state.  Keys, queries, the record's M and the
// chunk's weighted q . k (formed by all wavefronts together) are in LDS; the state stays in the accumulators.  A chunk's three products after
// each other -- what the keys read, the corrections, the state's update -- pass results on as operands in registers: a result's lane holds a
// column and 4 consecutive rows, which is the next product's inner index.  Columns do not meet, so neither do wavefronts.
//
// Bound by a chunk's chain: three products and the splits between them after each other (1300 vector instructions and 150 matrix products a wavefront and
// chunk of 64 rows), two barriers, two wavefronts a SIMD to fill the waits (registers: a state of 128 rows, its split and the next chunk on its
// way; LDS: 77 KB in bf16, 145 KB in float32).  GPU time, us: [64,1024,8,64+64] bf16 forward 194 (3.2 TB/s of what it reads and leaves for
// the way back), back 176 (3.5 TB/s); [1,16384,16,128+128] bf16 194 in 16 segments, the segments' states 185 before them and 43 for joining;
// [37,333,4,40+72] float32 forward 75, back 66 (111 and 124 while keys were padded to the dims of the values).  The walk back is one workgroup a pair
// however few there are: training [1,16384,16,128+128] 3980.
#include "rlk_delta.hpp"

namespace rlk {
namespace delta {
namespace {

// D: dims of the keys padded to 64 or 128.
template <class E, int D>
struct Lds {
  typedef Tile<E, D> Rows_;
  typedef Tri<3> M;  // (the weighted q . k too)
  static constexpr int K = 0, Q = Rows_::BYTES, MT = 2 * Rows_::BYTES, PT = MT + M::BYTES, REST = PT + M::BYTES;
  static constexpr int BYTES = REST + (int)(sizeof(Record) - offsetof(Record, ghi));
};

// The shared part of a walk: a chunk's arrays on their way to LDS, and the weighted q . k.
// QUERIES: else only the keys and M are.
template <class E, int D, int WAVES, bool VEC, bool QUERIES = true>
struct Shared {
  static constexpr int NT = 64 * WAVES;
  typedef Lds<E, D> M;
  static constexpr int TILE_QUADS = 640, REST_QUADS = (int)(sizeof(Record) - offsetof(Record, ghi)) / 16, TILES_PER = (TILE_QUADS + NT - 1) / NT;
  Rows<E, D, NT, VEC> k, q;
  f32x4 m[TILES_PER], rest_quad;

  __device__ __forceinline__ void fetch(const Rule<E>& r, int64_t env, int head, int64_t pair, int64_t chunk) {
    const int64_t s0 = chunk * C;
    const int n = (int)(r.seq_len - s0 < C ? r.seq_len - s0 : C);
    k.fetch(r.k.data + env * r.k.env + head * r.k.head + s0 * r.k.step, r.k.step, r.dk, n);
    if constexpr (QUERIES) q.fetch(r.q.data + env * r.q.env + head * r.q.head + s0 * r.q.step, r.q.step, r.dk, n);
    const f32x4* rec = reinterpret_cast<const f32x4*>(r.records + pair * r.chunks + chunk);
#pragma unroll
    for (int i = 0; i < TILES_PER; ++i) {
      const int u = threadIdx.x + NT * i;
      m[i] = rec[u < TILE_QUADS ? u : 0];
    }
    rest_quad = rec[TILE_QUADS + (threadIdx.x < REST_QUADS ? threadIdx.x : 0)];
  }
  __device__ __forceinline__ void put(char* lds, int dk, int n) const {
    k.put(lds + M::K, dk, 0, n);
    if constexpr (QUERIES) q.put(lds + M::Q, dk, 0, n);
#pragma unroll
    for (int i = 0; i < TILES_PER; ++i) {
      const int u = threadIdx.x + NT * i;
      if (u < TILE_QUADS) {
        const int tile = u / 64, ti = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, tj = tile - ti * (ti + 1) / 2;
        Four<float>{m[i]}.put(lds + M::MT + M::M::row(16 * ti + u % 64 / 4) + 2 * (16 * tj + 4 * (u & 3)), M::M::PART);
        if (ti == tj && (ti == 0 || ti == 2))  // the tile above the diagonal that products go over
          Four<float>{zero4()}.put(lds + M::MT + M::M::row(16 * ti + u % 64 / 4) + 2 * (16 * tj + 16 + 4 * (u & 3)), M::M::PART);
      }
    }
    if (threadIdx.x < REST_QUADS) *reinterpret_cast<f32x4*>(lds + M::REST + 16 * threadIdx.x) = rest_quad;
  }
  __device__ static const Record& record(const char* lds) { return *reinterpret_cast<const Record*>(lds + M::REST - offsetof(Record, ghi)); }

  // P_ij = scale D_ij q_i . k_j.  Wavefronts share the 16 rows ti; computed transposed, so that a lane holds 4 consecutive j.
  __device__ static void form_p(char* lds, float scale, const At<typename M::Rows_>& at) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, l4 = lane >> 4;
    constexpr int SHARE = WAVES / 4;
    const Record& rec = record(lds);
    const uint64_t cuts = rec.cuts[0] | (uint64_t)rec.cuts[1] << 32;
    const int ti = wave / SHARE, i = 16 * ti + l16;
    const uint64_t before = cuts & (((uint64_t)2 << i) - 1);
    const int begin = before != 0 ? 63 - __clzll((long long)before) : 0;
    const float hi = rec.ghi[i], lo = rec.glo[i];
    const int upto = ti | 1;  // (to the end of the 32 columns that products go over)
    for (int tj = wave % SHARE; tj <= upto; tj += SHARE) {
      f32x4 x = zero4();
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) x = mul<2>(at.rows(lds + M::K, tj, kk), at.rows(lds + M::Q, ti, kk), x);
      settle();
      const f32x4 hj = *reinterpret_cast<const f32x4*>(rec.ghi + 16 * tj + 4 * l4), lj = *reinterpret_cast<const f32x4*>(rec.glo + 16 * tj + 4 * l4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 16 * tj + 4 * l4 + e;
        x[e] = j <= i && j >= begin ? x[e] * (scale * __expf((hi - hj[e]) + (lo - lj[e]))) : 0.f;
      }
      Four<float>{x}.put(lds + M::PT + M::M::row(16 * ti) + l16 * (M::M::row(16 * ti + 1) - M::M::row(16 * ti)) + 2 * (16 * tj + 4 * l4), M::M::PART);
    }
  }
};

// 0 for each finite number, NaN for others.
__device__ __forceinline__ float odd(f32x4 x, float sum) { return fmaf(0.f, x[0], fmaf(0.f, x[1], fmaf(0.f, x[2], fmaf(0.f, x[3], sum)))); }

// The gate of a step on its own: 0 where an episode begins or nothing stays.
template <class E>
__device__ __forceinline__ float gate(const Rule<E>& r, int64_t env, int head, int64_t s) {
  if (r.dones != nullptr && s > 0 && r.dones[env * r.seq_len + s - 1] != 0.f) return 0.f;
  if (r.gates == nullptr) return 1.f;
  const float g = r.gates[(env * r.seq_len + s) * r.heads + head];
  return g <= kNoDecay ? 0.f : expf(g);
}

// The state of a pair as it lies outside, [dk, dv] row-major, in a wavefront's accumulators: column 16 wave + l16, rows 16 m + 4 l4 + 0..3.
template <int MT>
__device__ __forceinline__ void load_state(const float* p, int dk, int dv, bool none, f32x4 (&S)[MT]) {
  const int lane = threadIdx.x & 63, l4 = lane >> 4, j = 16 * (threadIdx.x >> 6) + (lane & 15), jc = j < dv ? j : 0;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    S[m] = zero4();
    if (p != nullptr && !none)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 16 * m + 4 * l4 + e;
        const float x = p[(d < dk ? d : 0) * dv + jc];
        S[m][e] = d < dk && j < dv ? x : 0.f;
      }
  }
}
template <int MT>
__device__ __forceinline__ void store_state(float* p, int dk, int dv, bool none, const f32x4 (&S)[MT]) {
  const int lane = threadIdx.x & 63, l4 = lane >> 4, j = 16 * (threadIdx.x >> 6) + (lane & 15);
  if (j >= dv) return;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 16 * m + 4 * l4 + e;
      if (d < dk) p[d * dv + j] = none ? 0.f : S[m][e];
    }
}
// ... into the workspace, [rows, columns] of whole tiles.
template <int MT>
__device__ __forceinline__ void keep_state(float* p, int stride, int rows, const f32x4 (&S)[MT]) {
  const int64_t columns = opaque_stride(stride);
  const int tid = opaque(threadIdx.x), lane = tid & 63;
  p += 4 * (lane >> 4) * columns + 16 * (tid >> 6) + (lane & 15);
#pragma unroll
  for (int m = 0; m < MT; ++m)
    if (16 * m < rows)
#pragma unroll
      for (int e = 0; e < 4; ++e) p[(16 * m + e) * columns] = S[m][e];
}
// ... a chunk's rows of a wavefront's columns.
__device__ __forceinline__ void keep_columns(float* p, int stride, const f32x4 (&x)[4]) {
  const int64_t columns = opaque_stride(stride);
  const int tid = opaque(threadIdx.x), lane = tid & 63;
  p += 4 * (lane >> 4) * columns + 16 * (tid >> 6) + (lane & 15);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) p[(16 * t + e) * columns] = x[t][e];
}

// A wavefront's 16 columns of an array's chunk: column 16 wave + l16, rows 16 t + 4 l4 + 0..3.
template <class E>
__device__ __forceinline__ void load_columns(const E* first, int64_t stride, int dim, int n, E (&x)[16]) {
  const int64_t step = opaque_stride(stride);
  const int tid = opaque(threadIdx.x), lane = tid & 63, l4 = lane >> 4, j = 16 * (tid >> 6) + (lane & 15);
  const E* p = first + (j < dim ? j : dim - 1);
  if (n == C) {
    p += 4 * l4 * step;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * t + e] = p[(16 * t + e) * step];
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 16 * t + 4 * l4 + e;
        x[4 * t + e] = p[(i < n ? i : n - 1) * step];
      }
  }
}
// ... as numbers, 0 where there is nothing.
template <class E>
__device__ __forceinline__ f32x4 columns_quad(const E (&x)[16], int t, int dim, int n) {
  if (n == C && 16 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + 16 <= dim)
    return f32x4{to_f32(x[4 * t]), to_f32(x[4 * t + 1]), to_f32(x[4 * t + 2]), to_f32(x[4 * t + 3])};
  const int lane = threadIdx.x & 63, l4 = lane >> 4, j = 16 * (threadIdx.x >> 6) + (lane & 15);
  f32x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = j < dim && 16 * t + 4 * l4 + e < n ? to_f32(x[4 * t + e]) : 0.f;
  return y;
}

// TRANSITION: no outputs, but what a segment does to the state that enters it: the state that it leaves from none (blockIdx.z 1), and from the
// unit vectors with no values (0).
template <class E, int D, int WAVES, bool VEC, bool TRANSITION>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || kParts<E> == 1 ? 2 : 1) void forward_kernel(const Rule<E> r) {
  constexpr int MT = D / 16, KK = D / 32;
  typedef Shared<E, D, WAVES, VEC, !TRANSITION> Sh;
  typedef typename Sh::M M;
  typedef typename M::Rows_ T;
  __shared__ __align__(16) char lds[M::BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, l4 = lane >> 4;
  const int64_t pair = blockIdx.x, env = r.first_env + pair / r.heads, eh = r.first_env * r.heads + pair;
  const int head = (int)(pair % r.heads), dk = r.dk, seg = blockIdx.y;
  const bool units = TRANSITION && blockIdx.z == 0;
  const int dv = units ? dk : r.dv, dvp = pad16(dv);
  const bool mine = 16 * wave < dv;
  const int j = 16 * wave + l16;
  int64_t first = seg * r.seg_chunks, last = first + r.seg_chunks < r.chunks ? first + r.seg_chunks : r.chunks;
  if (!TRANSITION && r.segs > 1 && r.wild[pair] != 0) {
    if (seg > 0) return;
    last = r.chunks;
  }
  const E* gv = r.v.data + env * r.v.env + head * r.v.head;
  E* gy = r.y.data + env * r.y.env + head * r.y.head;

  const At<T> at;
  const At<typename M::M> at_m;
  Sh sh;
  E v[16];
  sh.fetch(r, env, head, pair, first);
  if (mine && !units) load_columns(gv + first * C * r.v.step, r.v.step, dv, (int)(r.seq_len - first * C < C ? r.seq_len - first * C : C), v);
  f32x4 S[MT];
  if constexpr (TRANSITION) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int x = 0; x < 4; ++x) S[m][x] = units && 16 * m + 4 * l4 + x == j && j < dk ? 1.f : 0.f;
  } else if (seg == 0) {
    load_state(r.state ? r.state + eh * dk * dv : nullptr, dk, dv, false, S);
  } else {
    const float* p = r.seg_states + (pair * r.segs + seg) * (int64_t)pad16(dk) * dvp + j;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int x = 0; x < 4; ++x) S[m][x] = mine && 16 * m < dk ? p[(16 * m + 4 * l4 + x) * dvp] : 0.f;
  }

  for (int64_t chunk = first; chunk < last; ++chunk) {
    const int64_t s0 = chunk * C;
    const int n = (int)(r.seq_len - s0 < C ? r.seq_len - s0 : C);
    sh.put(lds, dk, n);
    __syncthreads();
    if (chunk + 1 < last) sh.fetch(r, env, head, pair, chunk + 1);
    if constexpr (!TRANSITION) Sh::form_p(lds, r.scale, at);
    const Record& rec = Sh::record(lds);

    f32x4 e[4], y[4];  // corrections (column j, steps 16 t + 4 l4 + ..); outputs, transposed (step 16 t + l16, columns 16 wave + 4 l4 + ..)
    Op<3> u[2];
    if (mine) {
      f32x4 ks[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) ks[t] = y[t] = zero4();
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const Op<3> s = split<3>(S[2 * kk], S[2 * kk + 1]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          ks[t] = mul<2>(at.rows(lds + M::K, t, kk), s, ks[t]);
          if constexpr (!TRANSITION) y[t] = mul<2>(s, at.rows(lds + M::Q, t, kk), y[t]);
          if (t & 1) apart();
        }
      }
      f32x4 be[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 back = *reinterpret_cast<const f32x4*>(rec.back + 16 * t + 4 * l4);
        e[t] = units ? zero4() : columns_quad(v, t, dv, n);
        // (a state that is not finite makes these NaN, where it does not reach a step too: then the chunk goes step by step)
#pragma unroll
        for (int x = 0; x < 4; ++x) e[t][x] = fmaf(-back[x], ks[t][x], e[t][x]);
        be[t] = e[t] * *reinterpret_cast<const f32x4*>(rec.beta + 16 * t + 4 * l4);
        if constexpr (!TRANSITION) y[t] *= rec.back[16 * t + l16] * r.scale;
      }
      if (chunk + 1 < last && !units)
        load_columns(gv + (s0 + C) * r.v.step, r.v.step, dv, (int)(r.seq_len - s0 - C < C ? r.seq_len - s0 - C : C), v);
      const Op<3> b[2] = {split<3>(be[0], be[1]), split<3>(be[2], be[3])};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 mb = zero4();
#pragma unroll
        for (int kk = 0; kk <= t / 2; ++kk) mb = mul<2>(at_m.rows(lds + M::MT, t, kk), b[kk], mb);
        e[t] -= mb;
        apart();
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) be[t] = e[t] * *reinterpret_cast<const f32x4*>(rec.beta + 16 * t + 4 * l4);
      u[0] = split<3>(be[0], be[1]), u[1] = split<3>(be[2], be[3]);
    }
    if constexpr (!TRANSITION) __syncthreads();
    if (mine) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int kk = 0; kk <= t / 2; ++kk) if constexpr (!TRANSITION) y[t] = mul<2>(u[kk], at_m.rows(lds + M::PT, t, kk), y[t]);
      float check = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) check = odd(e[t], odd(y[t], check));
      if (!TRANSITION && r.states != nullptr) keep_state(r.states + (pair * r.chunks + chunk) * (int64_t)pad16(dk) * dvp, dvp, pad16(dk), S);
      float* w = !TRANSITION && r.w != nullptr ? r.w + (pair * r.chunks + chunk) * (int64_t)C * dvp : nullptr;
      settle();
      if (rec.wild == 0 && __all(check == 0.f)) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int i = 16 * t + l16, c = 16 * wave + 4 * l4;
          if (!TRANSITION && i < n) {
            E* p = gy + (s0 + i) * r.y.step + c;
            if constexpr (VEC) {
              if (c < dv) store_quad<false>(p, float4{y[t][0], y[t][1], y[t][2], y[t][3]});
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (c + x < dv) p[x] = from_f32<E>(y[t][x]);
            }
          }
        }
        if (w != nullptr) keep_columns(w, dvp, e);
        // S' = keep S + sum_j into_j k_j u_j^T
        f32x4 x[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = (e[t] * *reinterpret_cast<const f32x4*>(rec.beta + 16 * t + 4 * l4)) * *reinterpret_cast<const f32x4*>(rec.into + 16 * t + 4 * l4);
        const Op<3> a[2] = {split<3>(x[0], x[1]), split<3>(x[2], x[3])};
        const float keep = rec.keep;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int z = 0; z < 4; ++z) S[m][z] *= keep;
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) S[m] = mul<2>(at.columns(lds + M::K, m, kk), a[kk], S[m]);
          if (m & 1) apart();
        }
        settle();
      } else if (TRANSITION) {
        if (lane == 0) r.wild[pair] = 1;
      } else {
        // step by step: what is not finite reaches no step before it, and none past its episode's end
        for (int i = 0; i < n; ++i) {
          const int l16 = opaque(lane & 15), l4 = opaque(lane >> 4), j = 16 * wave + l16;
          const int64_t s = s0 + i;
          const float a = gate(r, env, head, s), b = r.betas[(env * r.seq_len + s) * r.heads + head];
          float sum = 0.f;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int d = 16 * m + 4 * l4 + x;
              S[m][x] = a == 0.f ? 0.f : S[m][x] * a;
              if (d < dk) sum = fmaf(number_at<T>(lds + M::K, i, d), S[m][x], sum);
            }
          sum += __shfl_xor(sum, 16);
          sum += __shfl_xor(sum, 32);
          const float c = j < dv ? to_f32(gv[s * r.v.step + j]) - sum : 0.f;
          float out = 0.f;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int d = 16 * m + 4 * l4 + x;
              if (d < dk) {
                S[m][x] = fmaf(number_at<T>(lds + M::K, i, d), b * c, S[m][x]);
                out = fmaf(number_at<T>(lds + M::Q, i, d), S[m][x], out);
              }
            }
          out += __shfl_xor(out, 16);
          out += __shfl_xor(out, 32);
          if (l4 == 0) {
            if (j < dv) gy[s * r.y.step + j] = from_f32<E>(out * r.scale);
            if (w != nullptr) w[i * dvp + j] = c;
          }
        }
        if (w != nullptr && l4 == 0)
          for (int i = n; i < C; ++i) w[i * dvp + j] = 0.f;
      }
    }
    __syncthreads();
  }
  if constexpr (TRANSITION) {
    if (!mine) return;
    float check = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) check = odd(S[m], check);
    if (__any(check != 0.f) && lane == 0) r.wild[pair] = 1;
    const int64_t rows = pad16(dk);
    keep_state(units ? r.phi + (pair * r.segs + seg) * rows * rows : r.seg_states + (pair * r.segs + seg + 1) * rows * dvp, dvp, (int)rows, S);
    return;
  }
  if (mine && r.state_out != nullptr && last == r.chunks)
    store_state(r.state_out + eh * dk * dv, dk, dv, r.dones != nullptr && r.dones[env * r.seq_len + r.seq_len - 1] != 0.f, S);
}

// The states that enter the segments, one after the other: S' = phi S + n.  A workgroup per pair and 16 columns, a wavefront per 16 rows; the
// columns are exchanged through LDS, and the next segment's rows of phi are on their way.  A state that is not finite leaves a sum that is not
// finite in every row, where phi is 0 behind an episode's end too: such a pair is walked from the state itself.
template <int D>
__global__ __launch_bounds__(4 * D) void join_kernel(const Rule<float> r, const float* state) {
  constexpr int KK = D / 32, ROW = D + 4;
  __shared__ __align__(16) float S[2][16 * ROW];  // [column, row]
  __shared__ int wild;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, l4 = lane >> 4;
  const int64_t pair = blockIdx.x, eh = r.first_env * r.heads + pair;
  const int dk = r.dk, dv = r.dv, rows = pad16(dk), dvp = pad16(dv), j = 16 * blockIdx.y + l16, d0 = 16 * wave + 4 * l4;
  const bool mine = 16 * wave < rows;
  if (threadIdx.x == 0) wild = r.wild[pair];  // (once for all: a workgroup of other columns may write it)
  __syncthreads();
  if (wild != 0) return;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    S[0][l16 * ROW + d0 + x] = state != nullptr && d0 + x < dk && j < dv ? state[eh * dk * dv + (int64_t)(d0 + x) * dv + j] : 0.f;
  const float* phi = r.phi + pair * r.segs * (int64_t)rows * rows + (16 * wave + l16) * rows;
  float* n = r.seg_states + (pair * r.segs + 1) * (int64_t)rows * dvp + d0 * dvp + j;
  f32x4 next[KK][2], add;
  auto fetch = [&] {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int d = 32 * kk + 16 * h + 4 * l4;
        next[kk][h] = *reinterpret_cast<const f32x4*>(phi + (d < rows ? d : 0));
      }
#pragma unroll
    for (int x = 0; x < 4; ++x) add[x] = n[x * dvp];
  };
  if (mine) fetch();
  for (int s = 1; s < r.segs; ++s) {
    __syncthreads();
    const float* from = S[(s - 1) & 1];
    if (mine) {
      f32x4 acc = add;
      Op<3> a[KK];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) a[kk] = split<3>(next[kk][0], next[kk][1]);
      float* out = n;
      phi += (int64_t)rows * rows, n += (int64_t)rows * dvp;
      if (s + 1 < r.segs) fetch();
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        // (rows past the last are 0 in S, and what phi has in their place is finite)
        const f32x4 lo = *reinterpret_cast<const f32x4*>(from + l16 * ROW + 32 * kk + 4 * l4), hi = *reinterpret_cast<const f32x4*>(from + l16 * ROW + 32 * kk + 16 + 4 * l4);
        acc = mul<2>(a[kk], split<3>(lo, hi), acc);
      }
      settle();
      if (__any(odd(acc, 0.f) != 0.f) && lane == 0) r.wild[pair] = 1;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        out[x * dvp] = acc[x];
        S[s & 1][l16 * ROW + d0 + x] = acc[x];
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) S[s & 1][l16 * ROW + d0 + x] = 0.f;
    }
  }
}

// The way back: R, the gradient of the state, from the last chunk to the first.
template <class E, int D, int WAVES, bool VEC>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || kParts<E> == 1 ? 2 : 1) void backward_kernel(const Rule<E> r) {
  constexpr int MT = D / 16, KK = D / 32, N = kParts<E>;
  typedef Shared<E, D, WAVES, VEC> Sh;
  typedef typename Sh::M M;
  typedef typename M::Rows_ T;
  __shared__ __align__(16) char lds[M::BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, l4 = lane >> 4;
  const int64_t pair = blockIdx.x, env = r.first_env + pair / r.heads, eh = r.first_env * r.heads + pair;
  const int head = (int)(pair % r.heads), dk = r.dk, dv = r.dv, dvp = pad16(dv);
  const bool mine = 16 * wave < dv;
  const int j = 16 * wave + l16;
  const E* gg = r.gy.data + env * r.gy.env + head * r.gy.head;
  E* gv = r.gv.data + env * r.gv.env + head * r.gv.head;

  const At<T> at;
  const At<typename M::M> at_m;
  Sh sh;
  E g[16];
  const int64_t last = r.chunks - 1;
  sh.fetch(r, env, head, pair, last);
  if (mine) load_columns(gg + last * C * r.gy.step, r.gy.step, dv, (int)(r.seq_len - last * C), g);
  f32x4 R[MT];
  load_state(r.state ? r.state + eh * dk * dv : nullptr, dk, dv, r.dones != nullptr && r.dones[env * r.seq_len + r.seq_len - 1] != 0.f, R);

  for (int64_t chunk = last; chunk >= 0; --chunk) {
    const int64_t s0 = chunk * C;
    const int n = (int)(r.seq_len - s0 < C ? r.seq_len - s0 : C);
    sh.put(lds, dk, n);
    __syncthreads();
    if (chunk > 0) sh.fetch(r, env, head, pair, chunk - 1);
    Sh::form_p(lds, r.scale, at);
    const Record& rec = Sh::record(lds);

    f32x4 z[4];
    if (mine) {
#pragma unroll
      for (int t = 0; t < 4; ++t) z[t] = zero4();
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const Op<3> s = split<3>(R[2 * kk], R[2 * kk + 1]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          z[t] = mul<2>(at.rows(lds + M::K, t, kk), s, z[t]);
          if (t & 1) apart();
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        z[t] *= *reinterpret_cast<const f32x4*>(rec.into + 16 * t + 4 * l4);  // (NaN if R is not finite: then step by step)
      }
    }
    __syncthreads();
    if (mine) {
      f32x4 go[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) go[t] = columns_quad(g, t, dv, n);
      {
        const Op<N> a[2] = {split<N>(go[0], go[1]), split<N>(go[2], go[3])};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int kk = t / 2; kk < 2; ++kk) z[t] = mul<2>(at_m.columns(lds + M::PT, t, kk), a[kk], z[t]);
      }
      f32x4 x[4];
      {
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = z[t] * *reinterpret_cast<const f32x4*>(rec.beta + 16 * t + 4 * l4);
        const Op<3> a[2] = {split<3>(x[0], x[1]), split<3>(x[2], x[3])};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          f32x4 mb = zero4();
#pragma unroll
          for (int kk = t / 2; kk < 2; ++kk) mb = mul<2>(at_m.columns(lds + M::MT, t, kk), a[kk], mb);
          z[t] -= mb;
          apart();
        }
      }
      // the state's gradient before the chunk
      f32x4 next[MT];
      f32x4 dvs[4];
      {
        f32x4 bg[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const f32x4 back = *reinterpret_cast<const f32x4*>(rec.back + 16 * t + 4 * l4);
          dvs[t] = z[t] * *reinterpret_cast<const f32x4*>(rec.beta + 16 * t + 4 * l4);
          x[t] = -(back * dvs[t]), bg[t] = (back * r.scale) * go[t];
        }
        const Op<3> a[2] = {split<3>(x[0], x[1]), split<3>(x[2], x[3])}, b[2] = {split<3>(bg[0], bg[1]), split<3>(bg[2], bg[3])};
        const float keep = rec.keep;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int i = 0; i < 4; ++i) next[m][i] = R[m][i] * keep;
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            next[m] = mul<2>(at.columns(lds + M::K, m, kk), a[kk], next[m]);
            next[m] = mul<2>(at.columns(lds + M::Q, m, kk), b[kk], next[m]);
          }
          apart();
        }
      }
      if (r.dstates != nullptr) keep_state(r.dstates + (pair * r.chunks + chunk) * (int64_t)pad16(dk) * dvp, dvp, pad16(dk), R);
      float* gz = r.z + (pair * r.chunks + chunk) * (int64_t)C * dvp;
      float check = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) check = odd(z[t], check);
#pragma unroll
      for (int m = 0; m < MT; ++m) check = odd(next[m], check);
      settle();
      if (rec.wild == 0 && __all(check == 0.f)) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int s = 16 * t + 4 * l4 + i;
            if (r.gv.data != nullptr && s < n && j < dv) gv[(s0 + s) * r.gv.step + j] = from_f32<E>(dvs[t][i]);
          }
        keep_columns(gz, dvp, z);
#pragma unroll
        for (int m = 0; m < MT; ++m) R[m] = next[m];
      } else {
        for (int i = n - 1; i >= 0; --i) {
          const int l16 = opaque(lane & 15), l4 = opaque(lane >> 4), j = 16 * wave + l16;
          const int64_t s = s0 + i;
          const float a = gate(r, env, head, s), b = r.betas[(env * r.seq_len + s) * r.heads + head];
          const float up = j < dv ? r.scale * to_f32(gg[s * r.gy.step + j]) : 0.f;
          float sum = 0.f;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int d = 16 * m + 4 * l4 + x;
              if (d < dk) {
                R[m][x] = fmaf(number_at<T>(lds + M::Q, i, d), up, R[m][x]);
                sum = fmaf(number_at<T>(lds + M::K, i, d), R[m][x], sum);
              }
            }
          sum += __shfl_xor(sum, 16);
          sum += __shfl_xor(sum, 32);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int d = 16 * m + 4 * l4 + x;
              if (d < dk) R[m][x] = fmaf(number_at<T>(lds + M::K, i, d), -b * sum, R[m][x]);
              R[m][x] = a == 0.f ? 0.f : R[m][x] * a;
            }
          if (l4 == 0) {
            gz[i * dvp + j] = sum;
            if (r.gv.data != nullptr && j < dv) gv[s * r.gv.step + j] = from_f32<E>(b * sum);
          }
        }
        if (l4 == 0)
          for (int i = n; i < C; ++i) gz[i * dvp + j] = 0.f;
      }
    }
    __syncthreads();
    if (mine && chunk > 0) load_columns(gg + (s0 - C) * r.gy.step, r.gy.step, dv, C, g);
  }
  if (mine && r.state_out != nullptr) store_state(r.state_out + eh * dk * dv, dk, dv, false, R);
}

}  // namespace

// f(dims of the keys in whole tiles, wavefronts): of the values' 64 or 128 columns, a wavefront for 16; keys of over 64 elements always have 8,
// which share their loads and hold a segment's as many unit vectors.
template <class F>
void by_dims(int dk, int dv, F f) {
  typedef std::integral_constant<int, 64> D64;
  typedef std::integral_constant<int, 128> D128;
  typedef std::integral_constant<int, 4> Four_;
  typedef std::integral_constant<int, 8> Eight;
  if (dk > 64) f(D128{}, Eight{});
  else if (dv > 64) f(D64{}, Eight{});
  else f(D64{}, Four_{});
}
template <class E>
int launch_forward(const Rule<E>& r, int64_t envs, hipStream_t s) {
  const unsigned pairs = (unsigned)(envs * r.heads);
  const bool vec = fours(r.k, r.dk) && fours(r.q, r.dk) && fours(r.y, r.dv);
  by_dims(r.dk, r.dv, [&](auto d, auto waves) {
    constexpr int D = decltype(d)::value, W = decltype(waves)::value;
    if (r.segs > 1) {
      const dim3 grid(pairs, (unsigned)r.segs - 1, 2);
      if (vec) forward_kernel<E, D, W, true, true><<<grid, dim3(64 * W), 0, s>>>(r);
      else forward_kernel<E, D, W, false, true><<<grid, dim3(64 * W), 0, s>>>(r);
      Rule<float> j = {};
      j.first_env = r.first_env, j.heads = r.heads, j.dk = r.dk, j.dv = r.dv, j.segs = r.segs, j.phi = r.phi, j.seg_states = r.seg_states, j.wild = r.wild;
      join_kernel<D><<<dim3(pairs, (unsigned)pad16(r.dv) / 16), dim3(4 * D), 0, s>>>(j, r.state);
    }
    const dim3 grid(pairs, (unsigned)r.segs);
    if (vec) forward_kernel<E, D, W, true, false><<<grid, dim3(64 * W), 0, s>>>(r);
    else forward_kernel<E, D, W, false, false><<<grid, dim3(64 * W), 0, s>>>(r);
  });
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}
template <class E>
int launch_backward(const Rule<E>& r, int64_t envs, hipStream_t s) {
  const dim3 grid((unsigned)(envs * r.heads));
  const bool vec = fours(r.k, r.dk) && fours(r.q, r.dk);
  by_dims(r.dk, r.dv, [&](auto d, auto waves) {
    constexpr int D = decltype(d)::value, W = decltype(waves)::value;
    if (vec) backward_kernel<E, D, W, true><<<grid, dim3(64 * W), 0, s>>>(r);
    else backward_kernel<E, D, W, false><<<grid, dim3(64 * W), 0, s>>>(r);
  });
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}
template int launch_forward<bf16>(const Rule<bf16>&, int64_t, hipStream_t);
template int launch_forward<float>(const Rule<float>&, int64_t, hipStream_t);
template int launch_backward<bf16>(const Rule<bf16>&, int64_t, hipStream_t);
template int launch_backward<float>(const Rule<float>&, int64_t, hipStream_t);

}  // namespace delta
}  // namespace rlk
