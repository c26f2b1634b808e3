// rlk_delta_gradients.hip -- the gated delta rule: gradients of queries, keys, gates and betas, all chunks at once, from what the two walks
// have left (rlk_delta.hpp): states S before the chunk, gradients R of the states after it, the corrections w and z.
//
// With u = b w, dv = b z, Y1_ij = scale D_ij G_i . u_j (i >= j) and Y2_ij = -D_ij dv_i . u_j (i > j):
//   dq_i = scale back_i S G_i + sum_j Y1_ij k_j
//   dk_i = dk+ + dk-,   dk+_i = -back_i S dv_i + sum_j Y2_ij k_j,   dk-_j = into_j R u_j + sum_i (Y1_ij q_i + Y2_ij k_i)
//   db_i = z_i . w_i
// A gate's gradient is the sum of every term that its factor is in: with W_ij = Y1_ij q_i . k_j + Y2_ij k_i . k_j, which has the gates from j + 1 to i,
//   dg_t = keep R . S + sum_{i >= t} back_i (scale q_i . S G_i - k_i . S dv_i) + sum_{j < t} into_j k_j . R u_j + sum_{i >= t > j} W_ij.
// Nothing is taken off again, so the gradient of a gate that leaves little of the state is as exact as its terms, which are as small.  (As a sum from the
// end, of each W_ij added at i and taken away at j, it was a difference of numbers up to exp(-g) times its size: nothing was left of it from
// g = -16 on.)  The last sum by tiles of 16 steps: a tile's sums by rows (i) and by columns (j), and what one on the diagonal gives for each t.
//
// A workgroup per chunk, a wavefront per 16 rows of the state.  The sums over the state's columns go 64 columns at a time, G, u and dv in LDS;
// then keys, queries and both Y take their place.
//
// [64,1024,8,64+64] bf16 390 us, 2.2 TB/s of 104 KB a chunk.  Bound by waits, half of a wavefront's time, with two workgroups a CU: vector units
// issue for 42% of it, matrix units for 16, LDS conflicts take 27.  The gates' sums are 27 more than one sum from the end was.  Slices of 32
// columns and three workgroups a CU: 439 against 361 then, registers spilled; keys and queries fetched with the first arrays: as before;
// workgroups that go from chunk to chunk with the next one's arrays on their way: 360 bytes a lane spilled.
#include "rlk_delta.hpp"

namespace rlk {
namespace delta {
namespace {

template <class E, int D>
struct Lds {
  typedef Tile<E, 64> G;
  typedef Tile<float, 64> U;
  typedef Tile<E, D> K;
  typedef Tri<3> Y;
  static constexpr int UT = G::BYTES, DT = UT + U::BYTES, FIRST = DT + U::BYTES;
  static constexpr int QT = K::BYTES, Y1 = 2 * K::BYTES, Y2 = Y1 + Y::BYTES, SECOND = Y2 + Y::BYTES;
  static constexpr int BYTES = FIRST > SECOND ? FIRST : SECOND;
};

// 64 columns from c0 on of a chunk's rows of w or z, each row times its beta, as parts in a tile.
template <int NT>
struct Corrections {
  static constexpr int PER = C * 16 / NT;
  f32x4 x[PER];
  __device__ void fetch(const float* p, int c0, int dvp) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + NT * i, c = c0 + u % 16 * 4;
      x[i] = c < dvp ? *reinterpret_cast<const f32x4*>(p + u / 16 * dvp + c) : zero4();
    }
  }
  __device__ void put(char* tile, const float* beta) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + NT * i;
      Four<float>{x[i] * beta[u / 16]}.put(tile + Tile<float, 64>::row(u / 16) + u % 16 * 8, Tile<float, 64>::PART);
    }
  }
};

// Of a quarter's 16 lanes: the value of the lane N further on (UP: or before), 0 past the quarter's end.  All lanes have to take part.
template <int N, bool UP>
__device__ __forceinline__ float beside(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), (UP ? 0x110 : 0x100) + N, 0xf, 0xf, true));
}
// The sum over these lanes from the first (UP) or the last one to this one.
template <bool UP>
__device__ __forceinline__ float added_up(float x) {
  x += beside<1, UP>(x);
  x += beside<2, UP>(x);
  x += beside<4, UP>(x);
  x += beside<8, UP>(x);
  return x;
}
// x of the two quarters 0 + 1 and 2 + 3, and y's between them: (x, y, x, y) by quarters.
__device__ __forceinline__ float by_twos(float x, float y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// ... of the two halves: x in the lower one, y in the upper one.
__device__ __forceinline__ float by_halves(float x, float y) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float of_lane(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }

template <class E, int D, bool VEC>
__global__ __launch_bounds__(4 * D, D == 128 || kParts<E> == 1 ? 2 : 1) void gradients_kernel(const Rule<E> r) {
  constexpr int NT = 4 * D, WAVES = D / 16, N = kParts<E>;
  typedef Lds<E, D> M;
  typedef typename M::K T;
  __shared__ __align__(16) char lds[M::BYTES];
  __shared__ float kept_sums[WAVES];
  __shared__ int found[WAVES];
  constexpr int REST_QUADS = (int)(sizeof(Record) - offsetof(Record, ghi)) / 16;
  __shared__ f32x4 rest_of_record[REST_QUADS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, l4 = lane >> 4;
  const int64_t at = blockIdx.x, pair = at / r.chunks, chunk = at - pair * r.chunks, s0 = chunk * C;
  const int64_t env = r.first_env + pair / r.heads;
  const int head = (int)(pair % r.heads), dk = r.dk, dv = r.dv, dvp = pad16(dv);
  const int n = (int)(r.seq_len - s0 < C ? r.seq_len - s0 : C);
  const Record& rec = *reinterpret_cast<const Record*>(reinterpret_cast<const char*>(rest_of_record) - offsetof(Record, ghi));  // (in LDS, without M)

  // all of the first loads together
  const bool mine = 16 * wave < dk;
  const float *w = r.w + at * C * dvp, *z = r.z + at * C * dvp;
  const int64_t state = at * pad16(dk) * dvp + (int64_t)(16 * wave + l16) * dvp;
  Corrections<NT> ws, zs;
  Rows<E, 64, NT, VEC> gs;
  const E* gg = r.gy.data + env * r.gy.env + head * r.gy.head + s0 * r.gy.step;
  f32x4 sq[2][2], rq[2][2];  // 64 columns of the wavefront's rows of S and R
  auto fetch = [&](int c0) {
    gs.fetch(gg + c0, r.gy.step, dv - c0, n);
    ws.fetch(w, c0, dvp);
    zs.fetch(z, c0, dvp);
    if (mine)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = c0 + 32 * kk + 16 * h + 4 * l4, cc = c < dvp ? c : 0;
          sq[kk][h] = *reinterpret_cast<const f32x4*>(r.states + state + cc);
          rq[kk][h] = *reinterpret_cast<const f32x4*>(r.dstates + state + cc);
        }
  };
  if (threadIdx.x < REST_QUADS) rest_of_record[threadIdx.x] = reinterpret_cast<const f32x4*>(r.records[at].ghi)[threadIdx.x];
  fetch(0);
  Rows<E, D, NT, VEC> k, q;
  const At<typename M::G> at_g;
  const At<typename M::U> at_u;
  const At<T> at_k;
  const At<typename M::Y> at_y;

  // transposed results: step 16 t + l16, dims 16 wave + 4 l4 + 0..3
  f32x4 dq[4], up[4], down[4];  // (up, down: dk+ and dk-)
#pragma unroll
  for (int t = 0; t < 4; ++t) dq[t] = up[t] = down[t] = zero4();
  // Y1 and Y2: transposed too, steps i = 16 ti + l16, j = 16 tj + 4 l4 + 0..3.  A wavefront has rows of one of them: of 4 wavefronts two have
  // rows 3 and 0, two 2 and 1, 5 tiles each; of 8 each has one row.
  constexpr int ROWS = WAVES == 4 ? 2 : 1, TILES = WAVES == 4 ? 5 : 4;
  const bool second = wave & 1;
  const int row_a = ROWS == 2 ? 3 - (wave >> 1) : wave >> 1, row_b = wave >> 1;
  auto tile_of = [&](int slot, int& ti, int& tj) {  // whether there is one
    ti = ROWS == 2 && slot > row_a ? row_b : row_a, tj = ROWS == 2 && slot > row_a ? slot - row_a - 1 : slot;
    return tj <= ti;
  };
  f32x4 ya[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) ya[t] = zero4();
  float kept = 0.f;
  constexpr int PER = Corrections<NT>::PER;
  static_assert(PER <= 4);
  float db[PER];  // (of the steps of this thread's parts of w and z)
#pragma unroll
  for (int i = 0; i < PER; ++i) db[i] = 0.f;

  __syncthreads();  // the record is there
  const uint64_t cuts = rec.cuts[0] | (uint64_t)rec.cuts[1] << 32;
  for (int c0 = 0; c0 < dv; c0 += 64) {
    if (c0 > 0) __syncthreads();
    gs.put(lds, dv - c0, 0, n);
    ws.put(lds + M::UT, rec.beta);
    zs.put(lds + M::DT, rec.beta);
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) db[i] = fmaf(ws.x[i][x], zs.x[i][x], db[i]);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      if (c0 + 32 * kk >= dv) continue;
#pragma unroll
      for (int slot = 0; slot < TILES; ++slot) {
        int ti, tj;
        if (!tile_of(slot, ti, tj)) continue;
        const Op<3> u = at_u.rows(lds + M::UT, tj, kk);
        if (second) ya[slot] = mul<2>(u, at_u.rows(lds + M::DT, ti, kk), ya[slot]);
        else ya[slot] = mul<2>(u, at_g.rows(lds, ti, kk), ya[slot]);
      }
      settle();
      if (mine) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (c0 + 32 * kk + 16 * h + 4 * l4 >= dvp) sq[kk][h] = rq[kk][h] = zero4();
#pragma unroll
          for (int x = 0; x < 4; ++x) kept = fmaf(sq[kk][h][x], rq[kk][h][x], kept);
        }
        const Op<3> s = split<3>(sq[kk][0], sq[kk][1]), rr = split<3>(rq[kk][0], rq[kk][1]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          dq[t] = mul<2>(s, at_g.rows(lds, t, kk), dq[t]);
          up[t] = mul<2>(s, at_u.rows(lds + M::DT, t, kk), up[t]);
          down[t] = mul<2>(rr, at_u.rows(lds + M::UT, t, kk), down[t]);
          apart();
        }
      }
      settle();
    }
    if (c0 + 64 < dv) fetch(c0 + 64);
  }
  k.fetch(r.k.data + env * r.k.env + head * r.k.head + s0 * r.k.step, r.k.step, dk, n);
  q.fetch(r.q.data + env * r.q.env + head * r.q.head + s0 * r.q.step, r.q.step, dk, n);
  // db: a row's 16 parts
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    float x = db[i];
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d);
    const int row = (threadIdx.x + NT * i) / 16;
    if (l16 == 0 && row < n && r.gb != nullptr) r.gb[(env * r.seq_len + s0 + row) * r.heads + head] = x;
  }
  const float keep = rec.keep;
  kept = keep != 0.f ? kept * keep : 0.f;
  float back[4], into[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    back[t] = rec.back[16 * t + l16], into[t] = rec.into[16 * t + l16];
    // (what does not reach a step has no part, NaN included)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      dq[t][x] = back[t] != 0.f ? dq[t][x] * (back[t] * r.scale) : 0.f;
      up[t][x] = back[t] != 0.f ? -up[t][x] * back[t] : 0.f;
      down[t][x] = into[t] != 0.f ? down[t][x] * into[t] : 0.f;
    }
  }
  {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < Rows<E, D, NT, VEC>::PER; ++i) {
      const f32x4 a = k.x[i].floats(), b = q.x[i].floats();
#pragma unroll
      for (int x = 0; x < 4; ++x) sum = fmaf(0.f, a[x], fmaf(0.f, b[x], sum));
    }
    const bool any = __any(sum != 0.f);
    if (lane == 0) found[wave] = any;
  }
  __syncthreads();  // all have read the first arrays
#pragma unroll
  for (int slot = 0; slot < TILES; ++slot) {
    int ti, tj;
    if (!tile_of(slot, ti, tj)) continue;
    const int i = 16 * ti + l16;
    const uint64_t before = cuts & (((uint64_t)2 << i) - 1);
    const int begin = before != 0 ? 63 - __clzll((long long)before) : 0;
    const float hi = rec.ghi[i], lo = rec.glo[i];
    const f32x4 hj = *reinterpret_cast<const f32x4*>(rec.ghi + 16 * tj + 4 * l4), lj = *reinterpret_cast<const f32x4*>(rec.glo + 16 * tj + 4 * l4);
    f32x4 a = ya[slot];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = 16 * tj + 4 * l4 + e;
      const float d = __expf((hi - hj[e]) + (lo - lj[e]));
      a[e] = j >= begin && (second ? j < i : j <= i) ? a[e] * (second ? -d : d * r.scale) : 0.f;
    }
    ya[slot] = a;
    char* y = lds + (second ? M::Y2 : M::Y1);
    const int first = M::Y::row(16 * ti), stride = ti < 2 ? M::Y::row(1) : M::Y::row(33) - M::Y::row(32);
    Four<float>{a}.put(y + first + l16 * stride + 2 * (16 * tj + 4 * l4), M::Y::PART);
    if (tj == ti && (ti & 1) == 0)  // the tile above the diagonal that products go over
      Four<float>{zero4()}.put(y + first + l16 * stride + 2 * (16 * tj + 16 + 4 * l4), M::Y::PART);
  }
  // Where the gates' sums are kept: the record's gates have had their use, and there are 16 bytes behind each of Y's rows.  Of W's tiles, of Y1 and
  // of Y2, the sums of their rows (on the diagonal: what a tile gives for each step) and of their columns; a wavefront's sums of a step.
  float* by_row = reinterpret_cast<float*>(rest_of_record);
  static_assert(320 * sizeof(float) <= offsetof(Record, keep) - offsetof(Record, ghi));
  auto behind = [&](int y, int part, int i) { return lds + y + part * M::Y::PART + M::Y::row(i) + (i < 32 ? 64 : 128); };
  auto by_column = [&](bool y2, int tile, int quarter) { return reinterpret_cast<f32x4*>(behind(y2 ? M::Y2 : M::Y1, 2, 4 * tile + quarter)); };
  auto of_step = [&](int y, int w, int i) { return reinterpret_cast<float*>(behind(y, w >> 2, i)) + (w & 3); };
  k.put(lds, dk, 0, n);
  q.put(lds + M::QT, dk, 0, n);
  __syncthreads();
  if (r.gg != nullptr) {
    const char* rows_i = lds + (second ? 0 : M::QT);
    f32x4 qk[TILES];  // or k . k
#pragma unroll
    for (int slot = 0; slot < TILES; ++slot) qk[slot] = zero4();
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      if (32 * kk >= dk) continue;
#pragma unroll
      for (int slot = 0; slot < TILES; ++slot) {
        int ti, tj;
        if (tile_of(slot, ti, tj)) qk[slot] = mul<2>(at_k.rows(lds, tj, kk), at_k.rows(rows_i, ti, kk), qk[slot]);
      }
    }
    settle();
#pragma unroll
    for (int slot = 0; slot < TILES; ++slot) {
      int ti, tj;
      if (!tile_of(slot, ti, tj)) continue;
      const int i = 16 * ti + l16;
      f32x4 later;  // sums over the tile's rows from i on
      float row = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 16 * tj + 4 * l4 + e;
        // (Y is 0 between episodes, where q . k may be anything)
        const float y = ya[slot][e], w = y != 0.f && j < i ? y * qk[slot][e] : 0.f;
        row += w;
        later[e] = added_up<false>(w);
      }
      if (ti == tj) {
        row = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) row += 4 * l4 + e < l16 ? later[e] : 0.f;
      }
      row = by_twos(row, row);
      row = by_halves(row, row);
      const int tile = ti * (ti + 1) / 2 + tj;
      if (l4 == 0) by_row[160 * second + 16 * tile + l16] = row;
      if (l16 == 0) *by_column(second, tile, l4) = later;
    }
    if (mine) {
      // what the state before the chunk gives to a step, and what a step gives to the one after it
      float given[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = 16 * t + l16;
        const f32x4 q4 = numbers_at<T>(lds + M::QT, i, 16 * wave + 4 * l4), k4 = numbers_at<T>(lds, i, 16 * wave + 4 * l4);
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x = fmaf(q4[e], dq[t][e], fmaf(k4[e], up[t][e], x)), y = fmaf(k4[e], down[t][e], y);
        given[t] = by_twos(back[t] != 0.f ? x : 0.f, into[t] != 0.f ? y : 0.f);
      }
#pragma unroll
      for (int t = 0; t < 4; t += 2) {
        const int i = 16 * (t + (l4 >> 1)) + l16;
        const float x = by_halves(given[t], given[t + 1]);  // (x, y of t, x, y of t + 1)
        *of_step(l4 & 1 ? M::Y1 : M::Y2, wave, i) = x;
      }
    }
  }
  // Keys and queries that are not finite would reach other episodes as 0 inf: then an episode at a time.
  bool wild = false;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) wild |= found[i] != 0;
  for (int from = 0, to; from < n; from = to) {
    to = n;
    if (wild) {
      const uint64_t later = cuts & ~(((uint64_t)2 << from) - 1);
      to = later != 0 ? __ffsll((long long)later) - 1 : n;
      __syncthreads();
      k.put(lds, dk, from, to);
      q.put(lds + M::QT, dk, from, to);
      __syncthreads();
    }
    if (mine) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 a = dq[t], b = up[t], c = down[t];
        const int i = 16 * t + l16;
        const bool inside = i >= from && i < to;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const Op<N> kc = at_k.columns(lds, wave, kk), qc = at_k.columns(lds + M::QT, wave, kk);
          if (kk <= t / 2) {
            a = mul<2>(kc, at_y.rows(lds + M::Y1, t, kk), a);
            b = mul<2>(kc, at_y.rows(lds + M::Y2, t, kk), b);
          }
          if (kk >= t / 2) {
            c = mul<2>(qc, at_y.columns(lds + M::Y1, t, kk), c);
            c = mul<2>(kc, at_y.columns(lds + M::Y2, t, kk), c);
          }
        }
        settle();
        if (inside) dq[t] = a, up[t] = b, down[t] = c;
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) kept += __shfl_xor(kept, d);
  if (lane == 0) kept_sums[wave] = kept;
  __syncthreads();
  if (mine) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int i = 16 * t + l16, d = 16 * wave + 4 * l4;
      if (i >= n) continue;
      const f32x4 x = up[t] + down[t];
      const int64_t s = s0 + i;
      E* pq = r.gq.data != nullptr ? r.gq.data + env * r.gq.env + s * r.gq.step + head * r.gq.head + d : nullptr;
      E* pk = r.gk.data != nullptr ? r.gk.data + env * r.gk.env + s * r.gk.step + head * r.gk.head + d : nullptr;
      if constexpr (VEC) {
        if (d < dk) {
          if (pq != nullptr) store_quad<false>(pq, float4{dq[t][0], dq[t][1], dq[t][2], dq[t][3]});
          if (pk != nullptr) store_quad<false>(pk, float4{x[0], x[1], x[2], x[3]});
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < dk) {
            if (pq != nullptr) pq[e] = from_f32<E>(dq[t][e]);
            if (pk != nullptr) pk[e] = from_f32<E>(x[e]);
          }
      }
    }
  }
  if (wave == 0 && r.gg != nullptr) {
    const int used = (dk + 15) / 16, T = lane >> 4;
    float x = 0.f, before = 0.f, all = 0.f;  // of the steps from here on, of those before, of the whole chunk
    for (int i = 0; i < used; ++i) {
      if (lane < n) x += *of_step(M::Y2, i, lane), before += *of_step(M::Y1, i, lane);
      all += kept_sums[i];
    }
    // W's tiles in this step's rows, in its columns, and those that lie beyond it both ways
    float rows = 0.f, columns = 0.f, beyond = 0.f;
#pragma unroll
    for (int ti = 0; ti < 4; ++ti)
#pragma unroll
      for (int tj = 0; tj <= ti; ++tj) {
        const int tile = ti * (ti + 1) / 2 + tj;
        const float f = by_row[16 * tile + l16] + by_row[160 + 16 * tile + l16];
        if (ti == tj) {
          all += T == ti ? f : 0.f;
        } else {
          rows += T == ti ? f : 0.f;
          beyond += tj < T && T < ti ? f : 0.f;
          const int at = l16 & 3;
          columns += T == tj ? reinterpret_cast<const float*>(by_column(false, tile, l16 >> 2))[at] + reinterpret_cast<const float*>(by_column(true, tile, l16 >> 2))[at] : 0.f;
        }
      }
    // (each of these sums has terms of this gate alone, so nothing that is not finite comes in from another episode)
    x = added_up<false>(x), rows = added_up<false>(rows), beyond = added_up<false>(beyond);
    before = added_up<true>(before), columns = added_up<true>(columns);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float later = of_lane(x, 16 * t), earlier = of_lane(before, 16 * t + 15), past = of_lane(beyond, 16 * t);
      all += (t > T ? later : 0.f) + (t < T ? earlier : 0.f) + (t == T ? past : 0.f);
    }
    all += (x + rows) + beside<1, true>(before + columns);
    const float g = (cuts >> lane) & 1 || (r.from_zero && s0 + lane == 0) ? 0.f : all;
    if (lane < n) r.gg[(env * r.seq_len + s0 + lane) * r.heads + head] = g;
  }
}

}  // namespace

template <class E>
int launch_gradients(const Rule<E>& r, int64_t envs, hipStream_t s) {
  const dim3 grid((unsigned)(envs * r.heads * r.chunks));
  const bool vec = fours(r.k, r.dk) && fours(r.q, r.dk) && fours(r.gy, r.dv) && fours(r.gq, r.dk) && fours(r.gk, r.dk);
  // (longer values of short keys: the second 4 wavefronts have no rows of the state, but their part of Y and the loads; [37,333,4,40+72] float32
  // 86 us, 98 by 4)
  if (r.dk <= 64 && r.dv <= 64) {
    if (vec) gradients_kernel<E, 64, true><<<grid, dim3(256), 0, s>>>(r);
    else gradients_kernel<E, 64, false><<<grid, dim3(256), 0, s>>>(r);
  } else {
    if (vec) gradients_kernel<E, 128, true><<<grid, dim3(512), 0, s>>>(r);
    else gradients_kernel<E, 128, false><<<grid, dim3(512), 0, s>>>(r);
  }
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}
template int launch_gradients<bf16>(const Rule<bf16>&, int64_t, hipStream_t);
template int launch_gradients<float>(const Rule<float>&, int64_t, hipStream_t);

}  // namespace delta
}  // namespace rlk
