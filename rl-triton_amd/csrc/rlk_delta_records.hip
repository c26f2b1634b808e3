// rlk_delta_records.hip -- the gated delta rule: a record for every chunk (rlk_delta.hpp), all chunks at once.
//
// A wavefront per chunk.  k_i . k_j comes from the matrix instructions with the keys read straight into operands; then, in LDS and float32,
// M = (1 + L b)^-1 L: its four diagonal blocks of 16 by substitution, a lane per column (m_i = L_i - sum_{j < i} L_ij b_j m_j), and what is
// below them from halves, M_21 = (1 - M_22 b) L_21 (1 - b M_11), for blocks of 16 and then of 32, by float32 matrix products.
// Gates are added up in float64: D is a quotient of their sums' exponentials, and a head that forgets fast has large sums.
//
// Bound by the steps of a substitution after each other, 3 workgroups a CU: [64,1024,8,64] bf16 55 us (2.9 TB/s of keys in and records out; 66 with
// two workgroups a CU), [1,16384,16,128] 40 us.
#include "rlk_delta.hpp"

namespace rlk {
namespace delta {
namespace {

constexpr int kWaves = 4;
// Floats of a row of L in LDS, for its 16, 32 or 64 columns: 16 rows of 4 columns reach all banks, and a CU holds three workgroups.
__device__ __forceinline__ constexpr int row_floats(int tile) { return tile == 0 ? 20 : tile == 1 ? 36 : 68; }
__device__ __forceinline__ constexpr int row_at(int tile) { return tile == 0 ? 0 : 16 * 20 + (tile == 1 ? 0 : 16 * 36 + (tile - 2) * 16 * 68); }
constexpr int LFLOATS = 16 * (20 + 36 + 68 + 68);

// acc + a b for 16x16 blocks: a's rows from LDS, b as a result lies in a lane.
__device__ __forceinline__ f32x4 block_mma(f32x4 a, f32x4 b, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
  return acc;
}

template <class E, bool VEC>
__global__ __launch_bounds__(64 * kWaves) void records_kernel(const Rule<E> r, int64_t count) {
  __shared__ __align__(16) float lds[kWaves][LFLOATS + 3 * C];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, l4 = lane >> 4;
  const int64_t at = (int64_t)blockIdx.x * kWaves + wave;
  if (at >= count) return;  // (no barrier below: a wavefront has its own part of LDS)
  float *L = lds[wave], *ghi = L + LFLOATS, *glo = ghi + C, *beta = glo + C;
  const int64_t pair = at / r.chunks, chunk = at - pair * r.chunks;
  const int64_t env = r.first_env + pair / r.heads, T = r.seq_len, s0 = chunk * C;
  const int head = (int)(pair % r.heads), n = (int)(T - s0 < C ? T - s0 : C);
  Record& rec = r.records[at];
  bool wild = false;
  if (r.wild != nullptr && chunk == 0 && lane == 0) r.wild[pair] = 0;

  // gates and betas, a step per lane
  uint64_t cuts;
  {
    const int64_t s = s0 + (lane < n ? lane : n - 1), place = (env * T + s) * r.heads + head;
    float g = r.gates != nullptr ? r.gates[place] : 0.f, b = r.betas[place];
    const bool done = r.dones != nullptr && s > 0 && r.dones[env * T + s - 1] != 0.f;
    if (lane >= n) g = 0.f, b = 0.f;
    const bool cut = lane < n && (done || g <= kNoDecay);
    cuts = __ballot(cut);
    wild = (!cut && !finite(g)) || !finite(b);
    // sums from where the episode begins (nothing of a gate that is not finite reaches another one)
    double sum = cut ? 0.0 : (double)g;
    const uint64_t upto = cuts & (((uint64_t)2 << lane) - 1);
    const int begin = upto != 0 ? 63 - __clzll((long long)upto) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double before = __shfl_up(sum, d);
      if (lane - d >= begin) sum += before;
    }
    const double all = __shfl(sum, 63);
    const float hi = rintf((float)sum * 1024.f) * (1.f / 1024.f), lo = (float)(sum - (double)hi);
    const int first = cuts != 0 ? __ffsll((long long)cuts) - 1 : C, last = cuts != 0 ? 63 - __clzll((long long)cuts) : 0;
    ghi[lane] = hi, glo[lane] = lo, beta[lane] = b;
    rec.ghi[lane] = hi, rec.glo[lane] = lo, rec.beta[lane] = b;
    rec.back[lane] = lane < first ? expf((float)sum) : 0.f;
    rec.into[lane] = lane >= last && lane < n ? expf((float)(all - sum)) : 0.f;
    if (lane == 0) {
      rec.keep = cuts != 0 ? 0.f : expf((float)all);
      rec.cuts[0] = (uint32_t)cuts, rec.cuts[1] = (uint32_t)(cuts >> 32);
    }
  }

  // k_i . k_j: tiles of rows i, columns j <= i
  f32x4 acc[10];
#pragma unroll
  for (int t = 0; t < 10; ++t) acc[t] = zero4();
  const E* keys = r.k.data + env * r.k.env + head * r.k.head + s0 * r.k.step;
  for (int d0 = 0; d0 < r.dk; d0 += 32) {
    Op<kParts<E>> f[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = 16 * t + l16;
      const E* p = keys + (row < n ? row : n - 1) * r.k.step;
      Four<E> a = four<E, VEC>(p, d0 + 8 * l4, r.dk), b = four<E, VEC>(p, d0 + 8 * l4 + 4, r.dk);
      clip<E, VEC>(a, d0 + 8 * l4, r.dk, row < n);
      clip<E, VEC>(b, d0 + 8 * l4 + 4, r.dk, row < n);
      if constexpr (kParts<E> == 1) {
        union { u32x2 h[2]; bf16x8 v; } u;
        u.h[0] = a.w, u.h[1] = b.w;
        f[t].p[0] = u.v;
      } else {
        f[t] = split<3>(a.w, b.w);
      }
    }
#pragma unroll
    for (int ti = 0; ti < 4; ++ti)
#pragma unroll
      for (int tj = 0; tj <= ti; ++tj) acc[ti * (ti + 1) / 2 + tj] = mul<2>(f[ti], f[tj], acc[ti * (ti + 1) / 2 + tj]);
  }
  settle();
  wave_sync();

  // L, strictly lower, to LDS; what lies above the diagonal of its diagonal blocks is 0
#pragma unroll
  for (int ti = 0; ti < 4; ++ti) {
#pragma unroll
    for (int tj = 0; tj <= ti; ++tj) {
      const f32x4 x = acc[ti * (ti + 1) / 2 + tj];
      const int j = 16 * tj + l16;
      const float hj = ghi[j], lj = glo[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 16 * ti + 4 * l4 + e;
        wild |= !finite(x[e]);
        // no episode begins in (j, i]
        const uint64_t between = (cuts >> j >> 1) << 1 << j & (((uint64_t)2 << i) - 1);
        L[row_at(ti) + (4 * l4 + e) * row_floats(ti) + j] = i > j && between == 0 ? x[e] * __expf((ghi[i] - hj) + (glo[i] - lj)) : 0.f;
      }
    }
  }
  wave_sync();

  // diagonal blocks: lane (block l4, column l16)
  {
    float* block = L + row_at(l4) + 16 * l4;
    const int row = row_floats(l4);
    const float* b = beta + 16 * l4;
    float m[16], bm[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      m[i] = block[i * row + l16];
#pragma unroll
      for (int j = 0; j < i; ++j) m[i] = fmaf(-block[i * row + j], bm[j], m[i]);
      bm[i] = b[i] * m[i];
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < 16; ++i) block[i * row + l16] = m[i];
  }
  wave_sync();

  // a block's rows as the left factor, a block as a result lies in a lane (the right factor or a sum)
  auto left = [&](int ti, int tj) { return *reinterpret_cast<const f32x4*>(L + row_at(ti) + l16 * row_floats(ti) + 16 * tj + 4 * l4); };
  auto result = [&](int ti, int tj) {
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = L[row_at(ti) + (4 * l4 + e) * row_floats(ti) + 16 * tj + l16];
    return x;
  };
  auto betas = [&](int t) { return *reinterpret_cast<const f32x4*>(beta + 16 * t + 4 * l4); };  // (of columns of a left factor, of rows of a right one)
  auto put = [&](int ti, int tj, f32x4 x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) L[row_at(ti) + (4 * l4 + e) * row_floats(ti) + 16 * tj + l16] = x[e];
  };
#pragma unroll
  for (int h = 0; h < 4; h += 2) {
    f32x4 x = block_mma(left(h + 1, h), -(betas(h) * result(h, h)), result(h + 1, h));
    x = block_mma(-(left(h + 1, h + 1) * betas(h + 1)), x, x);
    settle();
    wave_sync();
    put(h + 1, h, x);
  }
  wave_sync();
  {
    f32x4 x[2][2];  // L_21 (1 - b M_11), then M_21
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[i][j] = result(2 + i, j);
#pragma unroll
        for (int k = j; k < 2; ++k) x[i][j] = block_mma(left(2 + i, k), -(betas(k) * result(k, j)), x[i][j]);
      }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4 y = x[1][j];
#pragma unroll
      for (int k = 0; k < 2; ++k) y = block_mma(-(left(3, 2 + k) * betas(2 + k)), x[k][j], y);
      x[0][j] = block_mma(-(left(2, 2) * betas(2)), x[0][j], x[0][j]);
      x[1][j] = y;
    }
    settle();
    wave_sync();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) put(2 + i, j, x[i][j]);
  }
  wave_sync();
#pragma unroll
  for (int ti = 0; ti < 4; ++ti)
#pragma unroll
    for (int tj = 0; tj <= ti; ++tj) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(L + row_at(ti) + (lane >> 2) * row_floats(ti) + 16 * tj + 4 * (lane & 3));
      wild |= !finite(x[0]) || !finite(x[1]) || !finite(x[2]) || !finite(x[3]);
      *reinterpret_cast<f32x4*>(rec.tiles[ti * (ti + 1) / 2 + tj] + 4 * lane) = x;
    }
  const bool any = __any(wild);
  if (lane == 0) rec.wild = any;
}

}  // namespace

template <class E>
int launch_records(const Rule<E>& r, int64_t envs, hipStream_t s) {
  const int64_t count = envs * r.heads * r.chunks;
  const dim3 grid((unsigned)((count + kWaves - 1) / kWaves)), block(64 * kWaves);
  if (fours(r.k, r.dk)) records_kernel<E, true><<<grid, block, 0, s>>>(r, count);
  else records_kernel<E, false><<<grid, block, 0, s>>>(r, count);
  return hipGetLastError() == hipSuccess ? RLK_OK : RLK_ERR_LAUNCH;
}
template int launch_records<bf16>(const Rule<bf16>&, int64_t, hipStream_t);
template int launch_records<float>(const Rule<float>&, int64_t, hipStream_t);

}  // namespace delta
}  // namespace rlk
