// rlk_attention.hpp -- what the two forms of linear attention share: arguments as the kernels take them, checks,
// and how a sequence is cut into segments.
#pragma once
#include "rlk_launch.hpp"
#include "rlk_policy.hpp"

namespace rlk {

// (environment, head) pairs of one launch, whose work-items are at most 2^32 - 1 (three workgroups of 512 a pair); more
// environments go in further launches.
constexpr int64_t kMaxPairs = (int64_t{1} << 21) - 8;

template <class E>
struct Sequence {
  E* data;
  int64_t env_stride, step_stride, head_stride;
};

template <class E>
struct Walk {
  Sequence<const E> a, b, c;
  Sequence<E> y;
  int da, dc;  // dims of a and b, of c and y
  const float* state;
  float* state_out;
  float* seg_states;  // [env, head, segment, da, dc]: what enters the segment (0 unused)
  float* seg_keep;    // [env, head, segment]: how much of what enters the segment before leaves it; below 0: nothing, an episode ends in it
  float scale, state_scale, state_out_scale;
  int transposed, reverse;
};

template <class E>
struct Walks {
  Walk<E> w[3];
  int64_t num_envs, seq_len, seg_len;
  int64_t first_env;  // of this launch, which has num_envs of them
  int count, heads, segs;
  const float *decay, *dones;
};

template <class E>
Sequence<E> sequence(const rlk_sequence& x) {
  return {static_cast<E*>(const_cast<void*>(x.data)), x.env_stride, x.step_stride, x.head_stride};
}

inline bool valid_attention(const rlk_attention& c, bool steps = true) {  // steps: there are any, so their arrays are
  if (c.num_envs < 0 || c.heads < 0 || c.dim_k < 1 || c.dim_k > 128 || c.dim_v < 1 || c.dim_v > 128) return false;
  if (!std::isfinite(c.scale) || !std::isfinite(c.state_scale) || !std::isfinite(c.state_out_scale)) return false;
  if (c.num_envs == 0 || c.heads == 0) return true;
  const uintptr_t low = c.bf16 ? 1u : 3u;
  for (const rlk_sequence* x : {&c.q, &c.k, &c.v, &c.out})
    if (steps && (!x->data || (reinterpret_cast<uintptr_t>(x->data) & low) != 0)) return false;
  return c.decay != nullptr;
}

struct SegmentPlan {
  int segs;
  int64_t seg_len;  // a multiple of 64
};

// Segments: none where the (environment, head) pairs fill the GPU by themselves; else as many as make one round of
// the workgroups that it holds (two per CU for dims of up to 64, one beyond), of at least 4 chunks (a segment's k and v are read
// twice, and its state is written and read once per segment).
inline SegmentPlan plan_segments(int64_t rows, int64_t T, bool small) {
  const int64_t cus = device_cus(), chunks = (T + 63) / 64;
  int64_t segs = rows >= cus ? 1 : (small ? 2 : 1) * cus / rows;
  if (segs > chunks / 4) segs = chunks / 4;
  if (segs < 1) segs = 1;
  const int64_t per = (chunks + segs - 1) / segs;
  segs = (chunks + per - 1) / per;
  return {(int)segs, per * 64};
}

}  // namespace rlk
