// What the matrix-core decodes over spans have in common (hs_q4_decode.hip,
// hs_window_decode.hip): which keys and heads a wave takes, and how the waves' outputs leave.
//
// One workgroup: one part of one row, for hw KV heads side by side.  Its four waves are these
// heads times np phases, which take neighbouring chunks of a step of np chunks in turn and
// put their states together at the end.  Waves share nothing before that.
#pragma once

#include "hs_span.h"

namespace hs {
namespace span_mma {

typedef float float4x __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;          // of a workgroup
constexpr int kXcds = 8;           // workgroups are dealt to them in turn
constexpr int kSlots = 16;         // columns of the products
constexpr float kSlack = 8.0f;     // lazy raise of the running max, log2 units
// Where running maxima start: no finite score lies below, so a row of one is never empty.
constexpr float kLowest = -0x1.fffffep127f;

// x of lanes l, l ^ 16, l ^ 32 and l ^ 48.
__device__ inline float max_across_groups(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ inline float sum_across_groups(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// One wave's LDS traffic is in order; this keeps the compiler's in order too.
__device__ inline void lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A wave's task.  `heads` query heads of a KV head a wave.
struct Task {
  int wv, hw, np, hsub, ph;   // wave; heads side by side, phases; this wave's
  int b, p, kvh, h0, gc;      // row, part; KV head, first query head, how many
  int64_t row0;               // head h0 of row b, of [B, H]

  // False: nothing there, for all of the workgroup.
  __device__ bool find(const SpanArgs& a, int heads) {
    wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    hw = a.heads;
    np = kWaves / hw;
    hsub = wv % hw;
    ph = wv / hw;
    const int group = a.H / a.Hkv, n_hc = (group + heads - 1) / heads, units = a.Hkv / hw * n_hc;
    // The heads of one part run on one XCD, one behind the other: they share lines of 128 bytes.
    const uint32_t turn = blockIdx.x / kXcds, rp = turn / (uint32_t)units * kXcds + blockIdx.x % kXcds;
    if (rp >= (uint64_t)a.B * a.P) return false;
    const int unit = turn % (uint32_t)units;
    // Parts of all rows next to each other, and a row's parts on every XCD in turn.
    const uint32_t B = a.B;
    p = rp / B;
    b = (rp - p * B + (B % 2 == 0 ? p : 0)) % B;
    kvh = unit / n_hc * hw + hsub;
    const int hc = unit % n_hc;
    h0 = kvh * group + hc * heads;
    gc = min(heads, group - hc * heads);
    row0 = (int64_t)b * a.H + h0;
    return true;
  }
};

// The rows of a sequence without keys.
template <int D>
__device__ inline void zero_rows(const SpanArgs& a, const Task& t) {
  if (t.ph == 0)
    for (int d = threadIdx.x & 63; d < t.gc * D; d += 64) a.out[t.row0 * D + d] = 0.0f;
}

// The outputs of a part: lane (j, g) holds elements 16 d + 4 g .. of head jh in o[d], not
// normalised, where mine(d), and the head's maximum m (log2 units) and sum l; `lead` lanes
// are one for each head.  stage(wave): LDS of kHeads (D + 4) floats, done with.  All waves of
// the workgroup call it.
template <int D, int kHeads, typename Mine, typename Stage>
__device__ inline void finish(const SpanArgs& a, const Task& t, bool whole, float4x (&o)[D / 16], float m,
                              float l, int jh, bool lead, Mine mine, Stage stage,
                              float2 (&states)[kWaves][kSlots]) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const int64_t pi = (t.row0 + jh) * a.P + t.p;
  auto over = [&](float sum) { return !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum; };
  if (t.np == 1) {
    const float inv = over(l);
    float* to = whole ? a.out + (t.row0 + jh) * D : a.part_acc + pi * D;
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
      if (jh < t.gc && mine(d)) *reinterpret_cast<float4x*>(to + 16 * d + 4 * g) = o[d] * inv;
    if (!whole && jh < t.gc && lead) reinterpret_cast<float2*>(a.part_ml)[pi] = make_float2(m, l);
    return;
  }
  lds_order();
  if (lead) states[t.wv][jh] = make_float2(m, l);
  __syncthreads();
  float mm = m;
  for (int i = 0; i < t.np; ++i) mm = fmaxf(mm, states[t.hsub + t.hw * i][jh].x);
  l = 0.0f;
  for (int i = 0; i < t.np; ++i) {
    const float2 x = states[t.hsub + t.hw * i][jh];
    l = fmaf(x.y, fast_exp2(x.x - mm), l);
  }
  const float keep = fast_exp2(m - mm) * over(l);
#pragma unroll
  for (int d = 0; d < D / 16; ++d)
    if (mine(d)) *reinterpret_cast<float4x*>(stage(t.wv) + jh * (D + 4) + 16 * d + 4 * g) = o[d] * keep;
  if (!whole && t.ph == 0 && jh < t.gc && lead)
    reinterpret_cast<float2*>(a.part_ml)[pi] = make_float2(mm, l);
  __syncthreads();
  for (int x = t.ph * 64 + lane; x < t.gc * (D / 4); x += t.np * 64) {
    const int h = x / (D / 4), d = x % (D / 4) * 4;
    float4x sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < t.np; ++i)
      sum += *reinterpret_cast<const float4x*>(stage(t.hsub + t.hw * i) + h * (D + 4) + d);
    float* to = whole ? a.out + (t.row0 + h) * D : a.part_acc + ((t.row0 + h) * a.P + t.p) * D;
    *reinterpret_cast<float4x*>(to + d) = sum;
  }
}

// Workgroups of `heads` query heads a wave; INT64_MAX when too many.
inline int64_t workgroups(const SpanArgs& a, int heads) {
  const int64_t units = a.Hkv / a.heads * ceil_div(a.H / a.Hkv, heads);
  return sat_mul(ceil_div(sat_mul(a.B, a.P), kXcds), kXcds, units);
}

// Short rows are whole: as many KV heads side by side as leave a workgroup for each CU, where
// their steps are at most eight, or one head and four phases where there are too few for
// that and they take two steps.  Longer rows are cut into parts of eight chunks, shorter ones
// (of two steps) and fewer heads side by side while the parts are fewer than the CUs; of
// sixteen where all waves are phases of one head and two workgroups a CU are left (64 rows of
// 16..8192 keys, 4 bits, 16 heads over 1: 31 us, 33.5 of eight; 512 rows of 8192 168, 196).
// Rows behind a window are as long as each other, so more of them are whole.  us, parts / whole,
// windows of 1024: over 64 rows of 32 / 8 heads, bf16, D 128 55 / 46, D 64 33 / 25, 4 bits, D 128
// 30 / 28; 8 heads, bf16, D 32 23.5 / 19; 8 rows of 32 heads, bf16, D 128 35 / 27.5.
inline void plan(int B, int H, int Hkv, int heads, int chunk, int64_t most, bool windowed, int cus, int* part,
                 int* side) {
  const int most_steps = windowed ? 20 : 8;
  const int64_t n_hc = ceil_div(H / Hkv, heads);
  int wide = kWaves;
  while (Hkv % wide) wide /= 2;
  auto wgs = [&](int hw, int64_t len) { return sat_mul(B, Hkv / hw * n_hc, ceil_div(most, len)); };
  for (int hw = wide; hw >= 1; hw /= 2) {
    const int64_t step = chunk * kWaves / hw, steps = ceil_div(most, step);
    if (steps <= most_steps && (wgs(hw, most) >= cus || (hw == 1 && steps <= 2))) {
      *part = (int)(steps * step);
      *side = hw;
      return;
    }
  }
  for (int hw = wide; hw >= 1; hw /= 2)
    for (int len = (hw == 1 ? 16 : 8) * chunk; len >= 2 * chunk * kWaves / hw; len /= 2)
      if (wgs(hw, len) >= (len > 8 * chunk ? 2 : 1) * (int64_t)cus) {
        *part = len;
        *side = hw;
        return;
      }
  *part = chunk * kWaves;
  *side = 1;
}

}  // namespace span_mma
}  // namespace hs
