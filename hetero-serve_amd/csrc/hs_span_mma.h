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

using namespace span;

typedef float float4x __attribute__((ext_vector_type(4)));

constexpr int kXcds = 8;           // workgroups are dealt to them in turn
constexpr int kSlots = 16;         // columns of the products
constexpr int kDealt = kSpanDealt / 64;   // rows of a lane
constexpr int kLongest = 32;       // steps of a fitted part: what the matrix cores cut off adds up

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

// The sum of x over lanes up to this one.
__device__ inline int sum_up_to(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // from 1, 2, 4, 8 lanes below
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // lane 15 of a row to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // lane 31 to rows 2 and 3
  return x;
}

// A wave's task.  `heads` query heads of a KV head a wave.
struct Task {
  int wv, hw, np, hsub, ph;   // wave; heads side by side, phases; this wave's
  uint32_t x;                 // number of the part among those of all rows
  int part, b, p, kvh, h0, gc;   // keys of a part; row, part; KV head, first query head, how many
  int64_t row0;               // head h0 of row b, of [B, H]

  // Part x of a call whose parts are fitted to the chip: they have the fewest steps, and those of
  // a.part at least, with which they are a.room at most, or kLongest.  Whole parts come first, then the
  // rows' last ones that are not whole, then the rows without keys: XCDs, to which
  // workgroups go in turn, have as many as each other, and long parts do not begin late.
  // Every wave finds all this by itself, in less than 1 us (which batches whose parts are few
  // anyway do not pay), and the grid holds a.tasks: 64 rows of 16..4096 keys in tables of 32768
  // take 57.5 us (79 with a workgroup for every part of the table), of 131072 70 (187).
  //   us, parts of 512 keys / fitted as it was added, D 128, 32 / 8 heads, 4 bits: 64 rows of 16..4096
  // keys 62 / 56, of 16..8192 97 / 88, of 8192 each 163 / 157, 16 of 8k..32k 117 / 103; 64 of 500..4000,
  // D 256, 85 / 61; over bf16, 64 of 64..4096 110 / 101.
  __device__ bool fit(const SpanArgs& a, int step) {
    const int lane = threadIdx.x & 63;
    int n[kDealt];                   // keys of row 64 r + lane; none behind the last row
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < kDealt; ++r) {
      n[r] = -1;
      if (64 * r >= a.B) continue;   // uniform
      n[r] = Span(a, min(64 * r + lane, a.B - 1)).n;
      if (64 * r + lane >= a.B) n[r] = -1;
      sum += (float)max(n[r], 0);
    }
    auto parts_of = [&](int keys) {
      int count = 0;
#pragma unroll
      for (int r = 0; r < kDealt; ++r)
        if (64 * r < a.B) count += ((uint32_t)max(n[r], 0) + (uint32_t)keys - 1) / (uint32_t)keys;
      return __builtin_amdgcn_readlane(sum_up_to(count), 63);
    };
    part = a.part;
    int parts = parts_of(part);
    if (parts > a.room) {
      sum = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(group_sum<64>(sum))));
      int steps = max(part / step, (int)(sum / ((float)step * (float)a.room)));
      for (;;) {
        steps = min(steps, kLongest);
        part = steps * step;
        parts = parts_of(part);
        if (steps == kLongest || parts <= a.room) break;
        steps += max(1, steps / 16);
      }
    }
    if (x == 0 && threadIdx.x == 0) *a.fitted = part;
    if (x >= (uint32_t)parts + a.B) return false;

    int whole[kDealt], left = x;
#pragma unroll
    for (int r = 0; r < kDealt; ++r) {
      whole[r] = 0;
      if (64 * r >= a.B) continue;
      whole[r] = (uint32_t)max(n[r], 0) / (uint32_t)part;
      const int up_to = sum_up_to(whole[r]), all = __builtin_amdgcn_readlane(up_to, 63);
      if (left < all) {              // uniform
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(up_to > left));
        const int mine = __builtin_amdgcn_readlane(whole[r], l), keys = __builtin_amdgcn_readlane(n[r], l);
        b = 64 * r + l;
        p = left - (__builtin_amdgcn_readlane(up_to, l) - mine) + a.P - mine - (keys > mine * part);
        return true;
      }
      left -= all;
    }
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
      for (int r = 0; r < kDealt; ++r) {
        const bool is = kind == 0 ? n[r] > whole[r] * part : n[r] == 0;
        const uint64_t rows = __builtin_amdgcn_ballot_w64(is);
        const int all = __builtin_popcountll(rows);
        if (left < all) {
          const int below = __builtin_amdgcn_mbcnt_hi(rows >> 32, __builtin_amdgcn_mbcnt_lo((uint32_t)rows, 0));
          const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(is && below == left));
          b = 64 * r + l;
          p = kind == 0 ? a.P - 1 : 0;
          return true;
        }
        left -= all;
      }
    return false;
  }

  // False: nothing there, for all of the workgroup.  p as Span::part counts.
  __device__ bool find(const SpanArgs& a, int heads, int chunk) {
    wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    hw = a.heads;
    np = kWaves / hw;
    hsub = wv % hw;
    ph = wv / hw;
    const int group = a.H / a.Hkv, n_hc = (group + heads - 1) / heads, units = a.Hkv / hw * n_hc;
    // The heads of one part run on one XCD, one behind the other: they share lines of 128 bytes.
    const uint32_t turn = blockIdx.x / kXcds;
    x = turn / (uint32_t)units * kXcds + blockIdx.x % kXcds;
    if (x >= (uint32_t)a.tasks) return false;
    const int unit = turn % (uint32_t)units;
    part = a.part;
    if (a.room) {                    // uniform
      if (!fit(a, chunk * np)) return false;
      if (unit == 0 && threadIdx.x == 0) {
        const int n = Span(a, b).parts(part), first = p - (a.P - n);
        if (first == 0) a.numbers[2 * b] = (int)x;
        if (first == n - 1) a.numbers[2 * b + 1] = (int)x;
      }
    } else {
      // Parts of all rows next to each other, and a row's parts on every XCD in turn.
      const uint32_t B = a.B;
      p = x / B;
      b = (x - p * B + (B % 2 == 0 ? p : 0)) % B;
    }
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
  // The state of head h of this wave's: parts of fitted length lie by their number.
  auto state = [&](int h) { return a.room ? (int64_t)t.x * a.H + t.h0 + h : (t.row0 + h) * a.P + t.p; };
  auto over = [&](float sum) { return !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum; };
  if (t.np == 1) {
    const float inv = over(l);
    float* to = whole ? a.out + (t.row0 + jh) * D : a.part_acc + state(jh) * D;
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
      if (jh < t.gc && mine(d)) *reinterpret_cast<float4x*>(to + 16 * d + 4 * g) = o[d] * inv;
    if (!whole && jh < t.gc && lead) reinterpret_cast<float2*>(a.part_ml)[state(jh)] = make_float2(m, l);
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
    reinterpret_cast<float2*>(a.part_ml)[state(jh)] = make_float2(mm, l);
  __syncthreads();
  for (int x = t.ph * 64 + lane; x < t.gc * (D / 4); x += t.np * 64) {
    const int h = x / (D / 4), d = x % (D / 4) * 4;
    float4x sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < t.np; ++i)
      sum += *reinterpret_cast<const float4x*>(stage(t.hsub + t.hw * i) + h * (D + 4) + d);
    float* to = whole ? a.out + (t.row0 + h) * D : a.part_acc + state(h) * D;
    *reinterpret_cast<float4x*>(to + d) = sum;
  }
}

// Workgroups of `heads` query heads a wave; INT64_MAX when too many.
inline int64_t workgroups(const SpanArgs& a, int heads) {
  const int64_t units = a.Hkv / a.heads * ceil_div(a.H / a.Hkv, heads);
  return sat_mul(ceil_div(a.tasks, kXcds), kXcds, units);
}

// Parts that are on the chip at a time, which holds `slots` workgroups, each XCD as many; where
// that is fewer than two a row, of as many rounds as give two.
inline int parts_on_chip(int B, int H, int Hkv, int heads, int side, int slots) {
  const int64_t units = Hkv / side * ceil_div(H / Hkv, heads);
  const int64_t round = std::max<int64_t>(slots / kXcds / units, 1) * kXcds;
  return (int)std::min<int64_t>(ceil_div(2 * (int64_t)B, round) * round, 0x7fffffff);
}

// Short rows are whole: as many KV heads side by side as leave a workgroup for each CU, where
// their steps are at most eight, or one head and four phases where there are too few for
// that and they take two steps.  Longer rows are cut into parts of eight chunks, shorter ones
// (of two steps) and fewer heads side by side while the parts are fewer than the CUs; of
// sixteen where all waves are phases of one head and two workgroups a CU are left (64 rows of
// 16..8192 keys, 4 bits, 16 heads over 1: 31 us, 33.5 of eight, as it was chosen, 33.3 since each group has
// its own scale; 512 rows of 8192 168, 196).
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
