// Decode over spans (hs_span.h) on the vector units: fp32 caches, and fp16 and bf16 ones of head
// dim 256; and the merge of rows whose keys are several parts.
//
// A workgroup serves G query heads of one KV head for one part of a row's visible keys; its
// four waves take the part's steps in turn and put their states together through LDS.  One
// key's head row is spread over kLpt lanes, kVec elements each, and a load of the wave
// covers kTpl keys; each such group of lanes runs an online softmax over its keys, in base
// 2 with scale * log2(e) folded into the query, and the groups' states are merged at the
// end.  Scores, sums and outputs are fp32.  A step's keys and values are on their way while
// the one before is computed, its table entries while the one before that is.  Behind a window
// of 1024, 64 fp32 rows of 12 heads of 64, 390 MB, take 80 us (4.9 TB/s; 130 with a wave
// for a part and nothing ahead), of 32 / 8 heads of 128, 520 MB, 100 (5.2 TB/s; 170).
#include "hs_kernels.h"
#include "hs_kvrows.h"
#include "hs_span.h"

#include <algorithm>

namespace hs {

namespace {

using namespace span;

template <typename T, int D, int G>
__global__ __launch_bounds__(64 * kWaves) void span_walk_kernel(SpanArgs a) {
  constexpr int kVec = Elem<T>::kVec, kLpt = D / kVec, kTpl = 64 / kLpt;
  constexpr int kU = G >= 4 || D > 128 ? 2 : 4;      // loads in flight, of keys and of values
  constexpr int kStep = kTpl * kU;
  __shared__ float s_m[kWaves][G], s_l[kWaves][G], s_acc[kWaves][G][D];
  const int lane = threadIdx.x & 63, slot = lane / kLpt, c = lane % kLpt;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n_hw = a.H / G, rp = blockIdx.x / n_hw;
  const int h0 = (int)(blockIdx.x - rp * n_hw) * G;
  const int b = (int)(rp / (uint32_t)a.P);
  int p = (int)(rp % (uint32_t)a.P);
  const Span span(a, b);
  const int64_t o0 = ((int64_t)b * a.H + h0) * D;
  int lo, hi, nparts;
  if (!span.part(a, a.part, p, lo, hi, nparts)) {   // all of the workgroup
    if (span.n == 0 && p == -a.P)    // nothing to attend to: zero rows
      for (int d = threadIdx.x; d < G * D; d += 64 * kWaves) a.out[o0 + d] = 0.0f;
    return;
  }
  const int64_t row = (int64_t)a.Hkv * D * sizeof(T);
  const uint8_t* kp = a.k + h0 / (a.H / a.Hkv) * (int64_t)(D * sizeof(T)) + 16 * c;
  const uint8_t* vp = a.v + h0 / (a.H / a.Hkv) * (int64_t)(D * sizeof(T)) + 16 * c;
  const int32_t* bt = a.bt + (int64_t)b * a.MB;

  Span::Place ahead[kU];
  uint4 kr[kU], vr[kU];
  auto look = [&](int t0) {
#pragma unroll
    for (int u = 0; u < kU; ++u) ahead[u] = span.place(a, bt, min(t0 + u * kTpl + slot, hi - 1));
  };
  auto load = [&](const int64_t (&at)[kU]) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      kr[u] = load16_stream(kp + at[u]);
      vr[u] = load16_stream(vp + at[u]);
    }
  };
  auto rows_of = [&](int64_t (&at)[kU]) {
#pragma unroll
    for (int u = 0; u < kU; ++u) at[u] = (int64_t)Span::slot(a, ahead[u]) * row;
  };
  const int first = lo + wv * kStep;
  if (first < hi) {
    int64_t at[kU];
    look(first);
    rows_of(at);
    look(first + kWaves * kStep);
    load(at);
  }
  float q[G][kVec], acc[G][kVec], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      q[g][e] = a.q[o0 + g * D + c * kVec + e] * a.qscale;
      acc[g][e] = 0.0f;
    }
    m[g] = kLowest;
    l[g] = 0.0f;
  }
  for (int t0 = first; t0 < hi; t0 += kWaves * kStep) {
    uint4 kc[kU], vc[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      kc[u] = kr[u];
      vc[u] = vr[u];
    }
    if (t0 + kWaves * kStep < hi) {   // uniform
      int64_t at[kU];
      rows_of(at);
      look(t0 + 2 * kWaves * kStep);
      load(at);
    }
    float pu[G][kU];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float mx = kLowest;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float f[kVec], d = 0.0f;
        Elem<T>::to_f32(kc[u], f);
#pragma unroll
        for (int e = 0; e < kVec; ++e) d = fmaf(q[g][e], f[e], d);
        d = group_sum<kLpt>(d);
        pu[g][u] = t0 + u * kTpl + slot < hi ? d : -INFINITY;
        mx = fmaxf(mx, pu[g][u]);
      }
      if (__builtin_amdgcn_ballot_w64(mx > m[g] + kSlack) != 0) {
        const float m_new = fmaxf(m[g], mx), keep = fast_exp2(m[g] - m_new);
        m[g] = m_new;
        l[g] *= keep;
#pragma unroll
        for (int e = 0; e < kVec; ++e) acc[g][e] *= keep;
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        pu[g][u] = fast_exp2(pu[g][u] - m[g]);
        l[g] += pu[g][u];
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const bool ok = t0 + u * kTpl + slot < hi;
      float f[kVec];
      Elem<T>::to_f32(vc[u], f);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        f[e] = ok ? f[e] : 0.0f;   // read twice where the part ends, and not added, not even times 0
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g][e] = fmaf(pu[g][u], f[e], acc[g][e]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int off = kLpt; off < 64; off <<= 1) {
      const float m_o = __shfl_xor(m[g], off), mm = fmaxf(m[g], m_o);
      const float w_s = fast_exp2(m[g] - mm), w_o = fast_exp2(m_o - mm);
      l[g] = l[g] * w_s + __shfl_xor(l[g], off) * w_o;
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        acc[g][e] = acc[g][e] * w_s + __shfl_xor(acc[g][e], off) * w_o;
      m[g] = mm;
    }
    if (slot != 0) continue;
#pragma unroll
    for (int e = 0; e < kVec; ++e) s_acc[wv][g][c * kVec + e] = acc[g][e];
    if (c == 0) {
      s_m[wv][g] = m[g];
      s_l[wv][g] = l[g];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += 64 * kWaves) {
    const int g = i / D, d = i % D;
    float mm = s_m[0][g], sum = 0.0f, x = 0.0f;
#pragma unroll
    for (int v = 1; v < kWaves; ++v) mm = fmaxf(mm, s_m[v][g]);
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float w = fast_exp2(s_m[v][g] - mm);
      sum = fmaf(s_l[v][g], w, sum);
      x = fmaf(s_acc[v][g][d], w, x);
    }
    if (nparts == 1) {
      a.out[o0 + i] = sum == 0.0f ? 0.0f : x * (1.0f / sum);
    } else {
      const int64_t pi = ((int64_t)b * a.H + h0 + g) * a.P + p;
      a.part_acc[pi * D + d] = x;
      if (d == 0) reinterpret_cast<float2*>(a.part_ml)[pi] = make_float2(mm, sum);
    }
  }
}

// The rows whose keys are several parts': one workgroup per (row, head), lanes over D, a
// quarter of the parts each wave.
template <int D>
__global__ __launch_bounds__(64 * kWaves) void span_merge_kernel(SpanArgs a) {
  constexpr int kPer = (D + 63) / 64, kBatch = 8;
  __shared__ float sums[kWaves][kPer * 64], most[kWaves], totals[kWaves];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t w = blockIdx.x;
  const int b = (int)(w / a.H), h = (int)(w - (int64_t)b * a.H);
  int part = a.part, number = 0, last = 0;
  if (a.room) {         // uniform; read with the row's length, not behind it
    part = *a.fitted;
    number = a.numbers[2 * b];
    last = a.numbers[2 * b + 1];
  }
  const int n = Span(a, b).parts(part);
  if (n <= 1) return;   // written already
  const int64_t base = a.room ? (int64_t)number * a.H + h : w * a.P, apart = a.room ? a.H : 1;
  const int64_t end_state = a.room ? (int64_t)last * a.H + h : base + n - 1;
  auto state = [&](int p) { return p < n - 1 ? base + p * apart : end_state; };
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
  const int each = (n + kWaves - 1) / kWaves, first = min(n, wv * each), end = min(n, first + each);
  float mm = kLowest;
  for (int p = first + lane; p < end; p += 64) mm = fmaxf(mm, ml[state(p)].x);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) mm = fmaxf(mm, __shfl_xor(mm, off));
  float acc[kPer] = {}, l = 0.0f;
  for (int p0 = first; p0 < end; p0 += 64) {
    const int here = min(64, end - p0);
    const float2 st = lane < here ? ml[state(p0 + lane)] : make_float2(kLowest, 0.0f);
    const float wt = lane < here ? fast_exp2(st.x - mm) : 0.0f;
    l = fmaf(st.y, wt, l);
    for (int p = 0; p < here; p += kBatch) {
      float v[kBatch][kPer];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float* pa = a.part_acc + state(p0 + min(p + u, here - 1)) * D;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int d = lane + 64 * i;
          v[u][i] = p + u < here && d < D ? pa[d] : 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float wu = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wt), min(p + u, 63)));
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] = fmaf(v[u][i], wu, acc[i]);
      }
    }
  }
  l = group_sum<64>(l);
#pragma unroll
  for (int i = 0; i < kPer; ++i) sums[wv][lane + 64 * i] = acc[i];
  if (lane == 0) {
    most[wv] = mm;
    totals[wv] = l;
  }
  __syncthreads();
  if (wv != 0) return;
  mm = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  l = 0.0f;
  float keep[kWaves];
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    keep[i] = fast_exp2(most[i] - mm);
    l = fmaf(totals[i], keep[i], l);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 64 * i;
    float x = 0.0f;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) x = fmaf(sums[u][d], keep[u], x);
    if (d < D) a.out[w * D + d] = x * inv;
  }
}

template <typename T, int D>
void launch_walk(const SpanArgs& a, hipStream_t stream) {
  const int G = row_attn_heads_per_wave(a.H, a.Hkv);
  const dim3 grid((unsigned)sat_mul(a.B, a.P, a.H / G)), block(64 * kWaves);
  switch (G) {
    case 8: hipLaunchKernelGGL((span_walk_kernel<T, D, 8>), grid, block, 0, stream, a); break;
    case 4: hipLaunchKernelGGL((span_walk_kernel<T, D, 4>), grid, block, 0, stream, a); break;
    case 2: hipLaunchKernelGGL((span_walk_kernel<T, D, 2>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((span_walk_kernel<T, D, 1>), grid, block, 0, stream, a); break;
  }
}

// fp32 and head dim 256: the others have the matrix cores (hs_window_decode.hip).
int launch_walk_type(const SpanArgs& a, int kv_dtype, int D, hipStream_t stream) {
  const int64_t wgs = sat_mul(a.B, a.P, a.H / row_attn_heads_per_wave(a.H, a.Hkv));
  if (!grid_fits(wgs, 64 * kWaves))
    return fail(HS_EUNSUPPORTED, "grid too large: sequences * parts * heads = " + std::to_string(wgs));
  if (D == 256) {
    if (kv_dtype == HS_DTYPE_F32) launch_walk<float, 256>(a, stream);
    else if (kv_dtype == HS_DTYPE_F16) launch_walk<_Float16, 256>(a, stream);
    else launch_walk<Bf16, 256>(a, stream);
  } else if (D == 128) {
    launch_walk<float, 128>(a, stream);
  } else if (D == 64) {
    launch_walk<float, 64>(a, stream);
  } else {
    launch_walk<float, 32>(a, stream);
  }
  return HS_OK;
}

}  // namespace

void launch_span_merge(const SpanArgs& a, int D, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.B * a.H)), block(64 * kWaves);
  switch (D) {
    case 32: hipLaunchKernelGGL((span_merge_kernel<32>), grid, block, 0, stream, a); break;
    case 64: hipLaunchKernelGGL((span_merge_kernel<64>), grid, block, 0, stream, a); break;
    case 128: hipLaunchKernelGGL((span_merge_kernel<128>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((span_merge_kernel<256>), grid, block, 0, stream, a); break;
  }
}

// Vector units: rows are whole where that makes a workgroup for each CU, or they are short;
// otherwise parts of 2048 keys, cut down to 256 while the workgroups are fewer than two for
// each CU.
void span_plan(int kv_dtype, int B, int H, int Hkv, int D, int64_t most, bool windowed, int cus, int* part,
               int* heads, int* room, int* longest) {
  if (kv_dtype < 0) return q4_decode_plan(B, H, Hkv, D, most, windowed, cus, part, heads, room, longest);
  if (window_decode_serves(kv_dtype, D))
    return window_decode_plan(B, H, Hkv, D, most, windowed, cus, part, heads, room, longest);
  *heads = *room = *longest = 0;
  const int64_t wgs = sat_mul(B, H / row_attn_heads_per_wave(H, Hkv));
  int len = 2048;
  while (len > 256 && sat_mul(wgs, ceil_div(most, len)) < 2 * (int64_t)cus) len /= 2;
  *part = most <= 512 || (most <= 4096 && wgs >= cus) ? (int)most : len;
}

// The parts, and the merge of rows of several.  kv_dtype -1: the 4-bit cache.
int launch_span(const SpanArgs& a, int kv_dtype, int D, hipStream_t stream) {
  if (!grid_fits(sat_mul(a.B, a.H), 64 * kWaves))
    return fail(HS_EUNSUPPORTED, "grid too large: sequences * heads");
  int rc;
  profile_begin(stream);
  if (kv_dtype < 0) rc = launch_q4_decode(a, D, stream);
  else if (window_decode_serves(kv_dtype, D)) rc = launch_window_decode(a, kv_dtype, D, stream);
  else rc = launch_walk_type(a, kv_dtype, D, stream);
  profile_end(stream);
  if (rc != HS_OK) return rc;
  if (a.P > 1) launch_span_merge(a, D, stream);
  return check_launch("span decode");
}

}  // namespace hs
