// Decode over spans (hs_span.h) on the vector units: fp32, fp16 and bf16 caches, and the
// 4-bit cache.
//
// A wave serves G query heads of one KV head for one part of a row's visible keys.  One
// key's head row is spread over kLpt lanes, kVec elements each, and a load of the wave
// covers kTpl keys; each such group of lanes runs an online softmax over its keys, in base
// 2 with scale * log2(e) folded into the query, and the groups' states are merged at the
// end.  Scores, sums and outputs are fp32.
#include "hs_kernels.h"
#include "hs_kvrows.h"
#include "hs_q4.h"
#include "hs_span.h"

#include <algorithm>

namespace hs {

namespace {

constexpr int kWaves = 4;         // of a workgroup
constexpr float kSlack = 8.0f;    // lazy raise of the running max, log2 units
// Where running maxima start: no finite score lies below, so a row of one is never empty.
constexpr float kLowest = -0x1.fffffep127f;

// What a lane holds of one key's or value's head row.
template <typename T, int D>
struct Plain {
  static constexpr int kVec = Elem<T>::kVec;
  static constexpr int kRow = D * 16 / Elem<T>::kVec;   // bytes of a head row
  struct Piece {
    uint4 w;
  };
  template <bool kKeys>
  __device__ static Piece load(const uint8_t* row, int c) {
    return {load16_stream(row + 16 * c)};
  }
  __device__ static void to_f32(const Piece& x, float* f) { Elem<T>::to_f32(x.w, f); }
};

struct FourBits {};
template <int D>
struct Plain<FourBits, D> {
  static constexpr int kVec = 8;
  static constexpr int kRow = q4_record_bytes(D);
  struct Piece {
    uint32_t w;
    _Float16 s, lo;
  };
  template <bool kKeys>
  __device__ static Piece load(const uint8_t* row, int c) {
    constexpr int G = D / kQ4Group;
    const _Float16* par = reinterpret_cast<const _Float16*>(row + D / 2) + (c >> 2);
    return {*reinterpret_cast<const uint32_t*>(row + 4 * q4_word<kKeys>(c, G)), par[0], par[G]};
  }
  __device__ static void to_f32(const Piece& x, float* f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fmaf((float)((x.w >> (4 * e)) & 15u), (float)x.s, (float)x.lo);
  }
};

template <typename T, int D, int G>
__global__ __launch_bounds__(64 * kWaves) void span_walk_kernel(SpanArgs a) {
  using C = Plain<T, D>;
  constexpr int kVec = C::kVec, kLpt = D / kVec, kTpl = 64 / kLpt;
  constexpr int kU = G >= 4 || D > 128 ? 2 : 4;      // loads in flight
  const int lane = threadIdx.x & 63, slot = lane / kLpt, c = lane % kLpt;
  const int n_hw = a.H / G;
  const int64_t w = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (w >= (int64_t)a.B * a.P * n_hw) return;
  const int h0 = (int)(w % n_hw) * G;
  const int64_t rp = w / n_hw;
  const int b = (int)(rp / a.P), p = (int)(rp % a.P);
  const Span span(a, b);
  const int64_t o0 = ((int64_t)b * a.H + h0) * D;
  int lo, hi, nparts;
  if (!span.part(a, p, lo, hi, nparts)) {
    if (span.n == 0 && p == 0)       // nothing to attend to: zero rows
      for (int d = lane; d < G * D; d += 64) a.out[o0 + d] = 0.0f;
    return;
  }
  const int kvh = h0 / (a.H / a.Hkv);
  const int64_t row = (int64_t)a.Hkv * C::kRow;
  const uint8_t* kp = a.k + (int64_t)kvh * C::kRow;
  const uint8_t* vp = a.v + (int64_t)kvh * C::kRow;
  const int32_t* bt = a.bt + (int64_t)b * a.MB;

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
  for (int t0 = lo; t0 < hi; t0 += kTpl * kU) {
    typename C::Piece kr[kU], vr[kU];
    bool ok[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int t = t0 + u * kTpl + slot;
      ok[u] = t < hi;
      const int64_t at = span.slot(a, bt, min(t, hi - 1)) * row;
      kr[u] = C::template load<true>(kp + at, c);
      vr[u] = C::template load<false>(vp + at, c);
    }
    float pu[G][kU];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float mx = kLowest;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float f[kVec], d = 0.0f;
        C::to_f32(kr[u], f);
#pragma unroll
        for (int e = 0; e < kVec; ++e) d = fmaf(q[g][e], f[e], d);
        d = group_sum<kLpt>(d);
        pu[g][u] = ok[u] ? d : -INFINITY;
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
      float f[kVec];
      C::to_f32(vr[u], f);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        f[e] = ok[u] ? f[e] : 0.0f;   // read twice where the part ends, and not added, not even times 0
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
    const bool whole = nparts == 1;
    const float inv = !whole ? 1.0f : l[g] == 0.0f ? 0.0f : 1.0f / l[g];
    const int64_t pi = ((int64_t)b * a.H + h0 + g) * a.P + p;
    float* to = (whole ? a.out + o0 + g * D : a.part_acc + pi * D) + c * kVec;
#pragma unroll
    for (int e = 0; e < kVec; e += 4)
      *reinterpret_cast<float4*>(to + e) = make_float4(acc[g][e] * inv, acc[g][e + 1] * inv,
                                                       acc[g][e + 2] * inv, acc[g][e + 3] * inv);
    if (!whole && c == 0) reinterpret_cast<float2*>(a.part_ml)[pi] = make_float2(m[g], l[g]);
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
  const Span span(a, (int)(w / a.H));
  int lo, hi, n;
  if (!span.part(a, 0, lo, hi, n) || n == 1) return;   // written already
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + w * a.P;
  const int each = (n + kWaves - 1) / kWaves, first = min(n, wv * each), end = min(n, first + each);
  float mm = kLowest;
  for (int p = first + lane; p < end; p += 64) mm = fmaxf(mm, ml[p].x);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) mm = fmaxf(mm, __shfl_xor(mm, off));
  float acc[kPer] = {}, l = 0.0f;
  for (int p0 = first; p0 < end; p0 += 64) {
    const int here = min(64, end - p0);
    const float2 st = lane < here ? ml[p0 + lane] : make_float2(kLowest, 0.0f);
    const float wt = lane < here ? fast_exp2(st.x - mm) : 0.0f;
    l = fmaf(st.y, wt, l);
    const float* pa = a.part_acc + (w * a.P + p0) * D;
    for (int p = 0; p < here; p += kBatch) {
      float v[kBatch][kPer];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int d = lane + 64 * i;
          v[u][i] = p + u < here && d < D ? pa[(p + u) * D + d] : 0.0f;
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
  const dim3 grid((unsigned)ceil_div(sat_mul(a.B, a.P, a.H / G), kWaves)), block(64 * kWaves);
  switch (G) {
    case 8: hipLaunchKernelGGL((span_walk_kernel<T, D, 8>), grid, block, 0, stream, a); break;
    case 4: hipLaunchKernelGGL((span_walk_kernel<T, D, 4>), grid, block, 0, stream, a); break;
    case 2: hipLaunchKernelGGL((span_walk_kernel<T, D, 2>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((span_walk_kernel<T, D, 1>), grid, block, 0, stream, a); break;
  }
}

template <typename T>
int launch_walk_dim(const SpanArgs& a, int D, hipStream_t stream) {
  switch (D) {
    case 32: launch_walk<T, 32>(a, stream); break;
    case 64: launch_walk<T, 64>(a, stream); break;
    case 128: launch_walk<T, 128>(a, stream); break;
    case 256: launch_walk<T, 256>(a, stream); break;
    default: return fail(HS_EUNSUPPORTED, "unsupported head_dim " + std::to_string(D));
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

// Keys of a part: 512, cut down to 64 while the waves of the longest rows would be fewer
// than eight for each CU.
void span_plan(int kv_dtype, int B, int H, int Hkv, int D, int64_t most, int cus, int* part, int* heads) {
  if (kv_dtype < 0) return q4_decode_plan(B, H, Hkv, D, most, cus, part, heads);
  if (window_decode_serves(kv_dtype, D)) return window_decode_plan(B, H, Hkv, most, cus, part, heads);
  *part = 512;
  *heads = 0;
  const int64_t waves = sat_mul(B, H / row_attn_heads_per_wave(H, Hkv));
  while (*part > 64 && sat_mul(waves, ceil_div(most, *part)) < 8 * (int64_t)cus) *part /= 2;
}

// The parts, and the merge of rows of several.  kv_dtype -1: the 4-bit cache.
int launch_span(const SpanArgs& a, int kv_dtype, int D, hipStream_t stream) {
  const int64_t rows = sat_mul(a.B, a.H), waves = sat_mul(rows, a.P);
  if (!grid_fits(rows, 64 * kWaves) || !grid_fits(ceil_div(waves, kWaves), 64 * kWaves))
    return fail(HS_EUNSUPPORTED, "grid too large: sequences * parts * heads = " + std::to_string(waves));
  int rc;
  profile_begin(stream);
  if (kv_dtype < 0) rc = launch_q4_decode(a, D, stream);
  else if (window_decode_serves(kv_dtype, D)) rc = launch_window_decode(a, kv_dtype, D, stream);
  else if (kv_dtype == HS_DTYPE_F32) rc = launch_walk_dim<float>(a, D, stream);
  else if (kv_dtype == HS_DTYPE_F16) rc = launch_walk_dim<_Float16>(a, D, stream);
  else rc = launch_walk_dim<Bf16>(a, D, stream);
  profile_end(stream);
  if (rc != HS_OK) return rc;
  if (a.P > 1) launch_span_merge(a, D, stream);
  return check_launch("span decode");
}

}  // namespace hs
