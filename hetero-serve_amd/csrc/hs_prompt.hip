// Causal attention over whole prompts: packed sequences of different lengths,
// grouped heads, K and V as the projection left them (no cache is read).
//
//   out[i, h] = sum_{j <= i} p_ij v[j, h'],  p_i = softmax_j(scale q[i, h] . k[j, h'])
// over the rows j <= i of row i's own sequence, h' = h / (H / Hkv).
#include "hs_kernels.h"
#include "hs_kvrows.h"

#include <algorithm>

namespace hs {

namespace {

struct PromptArgs {
  const uint8_t *q, *k, *v;
  uint8_t* out;               // [T, H, D]
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // bytes
  const int32_t* cu;          // [B + 1]
  int B, H, Hkv;
  int64_t T;
  int max_len;
  float qscale;               // scale * log2(e)
};

// First row and rows of sequence b, whatever cu holds: rows of [0, T), at most
// max_len of them.
__device__ inline void seq_rows(const PromptArgs& a, int b, int64_t& row0, int& len) {
  row0 = max((int64_t)0, min((int64_t)a.cu[b], a.T));
  const int64_t end = max(row0, min((int64_t)a.cu[b + 1], a.T));
  len = (int)min(end - row0, (int64_t)a.max_len);
}

// One wave: the output row of query `i` (of the sequence that starts at row0) and
// head h, in fp32 arithmetic.  A 16-byte load holds kVec elements, so a key's
// head row is spread over kLpt lanes and a load of the wave covers kTpl keys;
// each such group of lanes runs an online softmax of its own, and the states are
// merged at the end.  Keys behind the row are not added, not even times 0, so what
// they hold cannot reach it.
template <typename T, int D>
__device__ inline void row_walk(const PromptArgs& a, int64_t row0, int i, int h) {
  constexpr int kVec = Elem<T>::kVec, kLpt = D / kVec, kTpl = 64 / kLpt;
  constexpr int kU = 4;
  const int lane = threadIdx.x & 63, slot = lane / kLpt, c = lane % kLpt;
  const int kvh = h / (a.H / a.Hkv);
  const uint8_t* kp = a.k + row0 * a.k_row + kvh * a.k_head + c * 16;
  const uint8_t* vp = a.v + row0 * a.v_row + kvh * a.v_head + c * 16;
  float q[kVec], acc[kVec], m = kNegBig, l = 0.0f;
  Elem<T>::to_f32(load16(a.q + (row0 + i) * a.q_row + h * a.q_head + c * 16), q);
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    q[e] *= a.qscale;
    acc[e] = 0.0f;
  }
  for (int t0 = 0; t0 <= i; t0 += kTpl * kU) {
    uint4 kr[kU], vr[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t t = min(t0 + u * kTpl + slot, i);
      kr[u] = load16(kp + t * a.k_row);
      vr[u] = load16(vp + t * a.v_row);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float f[kVec], d = 0.0f;
      Elem<T>::to_f32(kr[u], f);
#pragma unroll
      for (int e = 0; e < kVec; ++e) d = fmaf(q[e], f[e], d);
      d = group_sum<kLpt>(d);
      const bool ok = t0 + u * kTpl + slot <= i;
      const float m_new = ok ? fmaxf(m, d) : m;
      const float keep = fast_exp2(m - m_new), p = ok ? fast_exp2(d - m_new) : 0.0f;
      m = m_new;
      l = l * keep + p;
      Elem<T>::to_f32(vr[u], f);
#pragma unroll
      for (int e = 0; e < kVec; ++e) acc[e] = ok ? fmaf(p, f[e], acc[e] * keep) : acc[e];
    }
  }
#pragma unroll
  for (int off = kLpt; off < 64; off <<= 1) {
    const float m_o = __shfl_xor(m, off), mm = fmaxf(m, m_o);
    const float w_s = fast_exp2(m - mm), w_o = fast_exp2(m_o - mm);
    l = l * w_s + __shfl_xor(l, off) * w_o;
#pragma unroll
    for (int e = 0; e < kVec; ++e) acc[e] = acc[e] * w_s + __shfl_xor(acc[e], off) * w_o;
    m = mm;
  }
  if (slot != 0) return;
  const float inv = 1.0f / l;
#pragma unroll
  for (int e = 0; e < kVec; ++e) acc[e] *= inv;
  uint8_t* dst = a.out + (((row0 + i) * a.H + h) * (int64_t)D) * (int)sizeof(T) + c * 16;
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(dst) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  else
    Codec<T>::store8(dst, acc);
}

// A wave per (row, head): grid (rows / 4, H).
template <typename T, int D>
__global__ __launch_bounds__(256) void prompt_rows_kernel(PromptArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.T) return;
  int lo = 0, hi = a.B;   // cu[lo] <= row < cu[hi], where cu ascends
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= row) lo = mid; else hi = mid;
  }
  int64_t row0;
  int len;
  seq_rows(a, lo, row0, len);
  if (row < row0 || row >= row0 + len) return;
  row_walk<T, D>(a, row0, (int)(row - row0), blockIdx.y);
}

template <typename T>
int launch_dim(const PromptArgs& a, int D, hipStream_t stream) {
  const dim3 g((unsigned)ceil_div(a.T, 4), (unsigned)a.H), t(256);
  switch (D) {
    case 32: hipLaunchKernelGGL((prompt_rows_kernel<T, 32>), g, t, 0, stream, a); break;
    case 64: hipLaunchKernelGGL((prompt_rows_kernel<T, 64>), g, t, 0, stream, a); break;
    case 128: hipLaunchKernelGGL((prompt_rows_kernel<T, 128>), g, t, 0, stream, a); break;
    case 256: hipLaunchKernelGGL((prompt_rows_kernel<T, 256>), g, t, 0, stream, a); break;
    default: return fail(HS_EUNSUPPORTED, "unsupported head_dim " + std::to_string(D));
  }
  return HS_OK;
}

}  // namespace

// Strides in elements; the sizes and pointers are checked (hs_api.hip).
int launch_prompt(const Prompt& w, hipStream_t stream) {
  const int64_t sb = dtype_bytes(w.dtype);
  PromptArgs a{};
  a.q = static_cast<const uint8_t*>(w.q);
  a.k = static_cast<const uint8_t*>(w.k);
  a.v = static_cast<const uint8_t*>(w.v);
  a.out = static_cast<uint8_t*>(w.out);
  a.q_row = w.q_row * sb;
  a.q_head = w.q_head * sb;
  a.k_row = w.k_row * sb;
  a.k_head = w.k_head * sb;
  a.v_row = w.v_row * sb;
  a.v_head = w.v_head * sb;
  a.cu = w.cu;
  a.B = w.B;
  a.H = w.H;
  a.Hkv = w.Hkv;
  a.T = w.T;
  a.max_len = w.max_len;
  a.qscale = w.scale * kLog2e;
  profile_begin(stream);
  int rc;
  if (w.dtype == HS_DTYPE_F32) rc = launch_dim<float>(a, w.D, stream);
  else if (w.dtype == HS_DTYPE_F16) rc = launch_dim<_Float16>(a, w.D, stream);
  else rc = launch_dim<Bf16>(a, w.D, stream);
  profile_end(stream);
  return rc == HS_OK ? check_launch("prompt attention") : rc;
}

}  // namespace hs
