// New K/V rows into the 4-bit cache, and cached rows out of it (hs_q4.h has the format).
//
// Quantising a group of 32 elements x:
//   lo = fp16(min x),  s = fp16(fp32((max x - lo) / 15)), not below 0,
//   n  = (x - lo) / s to the nearest, ties to even, of 0 .. 15, or 0 where s is;
// values beyond fp16's largest count as that; a group that holds a NaN is NaN as a whole (lo
// is NaN, s 0).
// A thread takes 8 elements, one word of a record, and 4 neighbouring threads a group,
// which find its ends with two exchanges inside the quad.  The quotients are fp32
// products with 1 / s, less than 2^-18 off; the few that come within 2^-16 of half
// way between two numbers, and the steps that lie as near to a border between two fp16
// numbers, are computed again in fp64.  So what is written is the definition's, to the bit,
// and does not depend on the order or precision of this code.
//
// Both kernels move each byte once and are bound by HBM, or by their launch for a decode
// step's rows.
#include "hs_kernels.h"
#include "hs_kvrows.h"
#include "hs_q4.h"

#include <algorithm>

namespace hs {

namespace {

constexpr int kThreads = 256;

struct Q4Args {
  uint8_t *k_cache, *v_cache;
  const uint8_t *k_src, *v_src;     // append: sources
  uint8_t *k_out, *v_out;           // read: rows without gaps
  int64_t k_row, v_row;             // bytes between source rows
  int64_t n;
  int Hkv, D;
  RowMap map;
};

// Row, head and word of the flat index i over rows of Hkv D / 8 words.
__device__ inline void split_word(const Q4Args& a, int64_t i, int64_t& row, int& h, int& w) {
  const uint32_t words = (uint32_t)a.D / 8, per = (uint32_t)a.Hkv * words;
  uint32_t in_row;
  if (a.n * per <= 0xffffffffLL) {   // uniform
    const uint32_t r = (uint32_t)i / per;
    row = r;
    in_row = (uint32_t)i - r * per;
  } else {
    row = i / per;
    in_row = (uint32_t)(i - row * per);
  }
  h = (int)(in_row / words);
  w = (int)(in_row - (uint32_t)h * words);
}

template <typename T, bool kVec>
__device__ inline void load_elements(const uint8_t* p, float* x) {
  if constexpr (kVec) {
    Codec<T>::load8(p, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Codec<T>::load1(p + e * Codec<T>::kBytes);
  }
}

// Both propagate NaN, unlike fmaxf and fminf.
__device__ inline float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ inline float nan_min(float a, float b) { return __builtin_elementwise_minimum(a, b); }

// The step of a group, rounded as from fp64: the fp32 quotient is within 2^-22 of it, so
// where both ends of twice that range round to one number, that is the one.
__device__ inline _Float16 q4_step(float most, float lo) {
  if (!(most > lo)) return (_Float16)0.0f;   // lo may lie above, rounded
  const float q = (most - lo) * (1.0f / 15.0f);
  const _Float16 a = (_Float16)(q * (1.0f - 0x1p-21f)), b = (_Float16)(q * (1.0f + 0x1p-21f));
  if (__builtin_expect(a == b, 1)) return a;
  float exact = (float)(((double)most - (double)lo) / 15.0);
  asm volatile("" : "+v"(exact));   // rounded to fp32 first, as defined: not to be folded into one
  return (_Float16)exact;
}

template <typename T, bool kVec, bool kKeys>
__device__ inline void append_word(const Q4Args& a, int64_t row, int h, int w) {
  const int64_t slot = a.map.slot(row);
  if (slot < 0) return;              // all four threads of a group
  const int G = a.D / kQ4Group;
  float x[8];
  load_elements<T, kVec>((kKeys ? a.k_src : a.v_src) + row * (kKeys ? a.k_row : a.v_row) +
                             ((int64_t)h * a.D + 8 * w) * Codec<T>::kBytes, x);
  float hi = x[0], lo = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    hi = nan_max(hi, x[e]);
    lo = nan_min(lo, x[e]);
  }
  hi = nan_max(hi, dpp<kDppQuadXor1>(hi));
  lo = nan_min(lo, dpp<kDppQuadXor1>(lo));
  hi = nan_max(hi, dpp<kDppQuadXor2>(hi));
  lo = nan_min(lo, dpp<kDppQuadXor2>(lo));
  const bool none = hi != hi;
  hi = fminf(fmaxf(hi, -kF16Most), kF16Most);
  const _Float16 lo16 = (_Float16)fminf(fmaxf(lo, -kF16Most), kF16Most);
  const float base = (float)lo16;
  const _Float16 s16 = none ? (_Float16)0.0f : q4_step(hi, base);
  const float s = (float)s16, inv = 1.0f / s;
  // adding 1.5 2^23 rounds to a whole number and leaves it in the low bits
  constexpr float kWhole = 12582912.0f;
  float t[8], r[8], far = 0.0f;
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    t[e] = __builtin_amdgcn_fmed3f((x[e] - base) * inv, 0.0f, 15.0f);
    r[e] = t[e] + kWhole;
    far = fmaxf(far, fabsf(t[e] - (r[e] - kWhole)));
    word += (__float_as_uint(r[e]) - __float_as_uint(kWhole)) << (4 * e);
  }
  if (far > 0.5f - 0x1p-16f) {
    word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double q = rint(((double)x[e] - (double)base) / (double)s);
      word |= (uint32_t)(q < 0.0 ? 0.0 : q > 15.0 ? 15.0 : q) << (4 * e);
    }
  }
  if (!(s > 0.0f)) word = 0;         // one value, or none
  uint8_t* rec = (kKeys ? a.k_cache : a.v_cache) +
                 (slot * a.Hkv + h) * (int64_t)q4_record_bytes(a.D);
  *reinterpret_cast<uint32_t*>(rec + 4 * q4_word<kKeys>(w, G)) = word;
  // the group's first thread stores the step, the second the lowest value
  const int part = w & 3, g = w >> 2;
  if (part < 2) {
    const uint16_t bits = part == 0 ? __builtin_bit_cast(uint16_t, s16)
                          : none    ? (uint16_t)0x7e00
                                    : __builtin_bit_cast(uint16_t, lo16);
    *reinterpret_cast<uint16_t*>(rec + a.D / 2 + 2 * (part * G + g)) = bits;
  }
}

// grid.x covers the words, grid.y K and V.
template <typename T, bool kVec>
__global__ __launch_bounds__(kThreads) void q4_append_kernel(Q4Args a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.n * ((int64_t)a.Hkv * (a.D / 8))) return;
  int64_t row;
  int h, w;
  split_word(a, i, row, h, w);
  if (blockIdx.y == 0) append_word<T, kVec, true>(a, row, h, w);
  else append_word<T, kVec, false>(a, row, h, w);
}

template <typename T, bool kKeys>
__device__ inline void read_word(const Q4Args& a, int64_t row, int h, int w) {
  const int G = a.D / kQ4Group;
  const int64_t slot = a.map.slot(row);
  float x[8];
  if (slot < 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  } else {
    const uint8_t* rec = (kKeys ? a.k_cache : a.v_cache) +
                         (slot * a.Hkv + h) * (int64_t)q4_record_bytes(a.D);
    const uint32_t word = *reinterpret_cast<const uint32_t*>(rec + 4 * q4_word<kKeys>(w, G));
    const _Float16* par = reinterpret_cast<const _Float16*>(rec + a.D / 2) + (w >> 2);
    const float s = (float)par[0], lo = (float)par[G];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((word >> (4 * e)) & 15u), s, lo);
  }
  Codec<T>::store8((kKeys ? a.k_out : a.v_out) +
                       ((row * a.Hkv + h) * (int64_t)a.D + 8 * w) * Codec<T>::kBytes, x);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void q4_read_kernel(Q4Args a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.n * ((int64_t)a.Hkv * (a.D / 8))) return;
  int64_t row;
  int h, w;
  split_word(a, i, row, h, w);
  if (blockIdx.y == 0) read_word<T, true>(a, row, h, w);
  else read_word<T, false>(a, row, h, w);
}

template <typename T>
void launch_append_type(const Q4Args& a, dim3 grid, bool vec, hipStream_t stream) {
  if (vec) hipLaunchKernelGGL((q4_append_kernel<T, true>), grid, dim3(kThreads), 0, stream, a);
  else hipLaunchKernelGGL((q4_append_kernel<T, false>), grid, dim3(kThreads), 0, stream, a);
}

Q4Args rows_args(const Q4Rows& w) {
  Q4Args a{};
  a.k_cache = static_cast<uint8_t*>(w.k_cache);
  a.v_cache = static_cast<uint8_t*>(w.v_cache);
  a.n = w.n;
  a.Hkv = w.Hkv;
  a.D = w.D;
  a.map.bt = w.bt;
  a.map.positions = w.positions;
  a.map.seq_ids = w.seq_ids;
  a.map.num_slots = (int64_t)w.NB * w.BS;
  a.map.NB = w.NB;
  a.map.BS = w.BS;
  a.map.B = w.B;
  a.map.MB = w.MB;
  return a;
}

// The grid over n rows' words, or false where no launch or offset holds it.
bool rows_grid(const Q4Rows& w, int64_t row_bytes, dim3& grid) {
  const int64_t words = sat_mul(w.n, sat_mul(w.Hkv, w.D / 8)), wgs = ceil_div(words, kThreads);
  if (sat_mul(w.Hkv, w.D) > 0x7fffffffLL || !grid_fits(wgs, kThreads) || wgs > 0x7fffffffLL ||
      sat_mul(w.n, row_bytes) == INT64_MAX ||
      sat_mul((int64_t)w.NB * w.BS, sat_mul(w.Hkv, q4_record_bytes(w.D))) == INT64_MAX)
    return false;
  grid = dim3((unsigned)wgs, 2);
  return true;
}

}  // namespace

// Sizes, pointers and the cache's alignment are checked by the caller (hs_api.hip).
int launch_q4_append(const Q4Rows& w, hipStream_t stream) {
  const int64_t sb = dtype_bytes(w.dtype);
  Q4Args a = rows_args(w);
  a.k_src = static_cast<const uint8_t*>(w.k_src);
  a.v_src = static_cast<const uint8_t*>(w.v_src);
  a.k_row = sat_mul(w.k_row, sb);
  a.v_row = sat_mul(w.v_row, sb);
  dim3 grid;
  if (!rows_grid(w, std::max(a.k_row, a.v_row), grid))
    return fail(HS_EUNSUPPORTED, "4-bit append too large for one launch");
  // 16-byte loads where every 8 elements lie so, single ones elsewhere
  const bool vec = aligned16(w.k_src) && aligned16(w.v_src) && a.k_row % 16 == 0 && a.v_row % 16 == 0;
  profile_begin(stream);
  if (w.dtype == HS_DTYPE_F32) launch_append_type<float>(a, grid, vec, stream);
  else if (w.dtype == HS_DTYPE_F16) launch_append_type<_Float16>(a, grid, vec, stream);
  else launch_append_type<Bf16>(a, grid, vec, stream);
  profile_end(stream);
  return check_launch("4-bit KV append");
}

int launch_q4_read(const Q4Rows& w, hipStream_t stream) {
  Q4Args a = rows_args(w);
  a.k_out = static_cast<uint8_t*>(w.k_out);
  a.v_out = static_cast<uint8_t*>(w.v_out);
  dim3 grid;
  if (!rows_grid(w, sat_mul(w.Hkv, w.D, dtype_bytes(w.dtype)), grid))
    return fail(HS_EUNSUPPORTED, "4-bit read too large for one launch");
  profile_begin(stream);
  if (w.dtype == HS_DTYPE_F32)
    hipLaunchKernelGGL((q4_read_kernel<float>), grid, dim3(kThreads), 0, stream, a);
  else if (w.dtype == HS_DTYPE_F16)
    hipLaunchKernelGGL((q4_read_kernel<_Float16>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((q4_read_kernel<Bf16>), grid, dim3(kThreads), 0, stream, a);
  profile_end(stream);
  return check_launch("4-bit KV read");
}

}  // namespace hs
