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
// Both kernels move each byte once.  8192 rows of 8 heads of 128, bf16, are written in 17 us (44 MB,
// 2.6 TB/s; bound by the arithmetic of steps and quotients) and read in 10.5 (4.2 TB/s); prefixes
// of 219 MB as fp16 are read in 40 us (5.5 TB/s, HBM).  A decode step's rows are bound by the launch.
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
  int row_shift, head_shift, bs_shift;   // log2 of a row's words, a head's, BS, or -1
  RowMap map;
};

// Row, record in the row and word in the record of the flat index i over rows of Hkv D / 8
// words.  Shifts where the row's words are a power of 2: divisions are a third of these
// kernels' instructions otherwise.
__device__ inline void split_word(const Q4Args& a, int64_t i, int64_t& row, int& h, int& w) {
  uint32_t in_row;
  if (a.row_shift >= 0) {   // uniform
    row = i >> a.row_shift;
    in_row = (uint32_t)i & ((1u << a.row_shift) - 1);
  } else {
    const uint32_t per = (uint32_t)a.Hkv << a.head_shift;
    if (a.n * per <= 0xffffffffLL) {   // uniform
      const uint32_t r = (uint32_t)i / per;
      row = r;
      in_row = (uint32_t)i - r * per;
    } else {
      row = i / per;
      in_row = (uint32_t)(i - row * per);
    }
  }
  h = (int)(in_row >> a.head_shift);
  w = (int)(in_row & ((1u << a.head_shift) - 1));
}

// RowMap's slot of row i, the page by a shift where BS is a power of 2.
__device__ inline int64_t slot_of(const Q4Args& a, int64_t i) {
  if (a.bs_shift < 0) return a.map.slot(i);   // uniform
  const int64_t b = a.map.seq_ids ? a.map.seq_ids[i] : i;
  const int pos = a.map.positions[i];
  if (b < 0 || b >= a.map.B || pos < 0 || pos >> a.bs_shift >= a.map.MB) return -1;
  const int blk = a.map.bt[b * a.map.MB + (pos >> a.bs_shift)];
  if (blk < 0 || blk >= a.map.NB) return -1;
  return ((int64_t)blk << a.bs_shift) + (pos & (a.map.BS - 1));
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

// One word of a record from its 8 elements; the three neighbouring threads have the rest of
// the group.
template <bool kKeys>
__device__ inline void write_word(const Q4Args& a, uint8_t* rec, int w, const float* x) {
  const int G = a.D / kQ4Group;
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
  const float s = (float)s16, inv = __builtin_amdgcn_rcpf(s);
  // Adding 1.5 2^23 rounds to a whole number and leaves it in the low bits, the rest of
  // which are taken off at the end.
  constexpr float kWhole = 12582912.0f;
  constexpr uint32_t kBits = 0x4b400000u * 0x11111111u;   // those of kWhole, every 4 bits
  float t[8], near = 0.5f;           // to half way
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    t[e] = __builtin_amdgcn_fmed3f((x[e] - base) * inv, 0.0f, 15.0f);
    word += __float_as_uint(t[e] + kWhole) << (4 * e);
  }
  word -= kBits;
#pragma unroll
  for (int e = 0; e < 8; e += 2)
    near = fminf(near, fminf(fabsf(__builtin_amdgcn_fractf(t[e]) - 0.5f),
                             fabsf(__builtin_amdgcn_fractf(t[e + 1]) - 0.5f)));
  if (near < 0x1p-16f) {
    word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double q = rint(((double)x[e] - (double)base) / (double)s);
      word |= (uint32_t)(q < 0.0 ? 0.0 : q > 15.0 ? 15.0 : q) << (4 * e);
    }
  }
  if (!(s > 0.0f)) word = 0;         // one value, or none
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

// A thread: one word of a key's record and the value's, whose slot is the same.
template <typename T, bool kVec>
__global__ __launch_bounds__(kThreads) void q4_append_kernel(Q4Args a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.n * ((int64_t)a.Hkv * (a.D / 8))) return;
  int64_t row;
  int h, w;
  split_word(a, i, row, h, w);
  const int64_t e = ((int64_t)h * a.D + 8 * w) * Codec<T>::kBytes;
  float k[8], v[8];                  // on their way while the slot is looked up
  load_elements<T, kVec>(a.k_src + row * a.k_row + e, k);
  load_elements<T, kVec>(a.v_src + row * a.v_row + e, v);
  const int64_t slot = slot_of(a, row);
  if (slot < 0) return;              // all four threads of a group
  const int64_t rec = (slot * a.Hkv + h) * q4_record_bytes(a.D);
  write_word<true>(a, a.k_cache + rec, w, k);
  write_word<false>(a, a.v_cache + rec, w, v);
}

// The values of 8 elements, not read again by this kernel or kept for it.
template <typename T>
__device__ inline void store8_stream(uint8_t* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    store16_stream(p, make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                                 __float_as_uint(x[3])));
    store16_stream(p + 16, make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]),
                                      __float_as_uint(x[7])));
  } else {
    uint4 w;
    Codec<T>::store8(reinterpret_cast<uint8_t*>(&w), x);
    store16_stream(p, w);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void q4_read_kernel(Q4Args a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.n * ((int64_t)a.Hkv * (a.D / 8))) return;
  int64_t row;
  int h, w;
  split_word(a, i, row, h, w);
  const int G = a.D / kQ4Group;
  const int64_t slot = slot_of(a, row);
  float x[2][8] = {};
  if (slot >= 0) {
    const int64_t at = (slot * a.Hkv + h) * q4_record_bytes(a.D);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint8_t* rec = (c == 0 ? a.k_cache : a.v_cache) + at;
      const int place = c == 0 ? q4_word<true>(w, G) : q4_word<false>(w, G);
      const uint32_t word = *reinterpret_cast<const uint32_t*>(rec + 4 * place);
      const _Float16* par = reinterpret_cast<const _Float16*>(rec + a.D / 2) + (w >> 2);
      const float s = (float)par[0], lo = (float)par[G];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] = fmaf((float)((word >> (4 * e)) & 15u), s, lo);
    }
  }
  const int64_t to = ((row * a.Hkv + h) * (int64_t)a.D + 8 * w) * Codec<T>::kBytes;
  store8_stream<T>(a.k_out + to, x[0]);
  store8_stream<T>(a.v_out + to, x[1]);
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
  auto shift = [](int64_t x) { return x > 0 && (x & (x - 1)) == 0 && x < 1 << 30 ? __builtin_ctzll(x) : -1; };
  a.head_shift = shift(w.D / 8);
  a.row_shift = shift((int64_t)w.Hkv * (w.D / 8));
  a.bs_shift = shift(w.BS);
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
  grid = dim3((unsigned)wgs);
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
