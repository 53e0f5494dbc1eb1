// New K/V rows into the 4-bit cache, and cached rows out of it (hs_q4.h has the format).
//
// Quantising a group of 32 elements x:
//   lo = fp16(min x),  s = fp16(fp32((max x - lo) / 15)), not below 0,
//   n  = (x - lo) / s to the nearest, ties to even, of 0 .. 15, or 0 where s is;
// values beyond fp16's largest count as that; a group that holds a NaN is NaN as a whole (lo
// is NaN, s 0).
// A thread takes 8 elements, one word of a record, and 4 neighbouring threads a group,
// which find its ends with two exchanges inside the quad (two words a thread: 20 us
// instead of 17 for 8192 rows).  The quotients are fp32 products with 1 / s; the few that
// come near half way between two numbers, and the steps that lie near a border between two
// fp16 numbers, are computed again in fp64.  So what is written is the definition's, to the
// bit, and does not depend on the order or precision of this code.
//
// Both kernels move each byte once.  8192 rows of 8 heads of 128, bf16, are written in 15 us (44 MB,
// 2.9 TB/s; the arithmetic of steps and quotients is active in 70 % of the cycles) and read in
// 8.5 to 9.5 (4.9 TB/s); prefixes of 219 MB are read in 33.5 us (6.5 TB/s, HBM).  (17.5, 10.2 and 39.5
// with places and addresses for each thread.)  A decode step's rows are bound by the launch.
#include "hs_kernels.h"
#include "hs_kvrows.h"
#include "hs_q4.h"

#include <algorithm>
#include <type_traits>

namespace hs {

namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 8;           // elements of a thread, of keys and of values: a word

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

// Row and word in the row of the flat index i over rows of Hkv D / 8 words.  Shifts where the
// row's words are a power of 2: divisions are a third of these kernels' instructions
// otherwise.
__device__ inline void split_word(const Q4Args& a, int64_t i, int64_t& row, uint32_t& in_row) {
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
}

// What a thread takes: row, record in the row, word in the record.  kWaveRow: a row has a
// multiple of 64 words, so a wave's threads are in one, and its place, its slot and their
// addresses are scalar.
struct Unit {
  int64_t row;
  int h, w;

  // False past the last row.
  template <bool kWaveRow>
  __device__ bool find(const Q4Args& a) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * kThreads + 64 * wave + (kWaveRow ? 0 : lane);
    if (i >= a.n * ((int64_t)a.Hkv << a.head_shift)) return false;
    uint32_t in_row;
    split_word(a, i, row, in_row);
    if constexpr (kWaveRow) in_row += lane;
    h = (int)(in_row >> a.head_shift);
    w = (int)(in_row & ((1u << a.head_shift) - 1));
    return true;
  }
};

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
    for (int e = 0; e < kUnit; ++e) x[e] = Codec<T>::load1(p + e * Codec<T>::kBytes);
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
  for (int e = 1; e < kUnit; ++e) {
    hi = nan_max(hi, x[e]);
    lo = nan_min(lo, x[e]);
  }
  hi = nan_max(hi, dpp<kDppQuadXor1>(hi));
  lo = nan_min(lo, dpp<kDppQuadXor1>(lo));
  hi = nan_max(hi, dpp<kDppQuadXor2>(hi));
  lo = nan_min(lo, dpp<kDppQuadXor2>(lo));
  const bool none = hi != hi;
  const float most = fminf(fmaxf(hi, -kF16Most), kF16Most), least = fminf(fmaxf(lo, -kF16Most), kF16Most);
  const _Float16 lo16 = (_Float16)least;
  const float base = (float)lo16;
  const _Float16 s16 = none ? (_Float16)0.0f : q4_step(most, base);
  const float s = (float)s16, inv = __builtin_amdgcn_rcpf(s);
  // The fp32 quotient is off by less than 2^-21 of it, so where both ends of twice that
  // range round to one number, that is the one.  Adding 1.5 2^23 rounds to a whole number
  // and leaves it in the low bits, the rest of which are taken off at the end.
  constexpr float kWhole = 12582912.0f;
  constexpr uint32_t kBits = 0x4b400000u * 0x11111111u;   // those of kWhole, every 4 bits
  const float inv_a = inv * (1.0f + 0x1p-20f), inv_b = inv * (1.0f - 0x1p-20f);
  uint32_t word = 0, other = 0;
#pragma unroll
  for (int e = 0; e < kUnit; ++e) {
    const float d = x[e] - base;
    word += __float_as_uint(fmaf(d, inv_a, kWhole)) << (4 * e);
    other += __float_as_uint(fmaf(d, inv_b, kWhole)) << (4 * e);
  }
  // No quotient lies below -0.48 or above 15.3: lo is near its fp16 number, the step far enough
  // above fp16's smallest (2^-24 apart) to have 6 bits, and no element counts as another.
  const bool inside = hi == most && lo == least && 2.1f * (base - lo) < s && s >= 0x1p-19f;
  word -= kBits;
  if (s > 0.0f && !(inside && word + kBits == other)) {
    word = 0;
#pragma unroll
    for (int e = 0; e < kUnit; ++e) {
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
template <typename T, bool kVec, bool kWaveRow>
__global__ __launch_bounds__(kThreads) void q4_append_kernel(Q4Args a) {
  Unit u;
  if (!u.find<kWaveRow>(a)) return;
  const uint32_t e = ((uint32_t)u.h * a.D + kUnit * u.w) * Codec<T>::kBytes;
  float k[kUnit], v[kUnit];          // on their way while the slot is looked up
  load_elements<T, kVec>(a.k_src + u.row * a.k_row + e, k);
  load_elements<T, kVec>(a.v_src + u.row * a.v_row + e, v);
  const int64_t slot = slot_of(a, u.row);
  if (slot < 0) return;              // all four threads of a group
  const uint32_t R = q4_record_bytes(a.D), rec = u.h * R;
  const int64_t at = slot * (a.Hkv * R);
  write_word<true>(a, a.k_cache + at + rec, u.w, k);
  write_word<false>(a, a.v_cache + at + rec, u.w, v);
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

template <typename T, bool kWaveRow>
__global__ __launch_bounds__(kThreads) void q4_read_kernel(Q4Args a) {
  Unit u;
  if (!u.find<kWaveRow>(a)) return;
  const int G = a.D / kQ4Group;
  const int64_t slot = slot_of(a, u.row);
  float x[2][8] = {};
  if (slot >= 0) {
    const uint32_t R = q4_record_bytes(a.D), in_row = u.h * R;
    const int64_t at = slot * (a.Hkv * R);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint8_t* rec = (c == 0 ? a.k_cache : a.v_cache) + at + in_row;
      const int place = c == 0 ? q4_word<true>(u.w, G) : q4_word<false>(u.w, G);
      const uint32_t word = *reinterpret_cast<const uint32_t*>(rec + 4 * place);
      const _Float16* par = reinterpret_cast<const _Float16*>(rec + a.D / 2) + (u.w >> 2);
      const float s = (float)par[0], lo = (float)par[G];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[c][e] = fmaf((float)((word >> (4 * e)) & 15u), s, lo);
        // s is rounded, so 15 s + lo may lie beyond what was written, and round to an infinity
        if constexpr (std::is_same<T, _Float16>::value) x[c][e] = nan_min(nan_max(x[c][e], -kF16Most), kF16Most);
      }
    }
  }
  const int64_t to = u.row * ((int64_t)a.Hkv * a.D * Codec<T>::kBytes);
  const uint32_t e = ((uint32_t)u.h * a.D + kUnit * u.w) * Codec<T>::kBytes;
  store8_stream<T>(a.k_out + to + e, x[0]);
  store8_stream<T>(a.v_out + to + e, x[1]);
}

bool wave_rows(const Q4Args& a) { return ((int64_t)a.Hkv << a.head_shift) % 64 == 0; }

template <typename T>
void launch_append_type(const Q4Args& a, dim3 grid, bool vec, hipStream_t stream) {
  const dim3 block(kThreads);
  if (!vec) hipLaunchKernelGGL((q4_append_kernel<T, false, false>), grid, block, 0, stream, a);
  else if (wave_rows(a)) hipLaunchKernelGGL((q4_append_kernel<T, true, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((q4_append_kernel<T, true, false>), grid, block, 0, stream, a);
}

template <typename T>
void launch_read_type(const Q4Args& a, dim3 grid, hipStream_t stream) {
  const dim3 block(kThreads);
  if (wave_rows(a)) hipLaunchKernelGGL((q4_read_kernel<T, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((q4_read_kernel<T, false>), grid, block, 0, stream, a);
}

Q4Args rows_args(const Q4Rows& w) {
  Q4Args a{};
  a.k_cache = static_cast<uint8_t*>(w.k_cache);
  a.v_cache = static_cast<uint8_t*>(w.v_cache);
  a.n = w.n;
  a.Hkv = w.Hkv;
  a.D = w.D;
  auto shift = [](int64_t x) { return x > 0 && (x & (x - 1)) == 0 && x < 1 << 30 ? __builtin_ctzll(x) : -1; };
  a.head_shift = shift(w.D / kUnit);
  a.row_shift = shift((int64_t)w.Hkv * (w.D / kUnit));
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
  const int64_t words = sat_mul(w.n, sat_mul(w.Hkv, w.D / kUnit)), wgs = ceil_div(words, kThreads);
  if (sat_mul(w.Hkv, w.D) > 1 << 29 || !grid_fits(wgs, kThreads) || wgs > 0x7fffffffLL ||
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
  if (w.dtype == HS_DTYPE_F32) launch_read_type<float>(a, grid, stream);
  else if (w.dtype == HS_DTYPE_F16) launch_read_type<_Float16>(a, grid, stream);
  else launch_read_type<Bf16>(a, grid, stream);
  profile_end(stream);
  return check_launch("4-bit KV read");
}

}  // namespace hs
