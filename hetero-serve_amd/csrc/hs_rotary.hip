// Rotary positions with several axes, fused with the write into the paged cache.
//
// Pair i of a head's first 2 P elements is turned by the angle
//   theta_i = positions[axis_i][row] * inv_freq[i]
//   (a, b) -> (a cos theta - b sin theta, b cos theta + a sin theta),
// a and b being elements i and P + i of the head, or 2 i and 2 i + 1
// (interleaved); elements past 2 P pass unchanged.  Text has one axis; images
// and video have the time, the height and the width on different pairs.  In the
// same launch the rotated keys and the values go to their slots of the paged
// cache, so keys are read once, and the write costs no second pass.
//
// The angle of a far position needs more than fp32 (at position 10^6 a step of
// fp32 is 0.06 radians), so position times frequency is formed in turns in fp64,
// reduced to half a turn exactly, and only the fraction is rounded to fp32 for
// the sine and cosine.  Everything else is fp32, rounded once to each output's
// type.
//
// A workgroup takes a few rows (tokens).  Its threads first fill LDS with the
// sines and cosines, one (row, pair) each, which all heads of a row then share;
// then each thread turns 8 pairs at a time (two 16-byte loads of a 16-bit
// source).  Sizes or addresses that are no multiples of 16 bytes take one pair
// at a time.
#include "hs_kernels.h"
#include "hs_kvrows.h"

#include <algorithm>
#include <type_traits>

namespace hs {

namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxPairs = 1024;   // of a head: their sines and cosines lie in LDS

struct RotaryArgs {
  const uint8_t *q, *k, *v;          // v null: no cache is written
  int64_t q_row, k_row, v_row;       // bytes
  const int32_t* positions;          // [axes, n]
  const float* inv_freq;             // [pairs]
  const int32_t* pair_axis;          // [pairs], or null: all on axis 0
  int64_t n;
  int axes, pairs, interleaved, H, Hkv, D;
  uint8_t *q_out, *k_out;            // [n, H, D], [n, Hkv, D]; k_out may be null
  uint8_t *k_cache, *v_cache;        // [num_slots, Hkv, D]
  RowMap map;
  int rows;                          // of a workgroup
};

// Sines and cosines of the workgroup's rows, and the cache slots of those rows.
__device__ inline void fill_angles(const RotaryArgs& a, int64_t row0, int rows, float2* cs,
                                   int64_t* slot) {
  constexpr double kTurn = 0.15915494309189533577;   // 1 / (2 pi)
  for (int e = threadIdx.x; e < rows * a.pairs; e += kRotThreads) {
    const int r = e / a.pairs, i = e - r * a.pairs;
    int axis = a.pair_axis ? a.pair_axis[i] : 0;
    if (axis < 0 || axis >= a.axes) axis = 0;
    const double t = (double)a.positions[axis * a.n + row0 + r] * (double)a.inv_freq[i] * kTurn;
    float s, c;
    sincospif((float)(2.0 * (t - rint(t))), &s, &c);
    cs[e] = make_float2(c, s);
  }
  if (a.v)
    for (int r = threadIdx.x; r < rows; r += kRotThreads) slot[r] = a.map.slot(row0 + r);
  __syncthreads();
}

template <typename S, typename O, typename C>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotaryArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int64_t row0 = (int64_t)blockIdx.x * a.rows;
  const int rows = (int)min((int64_t)a.rows, a.n - row0);
  float2* cs = reinterpret_cast<float2*>(lds);                          // [rows, pairs]
  int64_t* slot = reinterpret_cast<int64_t*>(cs + a.rows * a.pairs);   // [rows]
  fill_angles(a, row0, rows, cs, slot);

  const uint32_t per_head = (uint32_t)a.D / 16;   // groups of 16 elements
  const uint32_t heads = (uint32_t)(a.H + (a.v ? 2 : 1) * a.Hkv);
  const uint32_t per_row = heads * per_head;
  for (uint32_t u = blockIdx.y * kRotThreads + threadIdx.x; u < per_row * (uint32_t)rows;
       u += gridDim.y * kRotThreads) {
    const uint32_t r = u / per_row, in_row = u - r * per_row;
    const uint32_t head = in_row / per_head, g = in_row - head * per_head;
    const int64_t row = row0 + r;
    if (head >= (uint32_t)(a.H + a.Hkv)) {   // a value: cast (or copied) into the cache
      const int64_t sl = slot[r];
      if (sl < 0) continue;
      const int64_t e = (int64_t)(head - a.H - a.Hkv) * a.D + 16 * g;
      const uint8_t* src = a.v + row * a.v_row + e * Codec<S>::kBytes;
      uint8_t* dst = a.v_cache + (sl * ((int64_t)a.Hkv * a.D) + e) * Codec<C>::kBytes;
      if constexpr (std::is_same<S, C>::value) {   // a bit copy (NaN payloads included)
        uint4 w[Codec<S>::kBytes];
#pragma unroll
        for (int b = 0; b < Codec<S>::kBytes; ++b) w[b] = load16(src + 16 * b);
#pragma unroll
        for (int b = 0; b < Codec<S>::kBytes; ++b) *reinterpret_cast<uint4*>(dst + 16 * b) = w[b];
      } else {
        float x[16];
        Codec<S>::load8(src, x);
        Codec<S>::load8(src + 8 * Codec<S>::kBytes, x + 8);
        Codec<C>::store8(dst, x);
        Codec<C>::store8(dst + 8 * Codec<C>::kBytes, x + 8);
      }
      continue;
    }
    const bool is_q = head < (uint32_t)a.H;
    const uint32_t h = is_q ? head : head - a.H;
    const bool turned = g < (uint32_t)a.pairs / 8;
    int e0, e1;   // the two groups of 8 elements
    if (turned && !a.interleaved) {
      e0 = 8 * g;
      e1 = a.pairs + e0;
    } else {
      e0 = turned ? 16 * g : 2 * a.pairs + 16 * (g - a.pairs / 8);
      e1 = e0 + 8;
    }
    const uint8_t* src = (is_q ? a.q + row * a.q_row : a.k + row * a.k_row) +
                         (int64_t)h * a.D * Codec<S>::kBytes;
    float x[8], y[8];
    Codec<S>::load8(src + e0 * Codec<S>::kBytes, x);
    Codec<S>::load8(src + e1 * Codec<S>::kBytes, y);
    if (turned) {
      float2 t[8];
      const float4* c4 = reinterpret_cast<const float4*>(cs + r * a.pairs + 8 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 w = c4[i];
        t[2 * i] = make_float2(w.x, w.y);
        t[2 * i + 1] = make_float2(w.z, w.w);
      }
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = x[2 * i], q = x[2 * i + 1], v = y[2 * i], w = y[2 * i + 1];
          x[2 * i] = p * t[i].x - q * t[i].y;
          x[2 * i + 1] = q * t[i].x + p * t[i].y;
          y[2 * i] = v * t[4 + i].x - w * t[4 + i].y;
          y[2 * i + 1] = w * t[4 + i].x + v * t[4 + i].y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = x[i], q = y[i];
          x[i] = p * t[i].x - q * t[i].y;
          y[i] = q * t[i].x + p * t[i].y;
        }
      }
    }
    uint8_t* out = is_q ? a.q_out : a.k_out;
    if (out) {
      uint8_t* dst = out + ((row * (is_q ? a.H : a.Hkv) + h) * (int64_t)a.D) * Codec<O>::kBytes;
      Codec<O>::store8(dst + e0 * Codec<O>::kBytes, x);
      Codec<O>::store8(dst + e1 * Codec<O>::kBytes, y);
    }
    if (!is_q && a.v && slot[r] >= 0) {
      uint8_t* dst = a.k_cache + (slot[r] * ((int64_t)a.Hkv * a.D) + (int64_t)h * a.D) * Codec<C>::kBytes;
      Codec<C>::store8(dst + e0 * Codec<C>::kBytes, x);
      Codec<C>::store8(dst + e1 * Codec<C>::kBytes, y);
    }
  }
}

// Any size and alignment: one pair, or one element that passes, per thread.
template <typename S, typename O, typename C>
__global__ __launch_bounds__(kRotThreads) void rotary_scalar_kernel(RotaryArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int64_t row0 = (int64_t)blockIdx.x * a.rows;
  const int rows = (int)min((int64_t)a.rows, a.n - row0);
  float2* cs = reinterpret_cast<float2*>(lds);                          // [rows, pairs]
  int64_t* slot = reinterpret_cast<int64_t*>(cs + a.rows * a.pairs);   // [rows]
  fill_angles(a, row0, rows, cs, slot);

  const uint32_t per_head = (uint32_t)(a.D - a.pairs);
  const uint32_t turned_units = (uint32_t)(a.H + a.Hkv) * per_head;
  const uint32_t per_row = turned_units + (a.v ? (uint32_t)(a.Hkv * a.D) : 0u);
  for (uint32_t u = blockIdx.y * kRotThreads + threadIdx.x; u < per_row * (uint32_t)rows;
       u += gridDim.y * kRotThreads) {
    const uint32_t r = u / per_row, in_row = u - r * per_row;
    const int64_t row = row0 + r;
    if (in_row >= turned_units) {
      if (slot[r] < 0) continue;
      const int64_t e = in_row - turned_units;
      const uint8_t* src = a.v + row * a.v_row + e * Codec<S>::kBytes;
      uint8_t* dst = a.v_cache + (slot[r] * ((int64_t)a.Hkv * a.D) + e) * Codec<C>::kBytes;
      if constexpr (std::is_same<S, C>::value) {
        using Word = std::conditional_t<Codec<C>::kBytes == 4, uint32_t, uint16_t>;
        *reinterpret_cast<Word*>(dst) = *reinterpret_cast<const Word*>(src);
      } else {
        Codec<C>::store1(dst, Codec<S>::load1(src));
      }
      continue;
    }
    const uint32_t head = in_row / per_head;
    const int i = (int)(in_row - head * per_head);
    const bool is_q = head < (uint32_t)a.H;
    const uint32_t h = is_q ? head : head - a.H;
    const bool turned = i < a.pairs;
    const int e0 = !turned ? a.pairs + i : a.interleaved ? 2 * i : i;
    const int e1 = !turned ? e0 : a.interleaved ? e0 + 1 : a.pairs + i;
    const uint8_t* src = (is_q ? a.q + row * a.q_row : a.k + row * a.k_row) +
                         (int64_t)h * a.D * Codec<S>::kBytes;
    float x = Codec<S>::load1(src + e0 * Codec<S>::kBytes), y = x;
    if (turned) {
      const float p = x, q = Codec<S>::load1(src + e1 * Codec<S>::kBytes);
      const float2 t = cs[r * a.pairs + i];
      x = p * t.x - q * t.y;
      y = q * t.x + p * t.y;
    }
    uint8_t* out = is_q ? a.q_out : a.k_out;
    if (out) {
      uint8_t* dst = out + ((row * (is_q ? a.H : a.Hkv) + h) * (int64_t)a.D) * Codec<O>::kBytes;
      Codec<O>::store1(dst + e0 * Codec<O>::kBytes, x);
      if (turned) Codec<O>::store1(dst + e1 * Codec<O>::kBytes, y);
    }
    if (!is_q && a.v && slot[r] >= 0) {
      uint8_t* dst = a.k_cache + (slot[r] * ((int64_t)a.Hkv * a.D) + (int64_t)h * a.D) * Codec<C>::kBytes;
      Codec<C>::store1(dst + e0 * Codec<C>::kBytes, x);
      if (turned) Codec<C>::store1(dst + e1 * Codec<C>::kBytes, y);
    }
  }
}

struct RotaryLaunch {
  dim3 grid;
  size_t lds;
  bool vec;
};

template <typename S, typename O, typename C>
void launch_types(const RotaryArgs& a, const RotaryLaunch& l, hipStream_t stream) {
  if (l.vec)
    hipLaunchKernelGGL((rotary_kernel<S, O, C>), l.grid, dim3(kRotThreads), l.lds, stream, a);
  else
    hipLaunchKernelGGL((rotary_scalar_kernel<S, O, C>), l.grid, dim3(kRotThreads), l.lds, stream, a);
}

template <typename S, typename O>
void launch_cache(int kv, const RotaryArgs& a, const RotaryLaunch& l, hipStream_t stream) {
  if (kv == HS_DTYPE_F32) launch_types<S, O, float>(a, l, stream);
  else if (kv == HS_DTYPE_F16) launch_types<S, O, _Float16>(a, l, stream);
  else launch_types<S, O, Bf16>(a, l, stream);
}

template <typename S>
void launch_out(int out, int kv, const RotaryArgs& a, const RotaryLaunch& l, hipStream_t stream) {
  if (out == HS_DTYPE_F32) launch_cache<S, float>(kv, a, l, stream);
  else if (out == HS_DTYPE_F16) launch_cache<S, _Float16>(kv, a, l, stream);
  else launch_cache<S, Bf16>(kv, a, l, stream);
}

}  // namespace

// The sizes and pointers are checked (hs_api.hip); strides in elements.
int launch_rotary(const Rotary& w, hipStream_t stream, int cus) {
  const int64_t sb = dtype_bytes(w.src_dtype), cb = dtype_bytes(w.kv_dtype);
  const int64_t qe = sat_mul(w.H, w.D), ke = sat_mul(w.Hkv, w.D);
  const int64_t per_row = sat_add(qe, sat_mul(2, ke));
  if (w.pairs > kMaxPairs)
    return fail(HS_EUNSUPPORTED, "at most " + std::to_string(kMaxPairs) + " rotary pairs per head");
  if (per_row > (1 << 26)) return fail(HS_EUNSUPPORTED, "rotary rows too large");
  if (sat_mul(w.n, std::max({w.q_row, w.k_row, w.v_row}), sb) == INT64_MAX ||
      sat_mul(w.n, per_row, 4) == INT64_MAX || sat_mul(w.n, w.axes, 4) == INT64_MAX ||
      sat_mul((int64_t)w.NB, w.BS, sat_mul(ke, cb)) == INT64_MAX)
    return fail(HS_EUNSUPPORTED, "rotary sizes too large for 64-bit offsets");
  RotaryArgs a{};
  a.q = static_cast<const uint8_t*>(w.q);
  a.k = static_cast<const uint8_t*>(w.k);
  a.v = static_cast<const uint8_t*>(w.v);
  a.q_row = w.q_row * sb;
  a.k_row = w.k_row * sb;
  a.v_row = w.v_row * sb;
  a.positions = w.positions;
  a.inv_freq = w.inv_freq;
  a.pair_axis = w.pair_axis;
  a.n = w.n;
  a.axes = w.axes;
  a.pairs = w.pairs;
  a.interleaved = w.interleaved;
  a.H = w.H;
  a.Hkv = w.Hkv;
  a.D = w.D;
  a.q_out = static_cast<uint8_t*>(w.q_out);
  a.k_out = static_cast<uint8_t*>(w.k_out);
  a.k_cache = static_cast<uint8_t*>(w.k_cache);
  a.v_cache = static_cast<uint8_t*>(w.v_cache);
  a.map.bt = w.bt;
  a.map.positions = w.cache_positions;
  a.map.seq_ids = w.seq_ids;
  a.map.num_slots = (int64_t)w.NB * w.BS;
  a.map.NB = w.NB;
  a.map.BS = w.BS;
  a.map.B = w.B;
  a.map.MB = w.MB;
  RotaryLaunch l;
  l.vec = w.D % 16 == 0 && w.pairs % 8 == 0 && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) &&
          a.q_row % 16 == 0 && a.k_row % 16 == 0 && a.v_row % 16 == 0 && aligned16(a.q_out) &&
          aligned16(a.k_out) && aligned16(a.k_cache) && aligned16(a.v_cache);
  // Rows of a workgroup: as many as give its threads one (row, pair) each, where
  // that leaves every CU several workgroups; single rows, spread over several
  // workgroups, otherwise.
  const int64_t units = l.vec ? per_row / 16 : per_row;
  const int together = std::max(1, std::min(8, kRotThreads / w.pairs));
  a.rows = w.n >= (int64_t)together * 4 * cus ? together : 1;
  const int64_t parts = a.rows > 1 ? 1 : std::min((int64_t)64, ceil_div(units, kRotThreads));
  const int64_t groups = ceil_div(w.n, a.rows);
  if (groups > 0x7fffffffLL) return fail(HS_EUNSUPPORTED, "too many rows for one launch");
  l.grid = dim3((unsigned)groups, (unsigned)parts);
  l.lds = (size_t)a.rows * (8 + 8 * (size_t)w.pairs);
  profile_begin(stream);
  if (w.src_dtype == HS_DTYPE_F32) launch_out<float>(w.out_dtype, w.kv_dtype, a, l, stream);
  else if (w.src_dtype == HS_DTYPE_F16) launch_out<_Float16>(w.out_dtype, w.kv_dtype, a, l, stream);
  else launch_out<Bf16>(w.out_dtype, w.kv_dtype, a, l, stream);
  profile_end(stream);
  return check_launch("rotary");
}

}  // namespace hs
