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
// then each thread turns the pairs of two 16-byte loads.  Sizes or addresses that are no
// multiples of 16 bytes take one pair at a time.
//
// Bound by HBM: 8192 rows of 32 / 8 heads, D 128, bf16 in and out (218 MB), 39 us,
// 5.6 TB/s (a large copy reaches 6.6), with loads that leave the cache in front of
// HBM to what is written, 47 without that hint.  A decode step's few rows take 4.3 us,
// a launch and two dependent reads.  A thread per unit of a row, with several rows'
// loads in flight, was no faster (50 us).
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

__device__ inline void turn(float& a, float& b, float c, float s) {
  const float p = a;
  a = p * c - b * s;
  b = b * c + p * s;
}

// N elements (4 or 8) from fp32, each rounded once.
template <typename T, int N>
__device__ inline void store(uint8_t* p, const float* x) {
  if constexpr (N == 8) {
    Codec<T>::store8(p, x);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    float y[8] = {x[0], x[1], x[2], x[3], 0.0f, 0.0f, 0.0f, 0.0f};
    uint4 w;
    Codec<T>::store8(reinterpret_cast<uint8_t*>(&w), y);
    *reinterpret_cast<uint2*>(p) = make_uint2(w.x, w.y);
  }
}

// A unit is two 16-byte loads: the same place in both halves of a head's turned part
// (which pairs up the elements, or, interleaved, holds whole pairs), of the part that
// passes, or of a value's head.  Neighbouring lanes read neighbouring 16 bytes.
template <typename S, typename O, typename C>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotaryArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  constexpr int kV = Elem<S>::kVec, kS = Codec<S>::kBytes, kO = Codec<O>::kBytes, kC = Codec<C>::kBytes;
  const int64_t row0 = (int64_t)blockIdx.x * a.rows;
  const int rows = (int)min((int64_t)a.rows, a.n - row0);
  float2* cs = reinterpret_cast<float2*>(lds);                          // [rows, pairs]
  int64_t* slot = reinterpret_cast<int64_t*>(cs + a.rows * a.pairs);   // [rows]
  fill_angles(a, row0, rows, cs, slot);

  const uint32_t per_head = (uint32_t)a.D / (2 * kV);
  const uint32_t heads = (uint32_t)(a.H + (a.v ? 2 : 1) * a.Hkv);
  const uint32_t per_row = heads * per_head;
  const int turned_units = a.pairs / kV;
  for (uint32_t u = blockIdx.y * kRotThreads + threadIdx.x; u < per_row * (uint32_t)rows;
       u += gridDim.y * kRotThreads) {
    const uint32_t r = u / per_row, in_row = u - r * per_row;
    const uint32_t head = in_row / per_head;
    const int g = (int)(in_row - head * per_head);
    const int64_t row = row0 + r;
    if (head >= (uint32_t)(a.H + a.Hkv)) {   // a value: cast (or copied) into the cache
      const int64_t sl = slot[r];
      if (sl < 0) continue;
      const uint32_t h = head - a.H - a.Hkv;
      const uint8_t* src = a.v + row * a.v_row + ((int64_t)h * a.D + kV * g) * kS;
      uint8_t* dst = a.v_cache + ((sl * a.Hkv + h) * (int64_t)a.D + kV * g) * kC;
      const uint4 w[2] = {load16_stream(src), load16_stream(src + a.D / 2 * kS)};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (std::is_same<S, C>::value) {   // a bit copy (NaN payloads included)
          *reinterpret_cast<uint4*>(dst + i * (a.D / 2) * kC) = w[i];
        } else {
          float x[kV];
          Elem<S>::to_f32(w[i], x);
          store<C, kV>(dst + i * (a.D / 2) * kC, x);
        }
      }
      continue;
    }
    const bool is_q = head < (uint32_t)a.H, turned = g < turned_units;
    const uint32_t h = is_q ? head : head - a.H;
    const int e0 = kV * g + (turned ? 0 : a.pairs);   // behind both halves of the turned part
    const int e1 = e0 + (turned ? a.pairs : a.D / 2 - a.pairs);
    const uint8_t* src = (is_q ? a.q + row * a.q_row : a.k + row * a.k_row) + (int64_t)h * a.D * kS;
    float x[kV], y[kV];
    {
      const uint4 w0 = load16_stream(src + e0 * kS), w1 = load16_stream(src + e1 * kS);
      Elem<S>::to_f32(w0, x);
      Elem<S>::to_f32(w1, y);
    }
    if (turned) {
      const float2* t = cs + r * a.pairs;
      if (a.interleaved) {
        const float4* t0 = reinterpret_cast<const float4*>(t + e0 / 2);
        const float4* t1 = reinterpret_cast<const float4*>(t + e1 / 2);
#pragma unroll
        for (int i = 0; i < kV / 4; ++i) {
          const float4 c0 = t0[i], c1 = t1[i];
          turn(x[4 * i], x[4 * i + 1], c0.x, c0.y);
          turn(x[4 * i + 2], x[4 * i + 3], c0.z, c0.w);
          turn(y[4 * i], y[4 * i + 1], c1.x, c1.y);
          turn(y[4 * i + 2], y[4 * i + 3], c1.z, c1.w);
        }
      } else {
        const float4* t0 = reinterpret_cast<const float4*>(t + e0);
#pragma unroll
        for (int i = 0; i < kV / 2; ++i) {
          const float4 c = t0[i];
          turn(x[2 * i], y[2 * i], c.x, c.y);
          turn(x[2 * i + 1], y[2 * i + 1], c.z, c.w);
        }
      }
    }
    uint8_t* out = is_q ? a.q_out : a.k_out;
    if (out) {
      uint8_t* dst = out + ((row * (is_q ? a.H : a.Hkv) + h) * (int64_t)a.D) * kO;
      store<O, kV>(dst + e0 * kO, x);
      store<O, kV>(dst + e1 * kO, y);
    }
    if (!is_q && a.v && slot[r] >= 0) {
      uint8_t* dst = a.k_cache + ((slot[r] * a.Hkv + h) * (int64_t)a.D) * kC;
      store<C, kV>(dst + e0 * kC, x);
      store<C, kV>(dst + e1 * kC, y);
    }
  }
}

// Any size and alignment: one pair, or one element that passes, per thread.  Bound by its
// loads and stores of one element a lane, 8 times as many as of 16 bytes: 8192 rows of 32 / 8
// heads, bf16, keys kept, us: D 128 off a 16-byte boundary 88 (2.5 TB/s; on one 40), D 36 33
// (1.9 TB/s).  What a projection leaves is aligned, with D a multiple of 16.
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
      const float2 t = cs[r * a.pairs + i];
      y = Codec<S>::load1(src + e1 * Codec<S>::kBytes);
      turn(x, y, t.x, t.y);
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
  // Two rows share a workgroup's set-up where that leaves every CU several
  // workgroups (8192 rows, 32 / 8 heads, D 128, bf16, us at 1 / 2 / 4 / 8: 46 / 38 / 41 / 44);
  // otherwise one row is spread over several workgroups.
  const int64_t units = l.vec ? per_row / (32 / sb) : per_row;
  a.rows = w.n >= (int64_t)8 * cus ? 2 : 1;
  const int64_t parts = a.rows > 1 ? 1 : std::min((int64_t)64, ceil_div(units, kRotThreads));
  const int64_t groups = ceil_div(w.n, a.rows);
  if (!grid_fits(groups, kRotThreads)) return fail(HS_EUNSUPPORTED, "too many rows for one launch");
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
