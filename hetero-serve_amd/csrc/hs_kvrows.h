// What the kernels that write rows of new keys and values share: conversions of
// 8 elements at a time between the cache's types and fp32, and where a row
// lies in the paged cache.
#pragma once

#include "hs_common.h"

namespace hs {

// ---- element codecs: 8 elements <-> 8 fp32 ------------------------------
template <typename T>
struct Codec;

template <>
struct Codec<float> {
  static constexpr int kBytes = 4;
  __device__ static void load8(const uint8_t* p, float* x) {
    const uint4 a = load16(p), b = load16(p + 16);
    x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y);
    x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
    x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y);
    x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
  }
  __device__ static void store8(uint8_t* p, const float* x) {
    *reinterpret_cast<uint4*>(p) = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]),
                                              __float_as_uint(x[2]), __float_as_uint(x[3]));
    *reinterpret_cast<uint4*>(p + 16) = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]),
                                                   __float_as_uint(x[6]), __float_as_uint(x[7]));
  }
  __device__ static float load1(const uint8_t* p) { return *reinterpret_cast<const float*>(p); }
  __device__ static void store1(uint8_t* p, float x) { *reinterpret_cast<float*>(p) = x; }
};

// fp32 -> bf16 bits, round to nearest even; NaN -> 0x7FC0 (c10::BFloat16).
__device__ inline uint32_t f32_to_bf16_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0x7fc0u;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// fp32 -> fp16 bits, round to nearest even (v_cvt_f16_f32); NaN -> sign | 0x7E00
// as torch's CPU conversion gives.
__device__ inline uint32_t f32_to_f16_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return ((u >> 16) & 0x8000u) | 0x7e00u;
  return __builtin_bit_cast(uint16_t, (_Float16)f);
}

template <>
struct Codec<Bf16> {
  static constexpr int kBytes = 2;
  __device__ static void load8(const uint8_t* p, float* x) {
    const uint4 a = load16(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static void store8(uint8_t* p, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f32_to_bf16_bits(x[2 * i]) | (f32_to_bf16_bits(x[2 * i + 1]) << 16);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static float load1(const uint8_t* p) {
    return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
  }
  __device__ static void store1(uint8_t* p, float x) {
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)f32_to_bf16_bits(x);
  }
};

template <>
struct Codec<_Float16> {
  static constexpr int kBytes = 2;
  __device__ static void load8(const uint8_t* p, float* x) {
    const uint4 a = load16(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] & 0xffffu));
      x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
    }
  }
  __device__ static void store8(uint8_t* p, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f32_to_f16_bits(x[2 * i]) | (f32_to_f16_bits(x[2 * i + 1]) << 16);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static float load1(const uint8_t* p) {
    return (float)*reinterpret_cast<const _Float16*>(p);
  }
  __device__ static void store1(uint8_t* p, float x) {
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)f32_to_f16_bits(x);
  }
};

// Where row i goes: an explicit slot, or the slot of (sequence, position)
// through the block table.  Returns -1 for a row that must be skipped.
struct RowMap {
  const int64_t* slots;        // scatter form (null in the append form)
  const int32_t* bt;           // append form: [B, MB] tables
  const int32_t* positions;    //              [n] absolute positions
  const int32_t* seq_ids;      //              [n] row -> sequence, or null (row i = sequence i)
  int64_t num_slots;           // NB * BS
  int NB, BS, B, MB;           // B: table rows; a sequence index must be below it
  int wrap;                    // scatter form: negative slots count from the end

  __device__ int64_t slot(int64_t i) const {
    if (slots) {
      int64_t s = slots[i];
      if (wrap && s < 0) s += num_slots;
      return (s >= 0 && s < num_slots) ? s : -1;
    }
    const int64_t b = seq_ids ? seq_ids[i] : i;
    const int pos = positions[i];
    if (b < 0 || b >= B || pos < 0 || pos / BS >= MB) return -1;
    const int blk = bt[b * MB + pos / BS];
    if (blk < 0 || blk >= NB) return -1;
    return (int64_t)blk * BS + pos % BS;
  }
};

// A launch holds fewer than 2^32 work-items along x.
inline bool grid_fits(int64_t workgroups, int threads) {
  return workgroups < ((int64_t)1 << 32) / threads;
}

inline int dtype_bytes(int code) { return code == HS_DTYPE_F32 ? 4 : 2; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace hs
