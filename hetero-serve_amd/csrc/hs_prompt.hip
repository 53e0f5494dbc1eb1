// Causal attention over whole prompts: packed sequences of different lengths,
// grouped heads, K and V as the projection left them (no cache is read).
//
//   out[i, h] = sum_{j <= i} p_ij v[j, h'],  p_i = softmax_j(scale q[i, h] . k[j, h'])
// over the rows j <= i of row i's own sequence, h' = h / (H / Hkv).
//
// A workgroup of 4 waves takes 128 query rows of one (sequence, head), 32 a wave, and
// walks the keys once with a running maximum and sum.  K and V tiles go from global
// memory straight to LDS (two of each; the next ones are on their way while one is
// used), swizzled by permuting the addresses that the lanes load from, since the LDS
// side of such a load is linear (fp32 tiles pass through registers, see Split3).
// S^T = K Q^T and O^T = V^T P^T: a lane holds one query's scores, so its maximum and sum
// need one exchange of the two lane halves, and the probabilities are the second
// product's operand where they stand.  Short prompts take a wave each, and batches of
// different short lengths 64 rows a workgroup (see few and launch_dim).  Rows are
// otherwise 128 and not 256 a workgroup because two workgroups then share a CU: one's
// set-up and barriers pass beside the other's products.  us at 256 / 128 rows, bf16:
// one prompt of 2048 tokens, 32 / 8 heads, D 128 55 / 49, 32 of 128 tokens 50 / 27, one
// of 8192 493 / 496.
//
// What bounds it: the matrix cores' power.  One prompt of 8192 tokens, 32 / 8 heads,
// D 128, bf16: 485 us, 1135 TFLOP/s of useful products at 1.9 GHz (2.5 PFLOP/s
// nominal at 2.4; the library's product of two 8192 x 8192 matrices reaches 1226).  The
// same loop without softmax and without LDS reads reached 1534, without softmax 1347,
// without barriers and loads 1129.
//
// Numerics.  16-bit inputs are multiplied in their own type, the probabilities
// rounded to it (relative to a maximum that is at most 2^8 too low, so none
// overflows), and the sum adds the rounded ones, so that the rounding cancels where
// one key dominates; scores, maxima, sums and O are fp32.  fp16 probabilities are held
// 2^7 times larger (kLift), which 2^15 still fits: those far below 1, of which a long row
// may have thousands for each one near it, keep steps of 2^-31 of it instead of 2^-24.  fp32 inputs are split into
// three bf16 terms, which keeps fp32's accuracy (see Split3).  Scores are scaled in fp32
// behind the product, not in the query's type before it.
//
// O is a sum that is divided at its end, so values above fp32's largest over 2^8 times the
// number of keys can overflow it where their mean would not: such a row is not finite, and
// computed again with values scaled down (row_walk).
//
// Masked keys.  A score that a row does not see is -inf and its probability 0, but 0
// times an infinite or NaN value is NaN in a product.  A row whose result is not
// finite is therefore computed again by a walk that never touches the keys behind
// it (row_walk).  Rows that hold such values by right pay for it too: those of a key only
// up to it, those of a value for all of the row's keys, many times the products' price.
// One prompt of 8192 tokens, 32 / 8 heads, D 128, bf16, 0.51 ms: with an infinity in the
// first value of one KV head 33 ms, in the middle one 26; with a NaN in the first key of
// one 0.76, in the middle one 18 (1024 tokens, 25 us: 1.4 ms, 1.4, 69 us and 0.77 ms).
#include "hs_kernels.h"
#include "hs_kvrows.h"

#include <algorithm>

namespace hs {

namespace {

// Where running maxima start: no finite score lies below, so a row of one is never empty.
constexpr float kLowest = -0x1.fffffep127f;

struct PromptArgs {
  const uint8_t *q, *k, *v;
  uint8_t* out;               // [T, H, D]
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // bytes
  const int32_t* cu;          // [B + 1]
  int B, H, Hkv;
  int64_t T;
  int max_len;
  float qscale;               // scale * log2(e)
  int by_level, per;          // order of the tiles: see Task
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
// they hold cannot reach it.  Values are added times a power of 2 that keeps the sum of
// i + 1 of them in range, and a mean of finite ones that rounds past the largest number is
// that number.
template <typename T, int D>
__device__ inline void row_walk(const PromptArgs& a, int64_t row0, int i, int h) {
  constexpr int kVec = Elem<T>::kVec, kLpt = D / kVec, kTpl = 64 / kLpt;
  constexpr int kU = 4;
  const int lane = threadIdx.x & 63, slot = lane / kLpt, c = lane % kLpt;
  const int kvh = h / (a.H / a.Hkv);
  const uint8_t* kp = a.k + row0 * a.k_row + kvh * a.k_head + c * 16;
  const uint8_t* vp = a.v + row0 * a.v_row + kvh * a.v_head + c * 16;
  float q[kVec], acc[kVec], m = kLowest, l = 0.0f;
  const float up = ldexpf(1.0f, 33 - __clz(i + 1)), down = 1.0f / up;   // up > 2 (i + 1)
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
      for (int e = 0; e < kVec; ++e) acc[e] = ok ? fmaf(p, f[e] * down, acc[e] * keep) : acc[e];
    }
    // a score that is none, or infinite: so is the sum, and every element of the row
    if (__builtin_amdgcn_ballot_w64(l != l) != 0) break;
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
  const float inv = up / l;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    const float mean = acc[e] * inv;
    acc[e] = fabsf(acc[e]) < INFINITY && fabsf(mean) == INFINITY ? copysignf(-kLowest, mean) : mean;
  }
  uint8_t* dst = a.out + (((row0 + i) * a.H + h) * (int64_t)D) * (int)sizeof(T) + c * 16;
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(dst) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  else
    Codec<T>::store8(dst, acc);
}

// ---- the matrix-core kernels ------------------------------------------------

// No scale is taken as this one, fp32's least number: all finite scores are below 5e-7 then.
constexpr float kLeastScale = 0x1p-149f;
constexpr float kSlack = 8.0f;   // lazy raise of the running max, log2 units

typedef short short4x __attribute__((ext_vector_type(4)));
typedef short short8x __attribute__((ext_vector_type(8)));
typedef float float16x __attribute__((ext_vector_type(16)));
typedef float float2x __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Half;   // kLift: powers of 2 that probabilities are held above themselves
template <>
struct Half<Bf16> {
  static constexpr float kLift = 0.0f;
  // acc + both halves' values, in fp32
  __device__ static float sum2(uint32_t w, float acc) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w),
                                           __builtin_bit_cast(bf16x2, 0x3f803f80u), acc, false);
  }
  __device__ static float16x mma(short8x a, short8x b, float16x c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ static uint32_t pack(float a, float b) {   // v_cvt_pk_bf16_f32, to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2x){a, b}, bf16x2));
  }
};
template <>
struct Half<_Float16> {
  static constexpr float kLift = 7.0f;
  __device__ static float sum2(uint32_t w, float acc) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3c003c00u),
                                  acc, false);
  }
  __device__ static float16x mma(short8x a, short8x b, float16x c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2x){a, b}, f16x2));
  }
};

__device__ inline int64_t readlane64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

__device__ inline int swap23(int r) { return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1); }

// Both lane halves' larger value, and sum.
__device__ inline float both_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float both_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 16 bytes from base + every lane's offset to LDS, at the wave's byte offset `to` + 16 lane;
// counted by vmcnt.  As a builtin, the compiler waits for all such loads before every
// transposing read.  No output register is in flight.  m0 is reserved: the compiler keeps no
// value there, and warns of it among the clobbers, where it says that one which the compiler
// sets for an instruction of its own is lost (of this file's none needs it).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void load_to_lds(const uint8_t* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to),
               "v"(offset), "s"(base)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Where the 16-byte chunk c of row r lies in its LDS row of kC chunks, so that each
// reading pattern covers all 64 banks: K rows are read 16 at a time at one chunk, V
// rows 4 at a time at 4 neighbouring chunks.
template <int kC>
struct KPlace {
  static constexpr int kPeriod = 16;   // rows
  __device__ static int at(int r, int c) {
    if constexpr (kC >= 16) return c ^ (r & 15);
    else if constexpr (kC == 8) return c ^ ((r >> 1) & 7);
    else return c ^ ((r >> 2) & 3);
  }
};
template <int kC>
struct VPlace {
  static constexpr int kPeriod = 4;
  __device__ static int at(int r, int c) {
    if constexpr (kC >= 16) return c ^ ((r & 3) << 2);
    else if constexpr (kC == 8) return c ^ (((r >> 1) & 1) << 2);
    else return c;
  }
};

// The loads of K's or V's rows, kKeys at a time; rows past the sequence are read as
// its last one (and masked), and behind the last tile it is read again.  A load of the
// workgroup covers kStep rows; the swizzle repeats after kOff of them, so those many
// offsets per lane serve all.
template <int kC, int kKeys, typename Place, int kThreads>
struct TileLoads {
  static constexpr int kLoads = kKeys * kC / kThreads, kStep = kThreads / kC;
  static constexpr int kOff = Place::kPeriod > kStep ? Place::kPeriod / kStep : 1;
  static_assert(kLoads >= 1 && kLoads * kThreads == kKeys * kC, "tile / thread split");
  const uint8_t* base;    // of the next tile
  int64_t stride;         // bytes between rows
  int left;               // rows of the sequence from the next tile on
  uint32_t lds;           // this wave's part of the first of two tiles
  uint32_t off[kOff];

  __device__ void init(const uint8_t* first, int64_t row_stride, int len, uint32_t to, int wave) {
    base = first;
    stride = row_stride;
    left = len;
    lds = __builtin_amdgcn_readfirstlane(to + wave * 1024);
    const int r = threadIdx.x / kC, c = threadIdx.x % kC;
#pragma unroll
    for (int u = 0; u < kOff; ++u)
      off[u] = (uint32_t)r * (uint32_t)stride + 16 * Place::at(u * kStep + r, c);
  }
  __device__ void load(int odd) {
    const uint32_t to = lds + odd * (kKeys * kC * 16);
    if (left >= kKeys) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u)
        load_to_lds(base + u * kStep * stride, off[u % kOff], to + u * kThreads * 16);
    } else {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int r = u * kStep + threadIdx.x / kC;
        load_to_lds(base, (uint32_t)min(r, left - 1) * (uint32_t)stride + 16 * Place::at(r, threadIdx.x % kC),
                    to + u * kThreads * 16);
      }
    }
    if (left > kKeys) {
      base += stride * kKeys;
      left -= kKeys;
    }
  }
};

// Sum over the wave, in every lane.
__device__ inline int wave_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, kDppQuadXor1, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kDppQuadXor2, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kDppRowHalfMirror, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kDppRowMirror, 0xF, 0xF, false);
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = r[0] + r[1];
  const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return s[0] + s[1];
}

// Sum of this lane's and the lanes' before it.
__device__ inline int wave_scan(int x) {
  constexpr int kRowShr = 0x110, kBcast15 = 0x142, kBcast31 = 0x143;
  x += __builtin_amdgcn_update_dpp(0, x, kRowShr + 1, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kRowShr + 2, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kRowShr + 4, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kRowShr + 8, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kBcast15, 0xA, 0xF, false);   // rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, kBcast31, 0xC, 0xF, false);   // rows 2 and 3
  return x;
}

// What a workgroup works on: rows q0 .. of a sequence, for one head.
struct Task {
  int h, kvh, q0, len;
  int64_t row0;
  __device__ bool find(const PromptArgs& a, int rows) {
    // neighbouring workgroups: the heads of one tile, a KV head's group on one XCD
    const int p = blockIdx.x % a.H;
    kvh = p % a.Hkv;
    h = kvh * (a.H / a.Hkv) + p / a.Hkv;
    int qt = 0;
    row0 = len = 0;
    const bool there = find_tile(a, rows, (int)(blockIdx.x / a.H), qt);
    // wave-uniform, and the loop's bounds with them
    row0 = readlane64(row0);
    len = __builtin_amdgcn_readfirstlane(len);
    qt = __builtin_amdgcn_readfirstlane(qt);
    q0 = qt * rows;
    return there && qt >= 0 && q0 < len;   // (cu that overlaps can count past 32 bits)
  }

 private:
  __device__ void take(int64_t lane_row0, int lane_len, int lane) {
    row0 = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(lane_row0 >> 32), lane) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)lane_row0, lane));
    len = __builtin_amdgcn_readlane(lane_len, lane);
  }

  // The tile of query rows that workgroup `i` takes, nt_b tiles of `rows` rows in
  // sequence b, of which tile qt walks the keys of qt + 1; sets row0 and len.  Every wave
  // finds it by itself, with the lengths of up to 64 sequences in its lanes.  False: there
  // is no such tile.
  //   by_level  tiles by falling qt, and by b among equals, so that the longest walks
  //             begin first: with F(l) = sum_b max(0, nt_b - l) tiles from level l on, i
  //             lies on the highest level l with F(l) > i
  //   else      a sequence's tiles are neighbours, the last one first, so that its keys
  //             are read again from the L2 of the XCD that its heads run on, and
  //             sequences go by falling nt_b
  //   per       `per` tiles a sequence, some of which may not be: no search, the sequences
  //             in their order
  // More than 64 sequences that are searched go in their order too.  A search costs a
  // workgroup 1 to 4 us, which two others on its CU do not hide where walks are short.
  __device__ bool find_tile(const PromptArgs& a, int rows, int i, int& qt) {
    const int lane = threadIdx.x & 63;
    auto tiles = [&](int n) { return (n + rows - 1) / rows; };
    if (a.per) {
      const int b = a.by_level ? i % a.B : i / a.per;
      qt = a.per - 1 - (a.by_level ? i / a.B : i % a.per);
      if (b >= a.B) return false;
      seq_rows(a, __builtin_amdgcn_readfirstlane(b), row0, len);
      return true;
    }
    int64_t r0 = 0;
    int n = 0;
    if (a.B > 64) {
      // every lane adds up a run of sequences; the run that holds tile i is then looked
      // at by itself
      for (int first = 0, left = a.B; left > 0;) {
        const int run = (left + 63) / 64;
        int nt = 0;
#pragma unroll 4
        for (int s = lane * run; s < min((lane + 1) * run, left); ++s) {
          seq_rows(a, first + s, r0, n);
          nt += tiles(n);
        }
        const int inc = wave_scan(nt);
        const uint64_t m = __builtin_amdgcn_ballot_w64(i < inc);
        if (m == 0) return false;
        const int at = __builtin_ctzll(m);
        i -= __builtin_amdgcn_readlane(inc, at) - __builtin_amdgcn_readlane(nt, at);
        if (run == 1) {
          qt = __builtin_amdgcn_readlane(nt, at) - 1 - i;
          take(r0, n, at);
          return at < left;
        }
        first += at * run;
        left = min(run, left - at * run);
      }
      return false;
    }
    if (lane < a.B) seq_rows(a, lane, r0, n);
    const int nt = tiles(n);
    if (!a.by_level) {
      // the tiles of the sequences in front of this lane's
      const int64_t key = (int64_t)nt << 6 | (63 - lane);
      int before = 0;
      for (int s = 0; s < a.B; ++s) {
        const int x = __builtin_amdgcn_readlane(nt, s);
        before += ((int64_t)x << 6 | (63 - s)) > key ? x : 0;
      }
      const uint64_t m = __builtin_amdgcn_ballot_w64(i >= before && i < before + nt);
      if (m == 0) return false;
      const int b = __builtin_ctzll(m);
      qt = __builtin_amdgcn_readlane(nt + before, b) - 1 - i;
      take(r0, n, b);
      return true;
    }
    auto from_level = [&](int l) { return wave_sum(max(0, nt - l)); };
    if (from_level(0) <= i) return false;
    int lo = 0, hi = tiles(a.max_len);   // F(lo) > i >= F(hi) = 0
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (from_level(mid) > i) lo = mid; else hi = mid;
    }
    qt = lo;
    // the lane of rank i - F(lo + 1) among those with nt_b > lo (the sum by all lanes)
    const int want = i - from_level(lo + 1);
    const uint64_t m = __builtin_amdgcn_ballot_w64(nt > lo);
    const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
    const uint64_t it = __builtin_amdgcn_ballot_w64(nt > lo && rank == want);
    if (it == 0) return false;
    take(r0, n, __builtin_ctzll(it));
    return true;
  }
};

// The softmax state of a wave's 32 rows, lane (j, hh): row j, accumulator register r
// of o[d] dim 32 d + 8 (r / 4) + 4 hh + r % 4; l over this lane's keys.
template <typename T, int D>
__device__ void walk_rows(const PromptArgs& a, const Task& t, uint32_t bad, int first_row) {
  for (; bad; bad &= bad - 1) {
    const int i = first_row + __builtin_ctz(bad);
    if (i < t.len) row_walk<T, D>(a, t.row0, i, t.h);
  }
}

template <int kDB>
struct State {
  static constexpr int kFloats = 64 * kDB * 16 + 128;   // of a wave, in LDS
  float m, l;
  float16x o[kDB];

  __device__ void clear() {
    m = kLowest;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  }
  // The maximum of this lane's new scores, times qs; the running one, m + lift, is only
  // raised where some row's lies more than kSlack above it.
  __device__ void raise(float mx, float qs, float lift) {
    mx = both_max(mx) * qs - lift;
    if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
      const float m_new = fmaxf(m, mx), keep = fast_exp2(m - m_new);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int d = 0; d < kDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= keep;
    }
  }
  __device__ void put(float* to) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(to + ((d * 4 + g) * 64 + lane) * 4) =
            make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    *reinterpret_cast<float2*>(to + 64 * kDB * 16 + 2 * lane) = make_float2(m, l);
  }
  __device__ void add(const float* from) {
    const int lane = threadIdx.x & 63;
    const float2 ml = *reinterpret_cast<const float2*>(from + 64 * kDB * 16 + 2 * lane);
    const float mm = fmaxf(m, ml.x), w_s = fast_exp2(m - mm), w_o = fast_exp2(ml.x - mm);
    m = mm;
    l = l * w_s + ml.y * w_o;
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 x = *reinterpret_cast<const float4*>(from + ((d * 4 + g) * 64 + lane) * 4);
        o[d][4 * g] = o[d][4 * g] * w_s + x.x * w_o;
        o[d][4 * g + 1] = o[d][4 * g + 1] * w_s + x.y * w_o;
        o[d][4 * g + 2] = o[d][4 * g + 2] * w_s + x.z * w_o;
        o[d][4 * g + 3] = o[d][4 * g + 3] * w_s + x.w * w_o;
      }
  }
  // O over its sum; rows (a bit each) that are not finite.
  __device__ uint32_t normalise() {
    const float inv = 1.0f / both_sum(l);
    bool fine = true;
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        o[d][r] *= inv;
        fine = fine && fabsf(o[d][r]) < INFINITY;
      }
    const uint64_t bad = __builtin_amdgcn_ballot_w64(!fine);
    return (uint32_t)bad | (uint32_t)(bad >> 32);
  }
};

// The normalised rows of a wave, but for the bad ones.
template <typename T, int D>
__device__ inline void store_rows(const PromptArgs& a, const Task& t, int qrow, const State<D / 32>& st,
                                  uint32_t bad) {
  constexpr int kDB = D / 32;
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    uint8_t* dst = a.out + (((t.row0 + qrow) * a.H + t.h) * (int64_t)D) * 2;
    if (qrow < t.len && !((bad >> j) & 1)) {
  #pragma unroll
      for (int d = 0; d < kDB; ++d)
  #pragma unroll
        for (int g = 0; g < 2; ++g) {
          // lane halves hold 4 dims each of two groups of 8: swapped into one group each
          uint32_t w[4];
  #pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = Half<T>::pack(st.o[d][8 * g + 2 * e], st.o[d][8 * g + 2 * e + 1]);
          const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
          const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
          *reinterpret_cast<uint4*>(dst + 64 * d + 32 * g + 16 * hh) = make_uint4(x[0], y[0], x[1], y[1]);
        }
    }
  } else {
    uint8_t* dst = a.out + (((t.row0 + qrow) * a.H + t.h) * (int64_t)D) * 4;
    if (qrow < t.len && !((bad >> j) & 1)) {
  #pragma unroll
      for (int d = 0; d < kDB; ++d)
  #pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(dst + 128 * d + 32 * g + 16 * hh) =
              make_float4(st.o[d][4 * g], st.o[d][4 * g + 1], st.o[d][4 * g + 2], st.o[d][4 * g + 3]);
    }
  }
}

// This wave's loads have landed, but for the last `kLater`; behind the barrier
// everybody's have.
template <int kLater>
__device__ inline void landed() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLater) : "memory");
}

// 16-bit types.  KS groups of W / KS waves take KS neighbouring tiles of kBN keys each
// step, for the same rows, and put their states together at the end: twice the
// workgroups, each half as long, where there are few.
//
// A 32x32x16 product's accumulator register r of lane half h is row 8 (r / 4) + 4 h +
// r % 4, its operand wants 8 h + r % 8 (+ 16 (r / 8)); lane j of K's operand reading key
// swap23(j) turns the one into the other for the probabilities.
template <typename T, int D, int kBN, int KS, int W>
__global__ __launch_bounds__(64 * W, KS > 1 || D == 256 ? 1 : D == 64 && W == 4 ? 3 : 2) void prompt_mma_kernel(
    PromptArgs a) {
  constexpr int R = W / KS, kC = D / 8, kKeys = KS * kBN, kRowBytes = 2 * D;
  constexpr int kKB = kBN / 32, kDC = D / 16, kDB = D / 32;
  using KLoads = TileLoads<kC, kKeys, KPlace<kC>, 64 * W>;
  using VLoads = TileLoads<kC, kKeys, VPlace<kC>, 64 * W>;
  __shared__ __align__(1024) uint8_t lds[2][2][kKeys * kRowBytes];   // [K, V][even, odd tiles]

  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Task t;
  if (!t.find(a, 32 * R)) return;
  const int n_kt = (min(t.q0 + 32 * R, t.len) + kKeys - 1) / kKeys;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  KLoads kl;
  VLoads vl;
  kl.init(a.k + t.row0 * a.k_row + t.kvh * a.k_head, a.k_row, t.len, lds0, wave);
  vl.init(a.v + t.row0 * a.v_row + t.kvh * a.v_head, a.v_row, t.len, lds0 + sizeof(lds[0]), wave);
  kl.load(0);
  kl.load(1);
  vl.load(0);

  const int kg = wave / R;                      // which of the step's tiles
  const int first_row = t.q0 + 32 * (wave % R);
  const int qrow = first_row + j;               // of the sequence
  short8x qf[kDC];
  {
    const uint8_t* src = a.q + (t.row0 + min(qrow, t.len - 1)) * a.q_row + t.h * a.q_head + 16 * hh;
#pragma unroll
    for (int c = 0; c < kDC; ++c)
      qf[c] = *reinterpret_cast<const short8x*>(src + 32 * c);
    if (a.qscale < 0) {                  // the running max is of scores times |scale|
#pragma unroll
      for (int c = 0; c < kDC; ++c) qf[c] ^= (short)0x8000;
    }
  }
  // the queries are here before the loop: a wait for them inside it would wait for the
  // tiles on their way as well
#pragma unroll
  for (int c = 0; c < kDC; ++c) asm volatile("" : "+v"(qf[c]));
  // above 0, so that the -inf of a key behind the row stays one, and so small that no
  // finite score counts
  const float qs = fmaxf(fabsf(a.qscale), kLeastScale);
  State<kDB> st;
  st.clear();
  const int last_kt = min(first_row / kKeys, n_kt - 1);   // the only step with keys behind some row

  // Tile kt's turn: its V and the next tile's K have landed, behind the barrier
  // everybody's part of them; and everybody is done with what the next loads replace
  // (K of tile kt, V of the tile before).
  auto arrive = [&](int odd) {
    landed<0>();
    kl.load(odd);
    vl.load(1 - odd);
  };
  // Fragments: lane (j, hh) of K's gets elements 16 c + 8 hh .. of key swap23(j) of the
  // 32 of block kb; of V^T's V[key0 + 8 hh + e][32 d + j], where the transposing read
  // takes 8 bytes of row i / 4 from lane i of 16 and gives it column i.  The swizzles
  // depend on the lane alone, so every read is a lane's offset and a constant.
  const int kr = swap23(j), vi = j & 15;
  auto k_frag = [&](int odd, int i) {               // i = c kKB + kb
    const int c = i / kKB, kb = i % kKB;
    return *reinterpret_cast<const short8x*>(lds[0][odd] + 32 * kb * kRowBytes + (kg * kBN + kr) * kRowBytes +
                                             16 * KPlace<kC>::at(kr, 2 * c + hh));
  };
  auto v_frag = [&](int odd, int i) {               // i = (kb 2 + c) kDB + d
    typedef __attribute__((address_space(3))) short4x lshort4x;
    const int d = i % kDB, r = 8 * hh + (vi >> 2), e0 = 32 * d + (j & 16) + 4 * (vi & 3);
    const uint8_t* p = lds[1][odd] + 16 * (i / kDB) * kRowBytes;
    const short4x lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lshort4x*)(p + ((kg * kBN + r) * kRowBytes + 16 * VPlace<kC>::at(r, e0 / 8) + 2 * (e0 % 8))));
    const short4x hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lshort4x*)(p + 4 * kRowBytes +
                    ((kg * kBN + r) * kRowBytes + 16 * VPlace<kC>::at(r + 4, e0 / 8) + 2 * (e0 % 8))));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // Keys behind the row, in the wave's last tile.
  auto mask = [&](float16x (&s)[kKB]) {
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (last_kt * kKeys + kg * kBN + 32 * kb + 16 * (r / 8) + 8 * hh + r % 8 > qrow) s[kb][r] = -INFINITY;
  };
  constexpr int kQk = kKB * kDC, kPv = kKB * 2 * kDB;      // products of a tile
  constexpr int kPairs = kKB * 8;                          // pairs of scores of a lane
  constexpr int kAhead = kQk < 3 ? kQk : 3;                // fragments read ahead
  uint32_t pw[kPairs];                                     // probabilities, two a word
  auto prob = [&](float16x (&s)[kKB], int e) {
    const float x = fast_exp2(fmaf(s[e / 8][2 * (e % 8)], qs, -st.m));
    const float y = fast_exp2(fmaf(s[e / 8][2 * (e % 8) + 1], qs, -st.m));
    pw[e] = Half<T>::pack(x, y);
    st.l = Half<T>::sum2(pw[e], st.l);
  };
  auto pv = [&](short8x v, int i) {
    const int g = 4 * (i / kDB);
    st.o[i % kDB] = Half<T>::mma(v, __builtin_bit_cast(short8x, make_uint4(pw[g], pw[g + 1], pw[g + 2], pw[g + 3])),
                                 st.o[i % kDB]);
  };

  // One tile: S^T of the next one beside this one's exponentials, then O^T beside the
  // next one's maxima, product by product in this order (the barriers keep the compiler
  // from gathering them).
  float mx = 0.0f;
  auto step = [&](int odd, int kt, float16x (&sc)[kKB], float16x (&sn)[kKB]) {
    st.raise(mx, qs, Half<T>::kLift);
    arrive(odd);
    short8x kf[kQk], vf[kPv];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = k_frag(1 - odd, i);
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) sn[kb][r] = 0.0f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kQk; ++i) {
      const int n = i + kAhead;
      if (n < kQk) kf[n] = k_frag(1 - odd, n);
      else if (n - kQk < kPv) vf[n - kQk] = v_frag(odd, n - kQk);
      sn[i % kKB] = Half<T>::mma(kf[i], qf[i / kKB], sn[i % kKB]);
#pragma unroll
      for (int e = i * kPairs / kQk; e < (i + 1) * kPairs / kQk; ++e) prob(sc, e);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (kt + 1 == last_kt) mask(sn);
    mx = sn[0][0];
#pragma unroll
    for (int i = 0; i < kPv; ++i) {
      if (i + kAhead < kPv) vf[i + kAhead] = v_frag(odd, i + kAhead);
      pv(vf[i], i);
#pragma unroll
      for (int e = i * kPairs / kPv; e < (i + 1) * kPairs / kPv; ++e)
        mx = fmaxf(fmaxf(mx, sn[e / 8][2 * (e % 8)]), sn[e / 8][2 * (e % 8) + 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto finish = [&](int odd, float16x (&sc)[kKB]) {
    st.raise(mx, qs, Half<T>::kLift);
    arrive(odd);
#pragma unroll
    for (int e = 0; e < kPairs; ++e) prob(sc, e);
#pragma unroll
    for (int i = 0; i < kPv; ++i) pv(v_frag(odd, i), i);
  };

  float16x sa[kKB], sb[kKB];
  landed<KLoads::kLoads + VLoads::kLoads>();
#pragma unroll
  for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
    for (int r = 0; r < 16; ++r) sa[kb][r] = 0.0f;
#pragma unroll
  for (int i = 0; i < kQk; ++i) sa[i % kKB] = Half<T>::mma(k_frag(0, i), qf[i / kKB], sa[i % kKB]);
  if (last_kt == 0) mask(sa);
  mx = sa[0][0];
#pragma unroll
  for (int e = 0; e < kPairs; ++e) mx = fmaxf(fmaxf(mx, sa[e / 8][2 * (e % 8)]), sa[e / 8][2 * (e % 8) + 1]);
  int kt = 0;
  for (; kt + 1 < last_kt; kt += 2) {
    step(0, kt, sa, sb);
    step(1, kt + 1, sb, sa);
  }
  if (kt < last_kt) {
    step(0, kt, sa, sb);
    ++kt;
    finish(1, sb);
  } else {
    finish(0, sa);
  }
  while (++kt < n_kt) arrive(kt & 1);                     // the other waves' last tiles
  landed<0>();   // the last loads, before the LDS is used again or given up
  if constexpr (KS == 2) {
    float* other = reinterpret_cast<float*>(&lds[0][0][0]) + wave % R * State<kDB>::kFloats;
    static_assert(R * State<kDB>::kFloats * 4 <= (int)sizeof(lds), "states fit the LDS");
    if (kg > 0) st.put(other);
    __syncthreads();
    if (kg > 0) return;
    st.add(other);
  }

  const uint32_t bad = st.normalise();
  store_rows<T, D>(a, t, qrow, st, bad);
  walk_rows<T, D>(a, t, bad, first_row);
}

// fp32 on the bf16 matrix cores.  An fp32 number is the sum of three bf16 ones, each
// the leading 8 bits of what is left (cutting, not rounding, makes the remainders
// exact), so a product of two is six bf16 products,
//   hh + hm + mh + mm + hl + lh,
// the three left out being 2^-23 of it on average and 2^-21 at most, no more than what
// adding 32 products in fp32 may lose.  Numbers below 2^-102 keep fewer bits, bf16 having
// no smaller terms.  Six 32x32x16 products take 192 cycles
// where the fp32 ones of the same size (8 of v_mfma_f32_32x32x2_f32) take 512.  K and V
// are split once for the workgroup, from registers into three planes each in LDS; Q
// stays split in registers, and the probabilities are split where they stand.  An
// infinity splits into NaNs: its rows are not finite, and computed again (row_walk).
// One prompt of 2048 tokens, 32 / 8 heads, D 128: 202 us, 170 TFLOP/s of fp32 products
// (with the fp32 ones 377); 500 and 834 tokens, 12 heads, D 64: 26.3 us (37).  At D 128 the
// planes of Q fill the registers: 16 of them are kept in scratch memory where keys are
// split (4 loads of 16 bytes a step, beside 96 products), 4 where not (1 load).
struct Split3 {
  uint32_t h, m, l;   // two numbers each
  __device__ Split3(float x, float y) {
    const uint32_t xh = __float_as_uint(x) & 0xffff0000u, yh = __float_as_uint(y) & 0xffff0000u;
    x -= __uint_as_float(xh);
    y -= __uint_as_float(yh);
    const uint32_t xm = __float_as_uint(x) & 0xffff0000u, ym = __float_as_uint(y) & 0xffff0000u;
    x -= __uint_as_float(xm);
    y -= __uint_as_float(ym);
    h = __builtin_amdgcn_perm(yh, xh, 0x07060302u);
    m = __builtin_amdgcn_perm(ym, xm, 0x07060302u);
    l = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
  }
};

// The three planes of sign times 8 numbers.
__device__ inline void split8(const float4& x, const float4& y, float sign, short8x (&to)[3]) {
  const Split3 a(sign * x.x, sign * x.y), b(sign * x.z, sign * x.w), c(sign * y.x, sign * y.y),
      d(sign * y.z, sign * y.w);
  to[0] = __builtin_bit_cast(short8x, make_uint4(a.h, b.h, c.h, d.h));
  to[1] = __builtin_bit_cast(short8x, make_uint4(a.m, b.m, c.m, d.m));
  to[2] = __builtin_bit_cast(short8x, make_uint4(a.l, b.l, c.l, d.l));
}

// acc + a . b, planes h, m, l, the small terms first.
__device__ inline float16x mma3(const short8x (&a)[3], const short8x (&b)[3], float16x acc) {
  acc = Half<Bf16>::mma(a[2], b[0], acc);
  acc = Half<Bf16>::mma(a[0], b[2], acc);
  acc = Half<Bf16>::mma(a[1], b[1], acc);
  acc = Half<Bf16>::mma(a[1], b[0], acc);
  acc = Half<Bf16>::mma(a[0], b[1], acc);
  return Half<Bf16>::mma(a[0], b[0], acc);
}

template <int D, int kBN, int KS, int W>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void prompt_f32_kernel(PromptArgs a) {
  constexpr int kThreads = 64 * W, R = W / KS, kC = D / 8, kKeys = KS * kBN, kRowBytes = 2 * D;
  constexpr int kKB = kBN / 32, kDC = D / 16, kDB = D / 32;
  constexpr int kLoads = kKeys * D / 4 / kThreads;   // of 4 elements, a thread, K and V each
  static_assert(kLoads >= 1 && kLoads * kThreads * 4 == kKeys * D, "tile / thread split");
  __shared__ __align__(1024) uint8_t lds[2][3][kKeys * kRowBytes];   // [K, V][planes]

  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Task t;
  if (!t.find(a, 32 * R)) return;
  const int n_kt = (min(t.q0 + 32 * R, t.len) + kKeys - 1) / kKeys;
  const int kg = wave / R, first_row = t.q0 + 32 * (wave % R);
  const int qrow = first_row + j;   // of the sequence

  // This thread's part of a tile: rows lr, lr + kStep, .. at elements 4 lc .. + 3.
  constexpr int kStep = kThreads / (D / 4);
  const int lr = threadIdx.x / (D / 4), lc = threadIdx.x % (D / 4);
  const uint8_t* kbase = a.k + t.row0 * a.k_row + t.kvh * a.k_head + 16 * lc;
  const uint8_t* vbase = a.v + t.row0 * a.v_row + t.kvh * a.v_head + 16 * lc;
  float4 kr[kLoads], vr[kLoads];
  auto load = [&](int kt) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t key = min(kt * kKeys + u * kStep + lr, t.len - 1);   // (past the last: masked)
      kr[u] = *reinterpret_cast<const float4*>(kbase + key * a.k_row);
      vr[u] = *reinterpret_cast<const float4*>(vbase + key * a.v_row);
    }
  };
  auto put = [&](uint8_t (*to)[kKeys * kRowBytes], int at, const float4& x) {
    const Split3 p(x.x, x.y), q(x.z, x.w);
    *reinterpret_cast<uint2*>(to[0] + at) = make_uint2(p.h, q.h);
    *reinterpret_cast<uint2*>(to[1] + at) = make_uint2(p.m, q.m);
    *reinterpret_cast<uint2*>(to[2] + at) = make_uint2(p.l, q.l);
  };
  load(0);

  short8x qf[kDC][3];
  {
    const uint8_t* src = a.q + (t.row0 + min(qrow, t.len - 1)) * a.q_row + t.h * a.q_head + 32 * hh;
    const float sign = a.qscale < 0 ? -1.0f : 1.0f;   // the running max is of scores times |scale|
#pragma unroll
    for (int c = 0; c < kDC; ++c) {
      const float4 x = *reinterpret_cast<const float4*>(src + 64 * c);
      const float4 y = *reinterpret_cast<const float4*>(src + 64 * c + 16);
      split8(x, y, sign, qf[c]);
    }
  }
  const float qs = fmaxf(fabsf(a.qscale), kLeastScale);

  State<kDB> st;
  st.clear();
  const int kl = swap23(j), vi = j & 15;
  const int last_kt = min(first_row / kKeys, n_kt - 1);   // the only step with keys behind some row
  for (int kt = 0; kt < n_kt; ++kt) {
    __syncthreads();                   // everybody is done with the tile before
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int r = u * kStep + lr;
      put(lds[0], r * kRowBytes + 16 * KPlace<kC>::at(r, lc / 2) + 8 * (lc & 1), kr[u]);
      put(lds[1], r * kRowBytes + 16 * VPlace<kC>::at(r, lc / 2) + 8 * (lc & 1), vr[u]);
    }
    if (kt + 1 < n_kt) load(kt + 1);
    // the tile is there; the next one's loads stay on their way
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (kt > last_kt) continue;        // the other waves' last steps
    float16x s[kKB];
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.0f;
#pragma unroll
    for (int c = 0; c < kDC; ++c)
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
        short8x kf[3];
#pragma unroll
        for (int p = 0; p < 3; ++p)
          kf[p] = *reinterpret_cast<const short8x*>(lds[0][p] + (kg * kBN + 32 * kb + kl) * kRowBytes +
                                                    16 * KPlace<kC>::at(kl, 2 * c + hh));
        s[kb] = mma3(kf, qf[c], s[kb]);
      }
    if (kt == last_kt) {
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kt * kKeys + kg * kBN + 32 * kb + 16 * (r / 8) + 8 * hh + r % 8 > qrow) s[kb][r] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
    st.raise(mx, qs, 0.0f);
    short8x pf[kKB * 2][3];
#pragma unroll
    for (int g = 0; g < kKB * 2; ++g) {
      uint32_t w[3][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = fast_exp2(fmaf(s[g / 2][8 * (g % 2) + 2 * e], qs, -st.m));
        const float y = fast_exp2(fmaf(s[g / 2][8 * (g % 2) + 2 * e + 1], qs, -st.m));
        st.l += x + y;
        const Split3 p(x, y);
        w[0][e] = p.h;
        w[1][e] = p.m;
        w[2][e] = p.l;
      }
#pragma unroll
      for (int p = 0; p < 3; ++p)
        pf[g][p] = __builtin_bit_cast(short8x, make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]));
    }
#pragma unroll
    for (int g = 0; g < kKB * 2; ++g)
#pragma unroll
      for (int d = 0; d < kDB; ++d) {
        typedef __attribute__((address_space(3))) short4x lshort4x;
        const int r = 8 * hh + (vi >> 2), e0 = 32 * d + (j & 16) + 4 * (vi & 3);
        short8x vf[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          const uint8_t* at = lds[1][p] + (kg * kBN + 16 * g + r) * kRowBytes + 2 * (e0 % 8);
          vf[p] = __builtin_shufflevector(
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lshort4x*)(at + 16 * VPlace<kC>::at(r, e0 / 8))),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (lshort4x*)(at + 4 * kRowBytes + 16 * VPlace<kC>::at(r + 4, e0 / 8))),
              0, 1, 2, 3, 4, 5, 6, 7);
        }
        st.o[d] = mma3(vf, pf[g], st.o[d]);
      }
  }
  __syncthreads();
  if constexpr (KS > 1) {
    // the groups' states, one after the other through one place in the LDS
    float* place = reinterpret_cast<float*>(&lds[0][0][0]) + wave % R * State<kDB>::kFloats;
    static_assert(R * State<kDB>::kFloats * 4 <= (int)sizeof(lds), "states fit the LDS");
#pragma unroll
    for (int k = 1; k < KS; ++k) {
      if (kg == k) st.put(place);
      __syncthreads();
      if (kg == 0) st.add(place);
      __syncthreads();
    }
    if (kg > 0) return;
  }
  const uint32_t bad = st.normalise();
  store_rows<float, D>(a, t, qrow, st, bad);
  walk_rows<float, D>(a, t, bad, first_row);
}

// ---- short prompts: a wave by itself ----------------------------------------

// A wave takes 32 rows of one (sequence, head) and shares nothing: the workgroup's waves
// are just neighbours (heads of a KV group, whose keys the L1 then holds; us at 1 / 2 / 4
// waves: 8 of 64 tokens, 8 / 4 heads, D 256 9.8 / 11.2 / 14.9, 300 of 100 on average, 32 / 8
// heads, D 128 268 / 253 / 232).  Its tile's number says which sequence and rows it is, `per`
// tiles a sequence, so nothing is searched for, and many fit a CU, so their loads hide one
// another: 512 prompts of 16 tokens, 32 / 8 heads, D 128, bf16 54 us, 3.1 TB/s.  K's operands come
// straight from memory (a lane's 16 bytes of one key).  V's: 16-bit types pass through
// 32 rows of LDS, for the transposing read; of fp32 a lane loads 8 keys' numbers of
// one dim, 128 neighbouring bytes a half wave.
constexpr int kWaves = 2;

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) void prompt_wave_kernel(PromptArgs a) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kC = D / 8, kDC = D / 16, kDB = D / 32, kRowBytes = 2 * D;
  __shared__ __align__(1024) uint8_t lds[kWaves][kF32 ? 16 : 32 * kRowBytes];
  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)blockIdx.x * kWaves + wave;
  const int64_t tile = item / a.H;
  const int64_t b = tile / a.per;
  if (b >= a.B) return;
  Task t;
  t.h = (int)(item - tile * a.H);
  t.kvh = t.h / (a.H / a.Hkv);
  seq_rows(a, (int)b, t.row0, t.len);
  t.row0 = readlane64(t.row0);
  t.len = __builtin_amdgcn_readfirstlane(t.len);
  const int qt = a.per - 1 - (int)(tile - b * a.per);
  t.q0 = 32 * qt;
  if (t.q0 >= t.len) return;
  const int qrow = t.q0 + j;
  const uint8_t* qp = a.q + (t.row0 + min(qrow, t.len - 1)) * a.q_row + t.h * a.q_head;
  const uint8_t* kb = a.k + t.row0 * a.k_row + t.kvh * a.k_head;
  const uint8_t* vb = a.v + t.row0 * a.v_row + t.kvh * a.v_head;
  const int kl = swap23(j), vi = j & 15;
  const float sign = a.qscale < 0 ? -1.0f : 1.0f;
  const float qs = fmaxf(fabsf(a.qscale), kLeastScale);
  const uint32_t to = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds[wave]);
  State<kDB> st;
  st.clear();
  short8x qf[kF32 ? 1 : kDC];
  if constexpr (!kF32) {
#pragma unroll
    for (int c = 0; c < kDC; ++c) {
      qf[c] = *reinterpret_cast<const short8x*>(qp + 32 * c + 16 * hh);
      if (a.qscale < 0) qf[c] ^= (short)0x8000;
    }
  }
  for (int kt = 0; kt <= qt; ++kt) {
    const uint8_t* krow = kb + (int64_t)min(32 * kt + kl, t.len - 1) * a.k_row;
    float16x s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
    if constexpr (kF32) {
#pragma unroll
      for (int c = 0; c < kDC; ++c) {
        const float4 x = *reinterpret_cast<const float4*>(krow + 64 * c + 32 * hh);
        const float4 y = *reinterpret_cast<const float4*>(krow + 64 * c + 32 * hh + 16);
        const float4 u = *reinterpret_cast<const float4*>(qp + 64 * c + 32 * hh);
        const float4 w = *reinterpret_cast<const float4*>(qp + 64 * c + 32 * hh + 16);
        short8x kf[3], qk[3];
        split8(x, y, 1.0f, kf);
        split8(u, w, sign, qk);
        s = mma3(kf, qk, s);
      }
    } else {
      short8x kf[kDC];
#pragma unroll
      for (int c = 0; c < kDC; ++c) kf[c] = *reinterpret_cast<const short8x*>(krow + 32 * c + 16 * hh);
      constexpr int kStep = 64 / kC;   // rows of a load
      const uint8_t* base = vb + (int64_t)32 * kt * a.v_row;
      const int left = t.len - 32 * kt;
#pragma unroll
      for (int u = 0; u < 32 / kStep; ++u) {
        const int r = u * kStep + lane / kC;
        load_to_lds(base, (uint32_t)min(r, left - 1) * (uint32_t)a.v_row + 16 * VPlace<kC>::at(r, lane % kC),
                    to + u * 1024);
      }
#pragma unroll
      for (int c = 0; c < kDC; ++c) s = Half<T>::mma(kf[c], qf[c], s);
    }
    if (kt == qt) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * kt + 16 * (r / 8) + 8 * hh + r % 8 > qrow) s[r] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    if constexpr (kF32) st.raise(mx, qs, 0.0f);
    else st.raise(mx, qs, Half<T>::kLift);
    if constexpr (kF32) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = fast_exp2(fmaf(s[r], qs, -st.m));
        st.l += p[r];
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        short8x pf[3];
        split8(make_float4(p[8 * g], p[8 * g + 1], p[8 * g + 2], p[8 * g + 3]),
               make_float4(p[8 * g + 4], p[8 * g + 5], p[8 * g + 6], p[8 * g + 7]), 1.0f, pf);
        const int key0 = 32 * kt + 16 * g + 8 * hh;
#pragma unroll
        for (int d = 0; d < kDB; ++d) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = *reinterpret_cast<const float*>(vb + (int64_t)min(key0 + e, t.len - 1) * a.v_row +
                                                   128 * d + 4 * j);
          short8x vf[3];
          split8(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), 1.0f, vf);
          st.o[d] = mma3(vf, pf, st.o[d]);
        }
      }
    } else {
      uint32_t pw[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pw[e] = Half<T>::pack(fast_exp2(fmaf(s[2 * e], qs, -st.m)), fast_exp2(fmaf(s[2 * e + 1], qs, -st.m)));
        st.l = Half<T>::sum2(pw[e], st.l);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const short8x pf = __builtin_bit_cast(
            short8x, make_uint4(pw[4 * g], pw[4 * g + 1], pw[4 * g + 2], pw[4 * g + 3]));
#pragma unroll
        for (int d = 0; d < kDB; ++d) {
          typedef __attribute__((address_space(3))) short4x lshort4x;
          const int r = 8 * hh + (vi >> 2), e0 = 32 * d + (j & 16) + 4 * (vi & 3);
          const uint8_t* at = lds[wave] + (16 * g + r) * kRowBytes + 2 * (e0 % 8);
          const short8x vf = __builtin_shufflevector(
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lshort4x*)(at + 16 * VPlace<kC>::at(r, e0 / 8))),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (lshort4x*)(at + 4 * kRowBytes + 16 * VPlace<kC>::at(r + 4, e0 / 8))),
              0, 1, 2, 3, 4, 5, 6, 7);
          st.o[d] = Half<T>::mma(vf, pf, st.o[d]);
        }
      }
      // the reads are done before the next tile's loads replace what they read
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
  const uint32_t bad = st.normalise();
  store_rows<T, D>(a, t, qrow, st, bad);
  walk_rows<T, D>(a, t, bad, t.q0);
}

// Tiles of `rows` rows of all sequences, at most.
int64_t tiles_of(const PromptArgs& a, int rows) {
  return std::min(sat_mul(a.B, ceil_div(a.max_len, rows)), a.T / rows + a.B);
}

// Workgroups of 32 W / KS rows.
template <typename T, int D, int kBN, int KS, int W>
int launch_one(PromptArgs a, hipStream_t stream) {
  constexpr int rows = 32 * W / KS;
  const int64_t per = ceil_div(a.max_len, rows), fewest = tiles_of(a, rows);
  // Tiles by their number where that launches no empty workgroups, or saves the search
  // through a thousand sequences.  us, searched for / by number: 64 prompts of 200 tokens,
  // 32 / 8 heads, D 128 117 / 92; 1024 of 100 903 / 650; 4000 of 1 to 300, 8 heads, D 64
  // 2207 / 719; 400 of 128 to 1000, 8 / 4 heads, D 256 1600 / 1800.
  a.per = sat_mul(a.B, per) <= (a.B < 1024 ? 1 : 2) * fewest ? (int)per : 0;
  const int64_t grid = sat_mul(a.per ? a.B * per : fewest, a.H);
  if (!grid_fits(grid, 64 * W)) return fail(HS_EUNSUPPORTED, "prompt grid too large");
  if constexpr (sizeof(T) == 4)
    hipLaunchKernelGGL((prompt_f32_kernel<D, kBN, KS, W>), dim3((unsigned)grid), dim3(64 * W), 0, stream, a);
  else
    hipLaunchKernelGGL((prompt_mma_kernel<T, D, kBN, KS, W>), dim3((unsigned)grid), dim3(64 * W), 0, stream, a);
  return HS_OK;
}

template <typename T, int D>
int launch_waves(PromptArgs a, hipStream_t stream) {
  a.per = (int)ceil_div(a.max_len, 32);
  const int64_t grid = ceil_div(sat_mul(a.B, a.per, a.H), kWaves);
  if (!grid_fits(grid, 64 * kWaves)) return fail(HS_EUNSUPPORTED, "prompt grid too large");
  hipLaunchKernelGGL((prompt_wave_kernel<T, D>), dim3((unsigned)grid), dim3(64 * kWaves), 0, stream, a);
  return HS_OK;
}

// Few workgroups of 128 rows split the keys over their waves: the longest walk, which the
// others' CUs would wait for, is half as long, for twice the set-up and a merge.  How many
// are few depends on how many fit a CU and on the walk's length.  us, one group of 4 waves /
// two of 2 (fp32: four of 2, at D 128 two of 4), workgroups in brackets:
//   D 128  2 at a time a CU: 1 prompt of 512 tokens, 32 / 8 heads (128 workgroups) 16.0 / 14.3,
//          640 (160) 18.2 / 18.2, 3 of 200, 32 heads (192) 11.7 / 16.7, 1024 (256) 24.1 / 26.3
//   D 256  1 at a time: 8 / 4 heads, 1 of 4096 (256) 134 / 114, 4 of 1024 (256) 43.2 / 45.6, 4736
//          (296) 147 / 153
//   D 64   12 heads, 4 of 640 (240) 13.1 / 11.7, 16 of 256 (384) 10.4 / 14.0; long walks: 2 of 1536
//          (288) 23.0 / 18.1, 2 of 2048 (384) 29.9 / 28.1, 2 of 2688 (504) 40.1 / 39.9
//   D 32   8 heads, 4 of 1024 (256) 14.2 / 11.0, 64 of 512 (2048) 36 / 73; long walks: 2 of 4096
//          (512) 41.2 / 37.5, 4 of 3200 (800) 46.0 / 44.6, 8 of 4096 (2048) 118 / 148
//   fp32   D 64, 12 heads: 500 and 834 (132) 46 / 28.5, 16 of 256 (384) 24 / 36; long walks: 3 of
//          1024 (288) 54 / 51, 2 of 2048 (384) 106 / 100, 1 of 6784 (636) 406 / 450
//          D 32, 8 heads, long walks: 1 of 8192 (512) 242 / 230, 2 of 6400 (800) 264 / 268
//          D 128 (2 at a time a CU, with 2 groups of 4 waves 1), 32 / 8 heads: 1 of 300 (96) 36 / 31,
//          4 of 300 (384) 48 / 55; long walks: 2048 (512) 233 / 202, 3200 (800) 441 / 468
template <typename T, int D>
bool few(const PromptArgs& a, int cus) {
  const int64_t n = sat_mul(tiles_of(a, 128), a.H);
  if constexpr (sizeof(T) == 2) {
    if (D == 128) return n <= (int64_t)cus * 5 / 8;
    if (D <= 64 && a.max_len >= 1536) return n <= (int64_t)cus * (D == 64 ? 3 : 6) / 2;
  } else {
    if (D == 128) return a.max_len > 256 && n <= (int64_t)cus * (a.max_len >= 512 ? 2 : 1);
    if (D <= 64 && a.max_len >= 1024) return n <= (int64_t)cus * (D == 64 ? 3 : 5) / 2;
  }
  return n <= cus;
}

// Short prompts take a wave each.  us, workgroups as above / waves: 512 of 16 tokens, 32 / 8
// heads, D 128 253 / 54; 8 of 64 10.6 / 8.7; 256 of 64 154 / 108; 256 of 128 194 / 255; fp32, 12
// heads, D 64, 512 of 16 115 / 26; 256 of 64 64 / 45.  fp32 heads of 128 and more need more of a
// wave than it can hide: 32 / 8 heads, D 128, 512 of 16 359 / 139, 16 of 24 13.5 / 12.2, 1 of 24
// 9.5 / 12.2, 256 of 64 271 / 277.
//
// Prompts of up to 768 tokens and different lengths (four fifths of the longest on average,
// or less) take, in 16-bit types or at head dims 32 and 64, workgroups of 2 waves, 64 rows, and steps of 32 keys: fewer rows
// past an end, and four workgroups a CU where two fitted, whose set-ups overlap.  us, 4 waves
// / 2, evenly spread lengths: 1 to 200, 32 / 8 heads, D 128, 64 prompts 57 / 45, 300 276 / 227;
// 1 to 400, 32 prompts 56 / 50; 200 to 400, 40 prompts 103 / 93; 1 to 700, 32 prompts 106 / 95;
// 1 to 1000, 64 prompts 370 / 370; 1 to 2000, 32 prompts 485 / 502; all of one length: 128 of 256
// tokens 221 / 228, 256 of 128, 12 heads, D 64 39 / 49; 1 to 200, 64 prompts, 32 / 8 heads, D 32
// 22.9 / 17.3, 8 / 4 heads, D 256 43 / 37; fp32, 12 heads, D 64 44 / 37, 32 / 8 heads, D 32
// 45 / 32, D 128 155 / 179, which splits each key's numbers for half the rows.
template <typename T, int D>
int launch_dim(const PromptArgs& a, int cus, hipStream_t stream) {
  constexpr bool kLarge = sizeof(T) == 4 && D >= 128;
  if (a.max_len <= (kLarge ? 32 : 64) && (!kLarge || sat_mul(a.B, a.H) >= 2 * cus))
    return launch_waves<T, D>(a, stream);
  const bool split = few<T, D>(a, cus);
  if constexpr (!kLarge)
    if (!split && a.max_len <= 768 && 5 * a.T <= 4 * sat_mul(a.B, a.max_len))
      return launch_one<T, D, 32, 1, 2>(a, stream);
  if constexpr (sizeof(T) == 2) {
    constexpr int kBN = D >= 256 ? 32 : 64;
    return split ? launch_one<T, D, kBN, 2, 4>(a, stream) : launch_one<T, D, kBN, 1, 4>(a, stream);
  } else if constexpr (D <= 64) {
    return split ? launch_one<T, D, 32, 4, 8>(a, stream) : launch_one<T, D, 64, 1, 4>(a, stream);
  } else if constexpr (D == 128) {
    return split ? launch_one<T, D, 32, 2, 8>(a, stream) : launch_one<T, D, 32, 1, 4>(a, stream);
  } else {
    return launch_one<T, D, 32, 1, 4>(a, stream);
  }
}

template <typename T>
int launch_type(const PromptArgs& a, int D, int cus, hipStream_t stream) {
  switch (D) {
    case 32: return launch_dim<T, 32>(a, cus, stream);
    case 64: return launch_dim<T, 64>(a, cus, stream);
    case 128: return launch_dim<T, 128>(a, cus, stream);
    case 256: return launch_dim<T, 256>(a, cus, stream);
    default: return fail(HS_EUNSUPPORTED, "unsupported head_dim " + std::to_string(D));
  }
}

}  // namespace

// Strides in elements; the sizes and pointers are checked (hs_api.hip).
int launch_prompt(const Prompt& w, int cus, hipStream_t stream) {
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
  // the keys and values of all heads stay in the XCDs' L2s (4 MB each)
  a.by_level = sat_mul(w.T, w.Hkv, w.D, 2 * sb) <= 8 * (4 << 20);
  profile_begin(stream);
  int rc;
  if (w.dtype == HS_DTYPE_F32) rc = launch_type<float>(a, w.D, cus, stream);
  else if (w.dtype == HS_DTYPE_F16) rc = launch_type<_Float16>(a, w.D, cus, stream);
  else rc = launch_type<Bf16>(a, w.D, cus, stream);
  profile_end(stream);
  return rc == HS_OK ? check_launch("prompt attention") : rc;
}

}  // namespace hs
