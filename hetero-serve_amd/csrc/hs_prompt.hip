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

// ---- matrix cores, 16-bit types ---------------------------------------------

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
struct Half;
template <>
struct Half<Bf16> {
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
  __device__ static float16x mma(short8x a, short8x b, float16x c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2x){a, b}, f16x2));
  }
};

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

// 16 bytes from every lane's address to LDS, at the wave's byte offset `to` + 16 lane;
// counted by vmcnt.  As a builtin, the compiler waits for all such loads before every
// transposing read.  No output register is in flight, and nothing else here uses m0.
__device__ inline void load_to_lds(const uint8_t* p, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(p)
               : "memory");
}

// Where the 16-byte chunk c of row r lies in its LDS row of kC chunks: K rows are
// read 16 at a time at one chunk, V rows 4 at a time at 4 neighbouring chunks, and
// each pattern shall cover all 64 banks.
template <int kC>
__device__ inline int k_place(int r, int c) {
  if constexpr (kC >= 16) return c ^ (r & 15);
  else if constexpr (kC == 8) return c ^ ((r >> 1) & 7);
  else return c ^ ((r >> 2) & 3);
}
template <int kC>
__device__ inline int v_place(int r, int c) {
  if constexpr (kC >= 16) return c ^ ((r & 3) << 2);
  else if constexpr (kC == 8) return c ^ (((r >> 1) & 1) << 2);
  else return c;
}

// The tile of query rows that workgroup `i` takes: tiles of all sequences, those
// that walk the most keys first.  nt_b tiles of `rows` rows in sequence b; tile
// qt of it walks qt + 1 tiles of keys, so the tiles go by falling qt, and by b
// among equals: with F(l) = sum_b max(0, nt_b - l) tiles from level l on, i lies
// on the highest level l with F(l) > i.  Every wave finds it by itself.  False:
// there is no such tile.
__device__ inline bool find_tile(const PromptArgs& a, int rows, int64_t i, int& b, int& qt) {
  const int lane = threadIdx.x & 63;
  auto tiles = [&](int s) {
    int64_t row0;
    int len;
    if (s >= a.B) return 0;
    seq_rows(a, s, row0, len);
    return (len + rows - 1) / rows;
  };
  auto from_level = [&](int l) {
    int64_t f = 0;
    for (int s0 = 0; s0 < a.B; s0 += 64) {
      int x = max(0, tiles(s0 + lane) - l);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
      f += x;
    }
    return f;
  };
  if (from_level(0) <= i) return false;
  int lo = 0, hi = (a.max_len + rows - 1) / rows;   // F(lo) > i >= F(hi) = 0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (from_level(mid) > i) lo = mid; else hi = mid;
  }
  qt = lo;
  int64_t k = i - from_level(lo + 1);               // the k-th sequence with nt_b > lo
  for (int s0 = 0; s0 < a.B; s0 += 64) {
    uint64_t m = __builtin_amdgcn_ballot_w64(tiles(s0 + lane) > lo);
    const int n = __builtin_popcountll(m);
    if (k < n) {
      for (; k > 0; --k) m &= m - 1;
      b = s0 + __builtin_ctzll(m);
      return true;
    }
    k -= n;
  }
  return false;
}

// A workgroup: W waves of 32 query rows of one (sequence, head).  It walks the keys
// in tiles of kBN, K and V going from global memory straight to LDS, kStages tiles
// deep.  S^T = K Q^T and O^T = V^T P^T on 32x32x16 products, so that a lane holds one
// query's scores and the probabilities are the second product's operand where they
// stand: accumulator register r of lane half h is row 8 (r / 4) + 4 h + r % 4, the
// operand wants 8 h + r % 8 (+ 16 (r / 8)), and lane j reading key swap23(j) turns
// the one into the other.
template <typename T, int D, int W, int kBN, int kStages>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void prompt_mma_kernel(PromptArgs a) {
  constexpr int kRows = 32 * W, kC = D / 8, kThreads = 64 * W;
  constexpr int kRowBytes = 2 * D, kTile = kBN * kRowBytes;
  constexpr int kLoads = kTile / (16 * kThreads);   // 16-byte loads of a thread, K and V each
  constexpr int kKB = kBN / 32, kDC = D / 16, kDB = D / 32;
  static_assert(kLoads >= 1 && kLoads * 16 * kThreads == kTile, "tile / thread split");
  __shared__ __align__(1024) uint8_t lds[kStages][2][kTile];

  const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // neighbouring workgroups: the heads of one tile, a KV head's group on one XCD
  const int hp = blockIdx.x % a.H;
  const int h = hp % a.Hkv * (a.H / a.Hkv) + hp / a.Hkv, kvh = hp % a.Hkv;
  int b, qt;
  if (!find_tile(a, kRows, blockIdx.x / a.H, b, qt)) return;
  b = __builtin_amdgcn_readfirstlane(b);
  int64_t row0;
  int len;
  seq_rows(a, b, row0, len);
  const int q0 = qt * kRows;
  const int n_kt = (min(q0 + kRows, len) + kBN - 1) / kBN;

  const uint8_t* kbase = a.k + row0 * a.k_row + kvh * a.k_head;
  const uint8_t* vbase = a.v + row0 * a.v_row + kvh * a.v_head;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds);
  // Keys past the sequence are read as its last one (and masked).
  auto load_tile = [&](int kt, int stage) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int at = (u * W + wave) * 64 + lane;      // 16-byte place in the tile
      const int r = at / kC, p = at % kC;
      const int64_t key = min(kt * kBN + r, len - 1);
      const uint32_t to = lds0 + (uint32_t)(2 * stage * kTile + (u * W + wave) * 1024);
      load_to_lds(kbase + key * a.k_row + 16 * k_place<kC>(r, p), to);
      load_to_lds(vbase + key * a.v_row + 16 * v_place<kC>(r, p), to + kTile);
    }
  };

  const int qrow = q0 + 32 * wave + j;   // of the sequence
  short8x qf[kDC];
  {
    const uint8_t* src = a.q + (row0 + min(qrow, len - 1)) * a.q_row + h * a.q_head + 16 * hh;
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
  // above 0, so that the -inf of a key behind the row stays one
  const float qs = fmaxf(fabsf(a.qscale), 1e-30f);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load_tile(s, s);

  float m = kNegBig, l = 0.0f;
  float16x o[kDB];
#pragma unroll
  for (int d = 0; d < kDB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;

  const int first_row = q0 + 32 * wave;
  int stage = 0;
  for (int kt = 0; kt < n_kt; ++kt) {
    // this wave's loads of tile kt have landed (those of later tiles may be on
    // their way); behind the barrier everybody's have, and everybody is done with
    // tile kt - 1, whose place the next loads take
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * kLoads * (kStages - 2)) : "memory");
    {
      int next = stage + kStages - 1;
      if (next >= kStages) next -= kStages;
      load_tile(kt + kStages - 1, next);
    }
    const uint8_t* ks = lds[stage][0];
    const uint8_t* vs = lds[stage][1];
    if (++stage == kStages) stage = 0;
    const int k0 = kt * kBN;
    if (k0 > first_row + 31) continue;   // every key lies behind this wave's rows

    float16x s[kKB];
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.0f;
    const int kr = swap23(j);
#pragma unroll
    for (int c = 0; c < kDC; ++c)
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
        const short8x kf = *reinterpret_cast<const short8x*>(
            ks + (32 * kb + kr) * kRowBytes + 16 * k_place<kC>(kr, 2 * c + hh));
        s[kb] = Half<T>::mma(kf, qf[c], s[kb]);
      }
    if (k0 + kBN - 1 > first_row) {      // some row does not see some key
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * kb + 16 * (r / 8) + 8 * hh + r % 8 > qrow) s[kb][r] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
    mx = both_max(mx) * qs;
    if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
      const float m_new = fmaxf(m, mx), keep = fast_exp2(m - m_new);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int d = 0; d < kDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= keep;
    }
    short8x pf[kKB][2];
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = fast_exp2(fmaf(s[kb][8 * c + 2 * e], qs, -m));
          const float y = fast_exp2(fmaf(s[kb][8 * c + 2 * e + 1], qs, -m));
          l += x + y;
          w[e] = Half<T>::pack(x, y);
        }
        pf[kb][c] = __builtin_bit_cast(short8x, make_uint4(w[0], w[1], w[2], w[3]));
      }
    // V^T: lane (j, hh) gets V[key0 + 8 hh + e][32 d + j]; the transposing read takes
    // 8 bytes of row i / 4 from lane i of 16 and gives it column i
    const int vi = j & 15;
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 0; d < kDB; ++d) {
          const int r = 32 * kb + 16 * c + 8 * hh + (vi >> 2);
          const int e0 = 32 * d + (j & 16) + 4 * (vi & 3);   // element of the row
          typedef __attribute__((address_space(3))) short4x lshort4x;
          const short4x lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lshort4x*)(vs + r * kRowBytes + 16 * v_place<kC>(r, e0 / 8) + 2 * (e0 % 8)));
          const short4x hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lshort4x*)(vs + (r + 4) * kRowBytes + 16 * v_place<kC>(r + 4, e0 / 8) + 2 * (e0 % 8)));
          o[d] = Half<T>::mma(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pf[kb][c], o[d]);
        }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last loads land before the LDS is given up

  // A value behind a row that is infinite or NaN has been added times 0: rows that
  // are not finite are computed again, without those keys.
  const float inv = 1.0f / both_sum(l);
  bool fine = true;
  uint8_t* dst = a.out + (((row0 + qrow) * a.H + h) * (int64_t)D) * 2;
#pragma unroll
  for (int d = 0; d < kDB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      o[d][r] *= inv;
      fine = fine && fabsf(o[d][r]) < INFINITY;
    }
  uint64_t bad = __builtin_amdgcn_ballot_w64(!fine && qrow < len);
  uint32_t bad_rows = (uint32_t)bad | (uint32_t)(bad >> 32);
  if (qrow < len && !((bad_rows >> j) & 1)) {
#pragma unroll
    for (int d = 0; d < kDB; ++d)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        // lane halves hold 4 dims each of two groups of 8: swapped into one group each
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = Half<T>::pack(o[d][8 * g + 2 * e], o[d][8 * g + 2 * e + 1]);
        const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        *reinterpret_cast<uint4*>(dst + 64 * d + 32 * g + 16 * hh) = make_uint4(x[0], y[0], x[1], y[1]);
      }
  }
  for (; bad_rows; bad_rows &= bad_rows - 1)
    row_walk<T, D>(a, row0, first_row + __builtin_ctz(bad_rows), h);
}

template <typename T>
int launch_dim(const PromptArgs& a, int D, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    const int W = D == 256 || D == 32 ? 4 : 8, rows = 32 * W;
    const int64_t tiles = std::min(sat_mul(a.B, ceil_div(a.max_len, rows)), a.T / rows + a.B);
    const int64_t grid = sat_mul(tiles, a.H);
    if (grid > 0x7fffffffLL) return fail(HS_EUNSUPPORTED, "prompt grid too large");
    const dim3 g((unsigned)grid), t(64 * W);
    switch (D) {
      case 32: hipLaunchKernelGGL((prompt_mma_kernel<T, 32, 4, 64, 3>), g, t, 0, stream, a); break;
      case 64: hipLaunchKernelGGL((prompt_mma_kernel<T, 64, 8, 64, 3>), g, t, 0, stream, a); break;
      case 128: hipLaunchKernelGGL((prompt_mma_kernel<T, 128, 8, 64, 3>), g, t, 0, stream, a); break;
      case 256: hipLaunchKernelGGL((prompt_mma_kernel<T, 256, 4, 32, 3>), g, t, 0, stream, a); break;
      default: return fail(HS_EUNSUPPORTED, "unsupported head_dim " + std::to_string(D));
    }
    return HS_OK;
  }
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
