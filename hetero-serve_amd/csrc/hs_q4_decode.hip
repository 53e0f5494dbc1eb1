// Decode over a 4-bit cache (hs_q4.h) on the matrix cores, through spans (hs_span.h).
//
// With k = n - 8 and mid = lo + 8 s, a group's middle, an element is k s + mid, and
//   score_t = sum_d (k_td s_tg + mid_tg) q_d = sum_g s_tg (sum_{d in g} k_td q_d) + sum_g mid_tg Q_g
//   out_d   = sum_t p_t (k_td s_tg + mid_tg) = sum_t (p_t s_tg) k_td + sum_t p_t mid_tg
// where g = d / 32 is the element's group and Q_g the sum of the query over it.  So whole
// numbers go to the products, and s is applied to fp32 sums (keys) or to the fp32
// probabilities (values); the elements themselves are never made.  With n and lo in the
// place of k and mid, the two sums are several times larger than what they add up to, and
// so was the error: 8e-6 of the row where it is 4e-7, at 4096 keys.  The sums over the mids are
// small: the keys' goes to the matrix cores, the values' and that of p are fp32 sums of the
// vector units.
//
// Numerics.  A nibble in the low bits of 1024's mantissa is 1024 + n, or 1024 + 16 n four bits
// further up; less 1032 or 1152 they are k and 16 k, exactly, and the 16 is taken out of the
// other operand.  (As masked, without the 1024, they are the subnormals n 2^-24, which the
// matrix cores take, but they align sums by the operands' exponents: an accuracy of 2^-16 was
// left.)  Query and probabilities are fp32 and go in as two fp16 terms, hi + lo, which have 22 bits
// down to 2^-3 and end at 2^-24.  A query's are times the power of two that brings its head's largest
// element to [2^14, 2^15), its sums times one that is 2^kQueryUp less, so that 8 times a sum is below
// 2^15: what is lost of an element is at most 2^-35 of the largest, of a sum 2^-31.  A key's mid is
// not made: mid Q is lo Q + s 8 Q, of halves as they are stored.
//   p s has a power of two R for each head and group, which follows the largest p s that the wave
// has met: it brings that to [2^12, 2^13), and is chosen again when one passes 2^15.  When the row's
// maximum rises, and the sums so far count for less, R rises with it.  So what is lost is 2^-32 of
// the largest one, as far as fp32 sums reach, however small p is next to the row's largest (a first
// key that takes nearly all of the weight and has next to no values), and whatever the steps of
// other groups and of keys without weight.  Products of such terms are exact in the fp32
// accumulators.
//
// A wave serves up to 16 query heads of one KV head over one part of a row's visible keys,
// 64 keys (a chunk) at a time:
//   S^T = K Q^T      16x16x32, A: 16 keys x 32 dims, a group a product, so that its sums can
//                    be scaled by the group's steps.  The record's order puts what a lane
//                    wants of all groups side by side: D / 8 bytes, one load for 16 keys.
//   O^T += V^T P^T   16x16x32, A: 16 dims x 32 keys, values transposed on their way out of LDS
//                    by ds_read_b64_tr_b4, which gives a lane 16 keys of one dim.
// Which key is which row of the first product is free; taking key 16 (j / 4) + 4 r + j % 4 for
// row j of product r leaves each lane with the 16 probabilities of the keys that the
// transposing read gives it.  They never leave the registers.
// Waves share nothing before their states are put together, so the walk has no barriers.  Keys
// past the part's end are read as its last one and count nothing: their scores are -inf.
//
// Times of a call in a graph, D 128, 32 / 8 heads: 64 rows of 16..4096 keys, 168 MB, 58 us (46 this
// kernel), of 2048 each 51.5, of 8192 each, 671 MB, 159 (4.2 TB/s; with parts of 512 keys and
// coarser sums 163, 152 of it without the arithmetic, 118 without the loads).  16 rows of 8k..32k, 419
// MB, 107 (100).  Loads two chunks ahead, three waves a SIMD and waves' priorities gained
// nothing.
#include "hs_kernels.h"
#include "hs_kvrows.h"
#include "hs_q4.h"
#include "hs_span_mma.h"

#include <algorithm>

// Contraction would take (float)(_Float16)x for x and leave a split's second term 0.
#pragma clang fp contract(off)

namespace hs {

namespace {

using namespace span_mma;

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef int int2x __attribute__((ext_vector_type(2)));

constexpr int kChunk = 64;         // keys of a step
// The largest p s so far times R is at most 2^kMost; when a larger one comes R is chosen so that
// it lies below 2^kAim.  R is 2^kFree at most.
constexpr int kMost = 15, kAim = 13, kFree = 127;
constexpr int kQueryUp = 8;        // powers of 2 that the query is held above its sums

// What a wave keeps in LDS: its chunk's records as they were loaded, and of its steps and its
// values' middles what lies by key there by group, so that a lane's 16 keys are a few 16-byte
// reads.  (Rows of records are 20 dwords apart at D 128: the keys' 16-byte reads of 16 rows
// cover all banks, the values' transposing ones half of them.)
template <int D>
struct Chunk {
  static constexpr int G = D / kQ4Group, kPar = kChunk + 8;
  alignas(16) uint8_t k[kChunk][q4_record_bytes(D)];
  alignas(16) uint8_t v[kChunk][(q4_record_bytes(D) + 7) / 8 * 8];   // (8-byte reads)
  alignas(16) _Float16 ks[G][kPar];
  alignas(16) _Float16 vs[G][kPar];
  alignas(16) float vmid[G][kPar];
};

template <int N>
struct Words {
  uint32_t w[N];
};

template <int N>
__device__ inline Words<N> load_words(const uint8_t* p) {
  Words<N> x;
  if constexpr (N == 1) {
    x.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    x.w[0] = t.x, x.w[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 t = load16(p + 4 * i);
      x.w[i] = t.x, x.w[i + 1] = t.y, x.w[i + 2] = t.z, x.w[i + 3] = t.w;
    }
  }
  return x;
}

// The k of a word's 8 numbers as operand halves, of elements 0 4 1 5 2 6 3 7, those of the second
// and fourth pair 16 times larger.  The masks are held in registers that the compiler does not
// see through, so that an and and an or are one instruction (as literals they are two).
struct Unpack {
  uint32_t low = 0x000f000fu, high = 0x00f000f0u, k1024 = 0x64006400u;

  __device__ Unpack() {
    asm("" : "+s"(low), "+s"(high));
    asm("" : "+v"(k1024));
  }
  __device__ half8 operator()(uint32_t x) const {
    const uint32_t y = x >> 8;
    constexpr _Float16 a = 1024.0f + 8.0f, b = 1024.0f + 128.0f;
    return __builtin_bit_cast(half8, make_uint4((x & low) | k1024, (x & high) | k1024, (y & low) | k1024,
                                                (y & high) | k1024)) -
           half8{a, a, b, b, a, a, b, b};
  }
};
// The element of a word that half e of Unpack's is.
__device__ constexpr int half_element(int e) { return (e >> 1) + 4 * (e & 1); }

__device__ inline float4x mma(half8 a, half8 b, float4x c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The terms, hi + lo with 22 bits, of keys 16 g + 8 t ..: their p s in the order of Unpack's halves,
// x of the first four and y of the others, times R (R / 16 where the key is odd).  An instruction
// for each term, where the compiler takes several.  One that writes half a register is not
// followed by one that reads it: a wait is needed between those.
__device__ inline void split_terms(const float4x& x, const float4x& y, float even, float odd, half8& hi,
                                   half8& lo) {
  uint32_t h0, h1, h2, h3, l0, l1, l2, l3;
  asm("v_fma_mixlo_f16 %0, %8, %16, 0\n\t"
      "v_fma_mixlo_f16 %1, %9, %17, 0\n\t"
      "v_fma_mixlo_f16 %2, %10, %16, 0\n\t"
      "v_fma_mixlo_f16 %3, %11, %17, 0\n\t"
      "v_fma_mixhi_f16 %0, %12, %16, 0\n\t"
      "v_fma_mixhi_f16 %1, %13, %17, 0\n\t"
      "v_fma_mixhi_f16 %2, %14, %16, 0\n\t"
      "v_fma_mixhi_f16 %3, %15, %17, 0\n\t"
      "v_fma_mixlo_f16 %4, %8, %16, -%0 op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixlo_f16 %5, %9, %17, -%1 op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixlo_f16 %6, %10, %16, -%2 op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixlo_f16 %7, %11, %17, -%3 op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %4, %12, %16, -%0 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %5, %13, %17, -%1 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %6, %14, %16, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %7, %15, %17, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "s_nop 1"
      : "=&v"(h0), "=&v"(h1), "=&v"(h2), "=&v"(h3), "=&v"(l0), "=&v"(l1), "=&v"(l2), "=&v"(l3)
      : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(y[0]), "v"(y[1]), "v"(y[2]), "v"(y[3]), "v"(even),
        "v"(odd));
  hi = __builtin_bit_cast(half8, make_uint4(h0, h1, h2, h3));
  lo = __builtin_bit_cast(half8, make_uint4(l0, l1, l2, l3));
}

template <int N>
__device__ inline void store_words(uint8_t* p, const Words<N>& x) {
  if constexpr (N == 1) *reinterpret_cast<uint32_t*>(p) = x.w[0];
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(p) = make_uint2(x.w[0], x.w[1]);
  else
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<uint4*>(p + 4 * i) = make_uint4(x.w[i], x.w[i + 1], x.w[i + 2], x.w[i + 3]);
}

// Half i of packed halves.
template <int N>
__device__ inline _Float16 half_of(const Words<N>& x, int i) {
  return __builtin_bit_cast(_Float16, (uint16_t)(x.w[i / 2] >> (16 * (i & 1))));
}

// The 16 columns of the products are 16 / S heads times S shares of the groups: column j has head
// j / S's sums over groups j % S * G / S .. alone.  So a lane scales its scores by G / S groups'
// steps, adds the shares up with its neighbours, and makes the second product's operand
// for these groups instead of all: 64 rows of 16..4096 keys, D 128, 32 / 8 heads, took 91 us with
// S = 4 where they took 119 with 1; behind a window of 4096, 32 / 4 heads, 48 with S = 2, 54 with 1.
template <int D, int S>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : D == 128 ? 2 : 3) void q4_decode_kernel(SpanArgs a) {
  constexpr int G = D / kQ4Group, kPiece = D / 8, kT = D / 16;
  constexpr int kRecord = q4_record_bytes(D), kLoads = kRecord / kPiece;   // 5 pieces a record
  constexpr int kHeads = kSlots / S;     // of a wave
  constexpr int kShare = G / S;          // groups of a column
  constexpr int kMid = G == 8 ? 8 : 4;   // groups that a lane has of the product of the mids
  __shared__ Chunk<D> chunks[kWaves];
  __shared__ float2 states[kWaves][kSlots];
  static_assert(kHeads * (D + 4) * 4 <= (int)sizeof(Chunk<D>), "a wave's outputs fit");
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  Task t;
  if (!t.find(a, kHeads, kChunk)) return;
  Chunk<D>& w = chunks[t.wv];
  const int jh = j / S, js = j % S;      // this column's head, share
  const Span span(a, t.b);
  int lo, hi, nparts;
  if (!span.part(a, t.part, t.p, lo, hi, nparts)) {   // all of the workgroup
    if (span.n == 0 && t.p == -a.P) zero_rows<D>(a, t);
    return;
  }
  const int32_t* bt = a.bt + (int64_t)t.b * a.MB;
  const uint32_t tok = (uint32_t)a.Hkv * kRecord;
  const uint8_t* kbase = a.k + (int64_t)t.kvh * kRecord;
  const uint8_t* vbase = a.v + (int64_t)t.kvh * kRecord;

  // A chunk's records come in pieces of D / 8 bytes, 64 lanes neighbouring pieces, and go to
  // LDS through registers: a chunk's loads are on their way while the one before is computed,
  // its slots' table entries while the one before that is.
  // (Operands straight from memory, the numbers and then the steps: 3.6 TB/s for the loads
  // alone; whole records 4.2.)
  Words<G> kr[kLoads], vr[kLoads];
  auto load = [&](int slot) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = lane + 64 * i, key = c / kLoads;
      const uint64_t at = (uint64_t)(uint32_t)__shfl(slot, key) * tok + (c - key * kLoads) * kPiece;
      kr[i] = load_words<G>(kbase + at);
      vr[i] = load_words<G>(vbase + at);
    }
  };
  const int step = kChunk * t.np, first = lo + kChunk * t.ph;
  auto place_of = [&](int c0) { return span.place(a, bt, min(c0 + lane, hi - 1)); };
  Span::Place ahead{};
  if (first < hi) {
    ahead = place_of(first + step);
    load(Span::slot(a, place_of(first)));
  }

  // The query in two terms, in the order of the keys' halves, and its sums by group.
  const Unpack unpack;
  half8 qf[G][2];
  _Float16 qsum[kMid];
  float back;     // what scores are to be multiplied by
  {
    const float* qp = a.q + (t.row0 + min(jh, t.gc - 1)) * D + 8 * g;
    const float sc = jh < t.gc ? a.qscale : 0.0f;
    float x[G][8], most = 0.0f;
#pragma unroll
    for (int st = 0; st < G; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[st][e] = qp[32 * st + e] * sc;
        most = fmaxf(most, fabsf(x[st][e]));
      }
    most = max_across_groups(most);
    int up = 0;
    if (most > 0.0f && most < INFINITY) up = min(7 - __builtin_amdgcn_frexp_expf(most), 120);
    back = ldexpf(1.0f, -up - kQueryUp);
    float sums[G];
#pragma unroll
    for (int st = 0; st < G; ++st) {
      sums[st] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[st][e] = ldexpf(x[st][e], up);
        sums[st] += x[st][e];
      }
      sums[st] = sum_across_groups(sums[st]);
      const bool mine = st / kShare == js;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = mine ? x[st][half_element(e)] * (float)(1 << (e & 2 ? kQueryUp - 4 : kQueryUp)) : 0.0f;
        qf[st][0][e] = (_Float16)y;
        qf[st][1][e] = (_Float16)(y - (float)qf[st][0][e]);
      }
    }
    // term g % 2 of the sums, against the lowest values, and of 8 of them, against the steps
#pragma unroll
    for (int e = 0; e < kMid; ++e) {
      const float y = e < G && e / kShare == js ? sums[e % G] * (g < 2 ? 1.0f : 8.0f) : 0.0f;
      const _Float16 h = (_Float16)y;
      qsum[e] = g & 1 ? (_Float16)(y - (float)h) : h;
    }
  }

  // Over this lane's keys: the sum l of p, and of p mid for each group of the share.  The outputs
  // are held times R, of the group's column.
  float4x o[kT];
  float om[kShare], R[kShare], l = 0.0f;
#pragma unroll
  for (int d = 0; d < kT; ++d) o[d] = float4x{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kShare; ++i) {
    om[i] = 0.0f;
    R[i] = ldexpf(1.0f, kFree);
  }
  float m = kLowest;

  for (int c0 = first; c0 < hi; c0 += step) {
    const bool last = hi - c0 < kChunk;   // uniform
    lds_order();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      store_words(w.k[0] + (lane + 64 * i) * kPiece, kr[i]);
      const int c = lane + 64 * i;
      store_words(w.v[0] + c * kPiece + (D == 32 ? c / kLoads * ((int)sizeof(w.v[0]) - kRecord) : 0), vr[i]);
    }
    if (c0 + step < hi) {
      const int slot = Span::slot(a, ahead);
      ahead = place_of(c0 + 2 * step);
      load(slot);
    }
    lds_order();
    {
      const Words<G> kp = load_words<G>(w.k[lane] + D / 2), vp = load_words<G>(w.v[lane] + D / 2);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        w.ks[i][lane] = half_of(kp, i);
        w.vs[i][lane] = half_of(vp, i);
        w.vmid[i][lane] = fmaf((float)half_of(vp, i), 8.0f, (float)half_of(vp, G + i));
      }
    }
    lds_order();

    Words<G> kw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) kw[i] = load_words<G>(w.k[16 * (j >> 2) + 4 * i + (j & 3)] + g * kPiece);
    // scores of keys 16 g + 4 i + e, for column j: the mids' part, then the steps'
    float4x s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // lowest values (lane groups 0 and 1) and steps of a key
      const _Float16* km = reinterpret_cast<const _Float16*>(w.k[16 * (j >> 2) + 4 * i + (j & 3)] + D / 2) +
                           (g < 2 ? G : 0);
      const float4x none = {0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (G == 8) {
        half8 q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = qsum[e];
        s[i] = mma(*reinterpret_cast<const half8*>(km), q, none);
      } else {
        half4 x = {(_Float16)0.0f, (_Float16)0.0f, (_Float16)0.0f, (_Float16)0.0f}, q;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e < G) x[e] = km[e % G];
          q[e] = qsum[e];
        }
        s[i] = __builtin_amdgcn_mfma_f32_16x16x16f16(x, q, none, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] *= (float)(1 << kQueryUp);
    }
#pragma unroll
    for (int i = 0; i < kShare; ++i) {   // group i of every share
      float4x x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = float4x{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int st = i; st < G; st += kShare)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const half8 kf = unpack(kw[r].w[st]);
          x[r] = mma(kf, qf[st][0], x[r]);
          x[r] = mma(kf, qf[st][1], x[r]);
        }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const half8 ks = *reinterpret_cast<const half8*>(&w.ks[js * kShare + i][16 * g + 8 * t]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int r = 2 * t + e / 4;
          s[r][e % 4] = fmaf((float)ks[e], x[r][e % 4], s[r][e % 4]);
        }
      }
    }
    if constexpr (S > 1) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][e] = group_sum<S>(s[r][e]);
    }
    if (last) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * g + 4 * i + e >= hi - c0) s[i][e] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[i][e]);
    mx *= back;
    if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
      const float m_new = fmaxf(m, max_across_groups(mx)), by = m_new - m, keep = fast_exp2(-by);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        // R grows as what is there shrinks: what comes may be as small
        const int more = min((int)fminf(by, 2.0f * kFree), kFree + 1 - __builtin_amdgcn_frexp_expf(R[i]));
        R[i] = ldexpf(R[i], more);
        om[i] *= keep;
        const float times = ldexpf(keep, more);
#pragma unroll
        for (int d = 0; d < kT; ++d)
          if (d / 2 % kShare == i) o[d] *= times;
      }
    }
    // (A chunk's sums are their own: fewer roundings where terms have one sign.)
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = fast_exp2(fmaf(s[i][e], back, -m));
        sum += s[i][e];
      }
    l += sum;
#pragma unroll
    for (int i = 0; i < kShare; ++i) {   // group i of every share
      float4x ps[4];
      float most = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const half8 vs = *reinterpret_cast<const half8*>(&w.vs[js * kShare + i][16 * g + 8 * t]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int r = 2 * t + e / 4;
          ps[r][e % 4] = fmaf(s[r][e % 4], (float)vs[e], 0.0f);   // (one instruction)
          most = fmaxf(most, fabsf(ps[r][e % 4]));
        }
      }
      float mids = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float4x mid = *reinterpret_cast<const float4x*>(&w.vmid[js * kShare + i][16 * g + 4 * r]);
#pragma unroll
        for (int e = 0; e < 4; ++e) mids = fmaf(s[r][e], mid[e], mids);
      }
      om[i] += mids;
      if (__builtin_amdgcn_ballot_w64(most * R[i] > ldexpf(1.0f, kMost)) != 0) {
        most = max_across_groups(most);
        if (most * R[i] > ldexpf(1.0f, kMost) && most < INFINITY) {
          const int less = kAim + 1 - __builtin_amdgcn_frexp_expf(most) - __builtin_amdgcn_frexp_expf(R[i]);
          const float times = ldexpf(1.0f, less);
          R[i] = ldexpf(R[i], less);
#pragma unroll
          for (int d = 0; d < kT; ++d)
            if (d / 2 % kShare == i) o[d] *= times;
        }
      }
      half8 hi2[2], lo2[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
        split_terms(ps[2 * t], ps[2 * t + 1], R[i], R[i] * 0x1p-4f, hi2[t], lo2[t]);
#pragma unroll
      for (int d = 2 * i; d < kT; d += d % 2 ? 2 * kShare - 1 : 1) {
        typedef __attribute__((address_space(3))) int2x lds_int2x;
        const int2x x = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_int2x*)(w.v[lane] + 8 * d));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const half8 vf = unpack((uint32_t)x[t]);
          o[d] = mma(vf, hi2[t], o[d]);
          o[d] = mma(vf, lo2[t], o[d]);
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < kShare; ++i) {
    const float mid = sum_across_groups(om[i]), over = 1.0f / R[i];
#pragma unroll
    for (int d = 0; d < kT; ++d)
      if (d / 2 % kShare == i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] = fmaf(o[d][e], over, mid);
  }
  finish<D, kHeads>(
      a, t, nparts == 1, o, m, sum_across_groups(l), jh, js == 0 && g == 0, [&](int d) { return js == d / 2 / kShare; },
      [&](int wave) { return reinterpret_cast<float*>(&chunks[wave]); }, states);
}

// Columns of a head: as many as leave a wave the KV head's query heads, the groups at most.
int shares(int H, int Hkv, int D) {
  int s = D / kQ4Group;
  while (s > 1 && H / Hkv * s > kSlots) s /= 2;
  return s;
}

template <int D, int S>
void launch_one(const SpanArgs& a, hipStream_t stream) {
  const int64_t wgs = workgroups(a, kSlots / S);
  hipLaunchKernelGGL((q4_decode_kernel<D, S>), dim3((unsigned)wgs), dim3(64 * kWaves), 0, stream, a);
}

template <int D, int S = D / kQ4Group>
void launch_dim(const SpanArgs& a, hipStream_t stream) {
  if constexpr (S > 1)
    if (shares(a.H, a.Hkv, D) < S) return launch_dim<D, S / 2>(a, stream);
  launch_one<D, S>(a, stream);
}

}  // namespace

// us, D 128, 32 / 8 heads, heads side by side x keys of a part (as planned, before they are
// fitted): 64 rows of 64..512 keys 4 x 512
// 24, 2 x 512 17.9, 1 x 512 19.8; 1 of 512 1 x 512 10.2, 4 x 64 10.5; 8 of 1024..2048 4 x 128 15.9,
// 2 x 256 16.7, 1 x 512 17.5; 64 of 16..4096 2 x 512 63, 4 x 512 66, 1 x 1024 68; 16 of 8k..32k
// 4 x 512 119, 2 x 1024 120, 4 x 1024 126; 1 of 4096 1 x 256 13.0, 4 x 64 15.2.
void q4_decode_plan(int B, int H, int Hkv, int D, int64_t most, bool windowed, int cus, int* part,
                    int* heads, int* room, int* longest) {
  const int hpw = kSlots / shares(H, Hkv, D);
  plan(B, H, Hkv, hpw, kChunk, most, windowed, cus, part, heads);
  *longest = kLongest * kChunk * kWaves / *heads;
  *room = parts_on_chip(B, H, Hkv, hpw, *heads, cus * (D == 256 ? 1 : D == 128 ? 2 : 3));
}

// The parts' states or rows; the caller merges.
int launch_q4_decode(const SpanArgs& a, int D, hipStream_t stream) {
  if (!grid_fits(workgroups(a, kSlots / shares(a.H, a.Hkv, D)), 64 * kWaves))
    return fail(HS_EUNSUPPORTED, "grid too large: sequences * parts * KV heads");
  switch (D) {
    case 32: launch_dim<32>(a, stream); break;
    case 64: launch_dim<64>(a, stream); break;
    case 128: launch_dim<128>(a, stream); break;
    case 256: launch_dim<256>(a, stream); break;
    default: return fail(HS_EUNSUPPORTED, "unsupported head_dim " + std::to_string(D));
  }
  return HS_OK;
}

}  // namespace hs
