// Decode over spans (hs_span.h) of fp16 and bf16 caches on the matrix cores, head dims 32, 64
// and 128; fp32 caches and head dim 256 are served by the vector units (hs_span_decode.hip).
//
// A wave serves up to 16 query heads of one KV head over one part of a row's visible keys, 32
// keys (a chunk) at a time:
//   S^T = K Q^T      16x16x32, A: 16 keys x 32 dims from LDS, B: the query, columns heads
//   O^T += V^T P^T   16x16x32, A: 16 dims x 32 keys, values transposed on their way out of LDS
//                    by ds_read_b64_tr_b16.  Row 4 g + i of the first product's tile r is key
//                    16 r + 4 g + i, and lane group g's keys of the second one are these for r
//                    = 0, 1 and i = 0 .. 3, so the probabilities stay where they are.
// Rows of keys and values are loaded whole, neighbouring lanes 16 bytes, a chunk ahead of the
// one that is computed, and go through LDS as they came.  Keys past the part's end are read as
// its last one, with scores of -inf.
//
// Numerics.  Keys and values are multiplied as they are stored.  Query and probabilities are
// fp32 and go in as terms of the cache's type.  Three bf16 ones have fp32's 24 bits and range
// (two would have 16).  Two fp16 ones have 22 bits down to 2^-3 and end at 2^-24.  So each head's
// query is first brought to [2^14, 2^15) by a power of two, taken back out of its scores, and what
// is lost of an element is at most 2^-39 of the largest.  The probabilities of a chunk are taken in
// ranges of 2^18, one in nearly all chunks: the largest of each head is brought there likewise, those
// down to 2^-3 go to the matrix cores, and the rest is taken in the same way until none is left, since
// the values of the larger ones may be next to nothing (a first key that takes nearly all of the
// weight).  Products of such terms are exact in the fp32 accumulators.
//
// Bound by HBM: behind a window of 1024, 64 rows of 32 / 8 heads, D 128, 265 MB, take 46 us of bf16 (5.8
// TB/s), 47.5 of fp16, 32 rows of 32 heads 90 of fp16 (5.9 TB/s); small batches by their steps'
// latency.
#include "hs_kernels.h"
#include "hs_kvrows.h"
#include "hs_span_mma.h"

// Contraction would take (float)(T)x for x and leave a split's other terms 0.
#pragma clang fp contract(off)

namespace hs {

namespace {

using namespace span_mma;

typedef short short4x __attribute__((ext_vector_type(4)));
typedef short short8x __attribute__((ext_vector_type(8)));
typedef float float2x __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 32;         // keys of a step

template <typename T>
struct Half;   // kTerms of its type a number
template <>
struct Half<Bf16> {
  static constexpr int kTerms = 3;
  __device__ static float4x mma(short8x a, short8x b, float4x c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                   c, 0, 0, 0);
  }
  __device__ static uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2x){x, y}, bf16x2));
  }
  __device__ static void rest(uint32_t w, float& x, float& y) {
    x -= __uint_as_float(w << 16);
    y -= __uint_as_float(w & 0xffff0000u);
  }
};
template <>
struct Half<_Float16> {
  static constexpr int kTerms = 2;
  __device__ static float4x mma(short8x a, short8x b, float4x c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                  0, 0, 0);
  }
  __device__ static uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2x){x, y}, f16x2));
  }
  __device__ static void rest(uint32_t w, float& x, float& y) {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    x -= (float)h[0];
    y -= (float)h[1];
  }
};

// The terms of 8 numbers.
template <typename T>
__device__ inline void split8(float (&x)[8], short8x (&term)[Half<T>::kTerms]) {
#pragma unroll
  for (int n = 0; n < Half<T>::kTerms; ++n) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = Half<T>::pack(x[2 * i], x[2 * i + 1]);
      asm("" : "+v"(w[i]));   // what is taken off is the term as used
      Half<T>::rest(w[i], x[2 * i], x[2 * i + 1]);
    }
    term[n] = __builtin_bit_cast(short8x, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// One chunk in LDS, rows as loaded.  Row paddings: keys are read as 16-byte fragments, 16 rows
// at one place, values by the transposing read, 4 rows at 16 neighbouring dims: at D + 8 and
// D + 16 elements apart, both cover the banks evenly.
template <int D>
struct Chunk {
  alignas(16) uint16_t k[kChunk][D + 8];
  alignas(16) uint16_t v[kChunk][D + 16];
};

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, 2) void window_decode_kernel(SpanArgs a) {
  using H = Half<T>;
  constexpr int kLanes = D / 8, kRows = 64 / kLanes, kLoads = kChunk / kRows;   // of a row; a load; a chunk
  constexpr int kSteps = D / 32, kT = D / 16, kTerms = H::kTerms;
  __shared__ Chunk<D> chunks[kWaves];
  __shared__ float2 states[kWaves][kSlots];
  static_assert(kSlots * (D + 4) * 4 <= (int)sizeof(Chunk<D>), "a wave's outputs fit");
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  Task t;
  if (!t.find(a, kSlots, kChunk)) return;
  Chunk<D>& w = chunks[t.wv];
  const Span span(a, t.b);
  int lo, hi, nparts;
  if (!span.part(a, t.part, t.p, lo, hi, nparts)) {   // all of the workgroup
    if (span.n == 0 && t.p == -a.P) zero_rows<D>(a, t);
    return;
  }
  const int32_t* bt = a.bt + (int64_t)t.b * a.MB;
  const uint32_t tok = (uint32_t)a.Hkv * D * 2;
  const uint8_t* kbase = a.k + ((int64_t)t.kvh * D + lane % kLanes * 8) * 2;
  const uint8_t* vbase = a.v + ((int64_t)t.kvh * D + lane % kLanes * 8) * 2;

  uint4 kr[kLoads], vr[kLoads];
  auto load = [&](int slot) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint64_t at = (uint64_t)(uint32_t)__shfl(slot, i * kRows + lane / kLanes) * tok;
      kr[i] = load16_stream(kbase + at);
      vr[i] = load16_stream(vbase + at);
    }
  };
  const int step = kChunk * t.np, first = lo + kChunk * t.ph;
  auto place_of = [&](int c0) { return span.place(a, bt, min(c0 + lane % kChunk, hi - 1)); };
  Span::Place ahead{};
  if (first < hi) {
    ahead = place_of(first + step);
    load(Span::slot(a, place_of(first)));
  }

  // The query's terms: dims 32 st + 8 g .. of column j.
  short8x qf[kSteps][kTerms];
  float back = 1.0f;     // what scores are to be multiplied by
  {
    const float* qp = a.q + (t.row0 + min(j, t.gc - 1)) * D + 8 * g;
    const float sc = j < t.gc ? a.qscale : 0.0f;
    float x[kSteps][8], most = 0.0f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[st][e] = qp[32 * st + e] * sc;
        most = fmaxf(most, fabsf(x[st][e]));
      }
    if constexpr (kTerms == 2) {
      most = max_across_groups(most);
      int up = 0;
      if (most > 0.0f && most < INFINITY) up = min(15 - __builtin_amdgcn_frexp_expf(most), 120);
      back = ldexpf(1.0f, -up);
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[st][e] = ldexpf(x[st][e], up);
    }
#pragma unroll
    for (int st = 0; st < kSteps; ++st) split8<T>(x[st], qf[st]);
  }

  float4x o[kT];
#pragma unroll
  for (int d = 0; d < kT; ++d) o[d] = float4x{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kLowest, l = 0.0f;    // l over this lane's keys

  for (int c0 = first; c0 < hi; c0 += step) {
    lds_order();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      *reinterpret_cast<uint4*>(&w.k[i * kRows + lane / kLanes][lane % kLanes * 8]) = kr[i];
      *reinterpret_cast<uint4*>(&w.v[i * kRows + lane / kLanes][lane % kLanes * 8]) = vr[i];
    }
    if (c0 + step < hi) {
      const int slot = Span::slot(a, ahead);
      ahead = place_of(c0 + 2 * step);
      load(slot);
    }
    lds_order();

    // scores of keys 16 r + 4 g + i, for column j
    float4x s[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      s[r] = float4x{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const short8x kf = *reinterpret_cast<const short8x*>(&w.k[16 * r + j][32 * st + 8 * g]);
#pragma unroll
        for (int n = 0; n < kTerms; ++n) s[r] = H::mma(kf, qf[st][n], s[r]);
      }
    }
    if (hi - c0 < kChunk) {      // uniform
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * r + 4 * g + i >= hi - c0) s[r][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[r][i]);
    mx *= back;
    if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
      const float m_new = fmaxf(m, max_across_groups(mx)), keep = fast_exp2(m - m_new);
      m = m_new;
      l *= keep;
#pragma unroll
      for (int d = 0; d < kT; ++d) o[d] *= keep;
    }
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = fast_exp2(fmaf(s[e / 4][e % 4], back, -m));
      l += p[e];
    }
    // V[16 (e / 4) + 4 g + e % 4][16 d + j], e = 0 .. 7: lane i of 16 supplies 8 bytes of row i / 4
    auto values = [&](int d) {
      typedef __attribute__((address_space(3))) short4x lds_short4x;
      const uint16_t* at = &w.v[4 * g + (j >> 2)][16 * d + 4 * (j & 3)];
      return __builtin_shufflevector(
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4x*)at),
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4x*)(at + 16 * (D + 16))), 0, 1, 2, 3, 4, 5, 6, 7);
    };
    short8x pf[kTerms];
    if constexpr (kTerms == 3) {
      split8<T>(p, pf);
#pragma unroll
      for (int d = 0; d < kT; ++d) {
        const short8x vf = values(d);
        float4x sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int n = kTerms - 1; n >= 0; --n) sum = H::mma(vf, pf[n], sum);
        o[d] += sum;
      }
    } else {
      bool more;
      do {
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, p[e]);
        const int up = min(15 - __builtin_amdgcn_frexp_expf(max_across_groups(most)), 127);
        const float over = ldexpf(1.0f, -up), least = up < 127 ? 0.125f : 0.0f;
        float x[8], lowest = INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = ldexpf(p[e], up);
          lowest = fminf(lowest, x[e]);
        }
        more = false;
        if (__builtin_amdgcn_ballot_w64(lowest < least) != 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool later = x[e] < least;  // (a NaN is not)
            x[e] = later ? 0.0f : x[e];
            p[e] = later ? p[e] : 0.0f;
            more |= p[e] > 0.0f;
          }
        }
        split8<T>(x, pf);
#pragma unroll
        for (int d = 0; d < kT; ++d) {
          const short8x vf = values(d);
          const float4x sum = H::mma(vf, pf[1], H::mma(vf, pf[0], float4x{0.0f, 0.0f, 0.0f, 0.0f}));
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][e] = fmaf(sum[e], over, o[d][e]);
        }
      } while (__builtin_amdgcn_ballot_w64(more) != 0);
    }
  }
  finish<D, kSlots>(
      a, t, nparts == 1, o, m, sum_across_groups(l), j, g == 0, [](int) { return true; },
      [&](int wave) { return reinterpret_cast<float*>(&chunks[wave]); }, states);
}

template <typename T>
void launch_type(const SpanArgs& a, int D, hipStream_t stream) {
  const dim3 grid((unsigned)workgroups(a, kSlots)), block(64 * kWaves);
  if (D == 32) hipLaunchKernelGGL((window_decode_kernel<T, 32>), grid, block, 0, stream, a);
  else if (D == 64) hipLaunchKernelGGL((window_decode_kernel<T, 64>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((window_decode_kernel<T, 128>), grid, block, 0, stream, a);
}

}  // namespace

bool window_decode_serves(int kv_dtype, int D) {
  return (kv_dtype == HS_DTYPE_F16 || kv_dtype == HS_DTYPE_BF16) && D <= 128;
}

void window_decode_plan(int B, int H, int Hkv, int D, int64_t most, bool windowed, int cus, int* part,
                        int* heads, int* room, int* longest) {
  plan(B, H, Hkv, kSlots, kChunk, most, windowed, cus, part, heads);
  *longest = kLongest * kChunk * kWaves / *heads;
  *room = parts_on_chip(B, H, Hkv, kSlots, *heads, cus * (D == 128 ? 2 : D == 64 ? 3 : 5));
}

int launch_window_decode(const SpanArgs& a, int kv_dtype, int D, hipStream_t stream) {
  if (!grid_fits(workgroups(a, kSlots), 64 * kWaves))
    return fail(HS_EUNSUPPORTED, "grid too large: sequences * parts * KV heads");
  if (kv_dtype == HS_DTYPE_F16) launch_type<_Float16>(a, D, stream);
  else launch_type<Bf16>(a, D, stream);
  return HS_OK;
}

}  // namespace hs
