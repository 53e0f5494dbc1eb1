// Decode over spans: the keys that a sequence's new token sees when it sees the first
// few of its context (sinks) and a window of the last ones, or all of them.
//
// The kernels number the visible keys 0 .. n - 1 and look every key's slot up in the block
// table by itself, so neither a window's start nor a sink's end has to lie at a page's
// border, and no key that is not seen is ever read.  Ranges of these numbers are the
// parts that waves take; parts of one row are merged by span_merge_kernel.
#pragma once

#include "hs_common.h"

#include <algorithm>

namespace hs {

constexpr int kSpanDealt = 256;   // rows at most whose parts are fitted and dealt by their number

namespace span {
constexpr int kWaves = 4;         // of a workgroup
constexpr float kSlack = 8.0f;    // lazy raise of the running max, log2 units
// Where running maxima start: no finite score lies below, so a row of one is never empty.
constexpr float kLowest = -0x1.fffffep127f;
}  // namespace span

struct SpanArgs {
  const float* q;             // [B, H, D]
  const uint8_t *k, *v;       // [NB, BS, Hkv, row of one head]
  const int32_t* bt;          // [B, MB]
  const int32_t* ctx;         // [B]
  float* out;                 // [B, H, D]
  // States of parts: [B, H, P] of them, or [states, H] where parts are fitted, by their number.
  float* part_acc;            // [.., D]        un-normalised outputs
  float* part_ml;             // [.., 2]        (max, sum), base-2 domain
  int B, H, Hkv, BS, MB, NB;
  int bs_shift;               // log2(BS), or -1
  int window, sinks;          // window 0: all keys
  int part, P;                // keys of a part at least, parts of the longest row at most
  int room;                   // parts in all that their length is fitted to, or 0
  int tasks;                  // parts and empty rows at most, over all rows
  int64_t states;             // parts at most then
  int32_t* fitted;            // their keys
  int32_t* numbers;           // [B, 2]         of a row's first part, which the next ones follow, and of its last
  int heads;                  // matrix cores: KV heads of a workgroup
  float qscale;               // scale * log2(e)
};

// The visible keys of one sequence.
struct Span {
  int n, sinks, skip;   // position of key i: i below sinks, i + skip from there on

  __device__ Span(const SpanArgs& a, int b) {
    const int64_t cap = (int64_t)a.MB * a.BS;
    const int len = (int)max((int64_t)0, min((int64_t)a.ctx[b], cap));
    const int first = a.window && len > a.window ? len - a.window : 0;   // of the window
    sinks = min(a.sinks, first);
    n = sinks + len - first;
    skip = first - sinks;
  }
  __device__ int parts(int part) const {
    return (int)(((uint32_t)n + (uint32_t)part - 1) / (uint32_t)part);
  }
  // Keys [lo, hi) of part p, nparts parts in all; p is counted so that every row's last part is
  // P - 1, and becomes its number in the row.  Work that begins with the lowest p begins with
  // whole parts and ends with the rows' last ones, which are shorter.
  __device__ bool part(const SpanArgs& a, int part, int& p, int& lo, int& hi, int& nparts) const {
    nparts = parts(part);
    p -= a.P - nparts;
    if (p < 0) return false;
    lo = p * part;
    hi = n - lo < part ? n : lo + part;
    return true;
  }
  // Where key i < n lies: its page's table entry and its place in the page.
  struct Place {
    int32_t block;
    uint32_t off;
  };
  __device__ Place place(const SpanArgs& a, const int32_t* bt, int i) const {
    const uint32_t pos = (uint32_t)(i < sinks ? i : i + skip);
    if (a.bs_shift >= 0)   // uniform
      return {bt[pos >> a.bs_shift], pos & (uint32_t)(a.BS - 1)};
    const uint32_t page = pos / (uint32_t)a.BS;
    return {bt[page], pos - page * (uint32_t)a.BS};
  }
  // As a row of the cache seen as [NB * BS] rows (below 2^31).
  __device__ static uint32_t slot(const SpanArgs& a, const Place& x) {
    return (uint32_t)safe_block(x.block, a.NB) * (uint32_t)a.BS + x.off;
  }
};

// Keys that the longest row of these sizes can see.
inline int64_t span_most(int64_t MB, int64_t BS, int window, int sinks) {
  const int64_t cap = sat_mul(MB, BS);
  return window ? std::min(cap, (int64_t)window + sinks) : cap;
}

// Where in the workspace the (max, sum) pairs and, where parts are fitted, their keys and numbers
// begin, and its bytes (INT64_MAX when too large; 0 when no row has parts).
struct SpanLayout {
  int64_t ml, fitted, numbers, end;

  SpanLayout(const SpanArgs& a, int D) : ml(0), fitted(0), numbers(0), end(0) {
    if (a.P <= 1) return;
    const int64_t states = sat_mul(a.room ? a.states : sat_mul(a.B, a.P), a.H);
    ml = sat_mul(states, D * 4);
    fitted = sat_add(ml, sat_mul(states, 8));
    numbers = sat_add(fitted, 16);
    end = a.room ? sat_add(numbers, (int64_t)a.B * 8) : fitted;
  }
};

void launch_span_merge(const SpanArgs& a, int D, hipStream_t stream);

}  // namespace hs
