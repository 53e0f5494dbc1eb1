// The 4-bit cache's records, as the kernels that write, read and attend to them see
// them.
//
// A cache is [NB, BS, Hkv, R] bytes, R = D / 2 + D / 8: one record for each token and KV
// head.  Every 32 elements of a head (a group) share a step s >= 0 and a lowest value
// lo, both fp16; an element is held as a whole number n of 0 .. 15 and stands for
// n s + lo.  A record is D / 8 words of 8 elements (element e in bits 4 e .. 4 e + 3),
// then the D / 32 steps, then the D / 32 lowest values.
//
// The words' order is the one that the attention reads.  Word w of a value's record holds
// elements 8 w ..; it is transposed on its way out of LDS, whatever its order.  Word w of
// a key's holds elements 32 (w % (D / 32)) + 8 (w / (D / 32)) ..: a lane of the first
// product wants 8 elements of each group, at 8 times its quarter of the wave, and these
// lie side by side so that they come in one load.
//
// Records are token-major like the rows of the other caches, so pages of them can be
// copied, forked, packed and moved as bytes.  Records and their steps begin at multiples of
// D / 8 bytes, lowest values half as much further on.
#pragma once

#include "hs_common.h"

namespace hs {

constexpr int kQ4Group = 32;
constexpr float kF16Most = 65504.0f;

constexpr int q4_record_bytes(int D) { return D / 2 + D / 8; }

// The place of the word that holds elements 8 i .. of a head, of G = D / 32 groups.
template <bool kKeys>
__device__ inline int q4_word(int i, int G) {
  return kKeys ? (i & 3) * G + (i >> 2) : i;
}

}  // namespace hs
