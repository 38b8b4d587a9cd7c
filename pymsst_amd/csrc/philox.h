// Counter-based random bits of the dropout: Philox4x32 with 7 rounds (Salmon, Moraes, Dror & Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011; 7 rounds are the fewest that pass its
// statistical tests, 10 would cost 1.4 times the multiplies and make the 16-bit dropout bound by them).
//
// Element e of a call takes 16 bits of the block with counter (e / 8 as two words, offset as two words)
// and key = seed as two words: word (e % 8) / 2, its low half for even e.  It is kept where these are at
// least `limit` = round(65536 p), so a probability is held to 2^-16 and what is kept is divided by exactly
// the share of values that keep.  The mask depends on (seed, offset, e) alone: the backward, another
// launch shape or the attention's tiles draw the same bits again, and nothing is stored.
#pragma once

#include "common.h"

namespace pmsst {

struct Dropout {
  uint32_t limit;      // kept where the element's 16 bits >= limit; 0: nothing is drawn
  float factor;        // 65536 / (65536 - limit)
  const int64_t* rng;  // device {seed, offset}
};

// (seed, offset) of a launch, read from device memory so that a captured graph may be replayed with others.
struct PhiloxKey {
  uint32_t k0, k1, c2, c3;
};

__device__ __forceinline__ PhiloxKey philox_key(const int64_t* __restrict__ rng) {
  const uint64_t seed = static_cast<uint64_t>(rng[0]), offset = static_cast<uint64_t>(rng[1]);
  return {static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), static_cast<uint32_t>(offset),
          static_cast<uint32_t>(offset >> 32)};
}

__device__ __forceinline__ void philox7(const PhiloxKey& key, uint64_t block, uint32_t (&w)[4]) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = key.c2, c3 = key.c3;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = __builtin_amdgcn_bitop3_b32(static_cast<uint32_t>(p1 >> 32), c1, k0, 0x96);  // a ^ b ^ c
    c1 = static_cast<uint32_t>(p1);
    c2 = __builtin_amdgcn_bitop3_b32(static_cast<uint32_t>(p0 >> 32), c3, k1, 0x96);
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// Whether element `e` (0..7) of the block is kept.
__device__ __forceinline__ bool philox_keep(const uint32_t (&w)[4], int e, uint32_t limit) {
  return static_cast<uint16_t>((e & 1) ? w[e >> 1] >> 16 : w[e >> 1]) >= static_cast<uint16_t>(limit);
}

// The same of both elements of a word: all ones in the half of one that is dropped.  A saturating difference of
// the halves, taken as signed numbers (both less 2^15), has the sign of the comparison.
__device__ __forceinline__ uint32_t philox_dropped(uint32_t w, uint32_t limit) {
  typedef short v2 __attribute__((ext_vector_type(2)));
  const v2 r = __builtin_bit_cast(v2, w ^ 0x80008000u), l = __builtin_bit_cast(v2, (limit ^ 0x8000u) * 0x10001u);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(r, l) >> static_cast<short>(15));
}

// The kept elements of a block as a byte, element e in bit e.
__device__ __forceinline__ uint32_t philox_kept8(const uint32_t (&w)[4], uint32_t limit) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bits |= ~philox_dropped(w[i], limit) & ((1u << (2 * i)) | (1u << (17 + 2 * i)));
  return (bits | bits >> 16) & 0xFFu;
}

// Host: limit and factor of a probability in [0, 1).
inline Dropout make_dropout(double p, const int64_t* rng) {
  double limit = p * 65536.0 + 0.5;
  uint32_t l = limit >= 65535.0 ? 65535u : static_cast<uint32_t>(limit);
  return {l, static_cast<float>(65536.0 / (65536.0 - l)), rng};
}

}  // namespace pmsst
