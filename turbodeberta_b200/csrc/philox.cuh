// Counter-based random bits for dropout: Philox4x32-10 as published by Salmon, Moraes, Dror and Shaw ("Parallel random numbers:
// as easy as 1, 2, 3", 2011).  A block of 128 bits is a function of a counter and a key, so a mask is made where it is needed,
// forward and backward, and never stored.
//
// An element takes 16 of the bits: eight elements share a block, and a drop probability is a multiple of 2^-16 (the scale of what
// stays is that of the rounded probability, so the expectation is exact).  With 32 bits an element the generator alone would take some
// 15 instruction slots an element, of the 22 that an SM has while 4 bytes of it pass through memory; with 16 it is half of that.
#pragma once
#include "tdb_internal.h"

namespace tdb {

__device__ __forceinline__ uint64_t dropout_seed(const Dropout& k) { return (uint64_t)(k.seed ? *k.seed : k.seed_value); }

__device__ __forceinline__ uint4 philox(uint64_t group, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0; c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1; c3 = (uint32_t)a;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The 16-bit numbers of eight consecutive elements, two to a word.  ALIGNED: `first` is a multiple of eight; otherwise they lie in
// two blocks.
template <bool ALIGNED>
__device__ __forceinline__ uint4 dropout_bits(uint64_t first, uint64_t offset, uint64_t seed) {
  const uint4 a = philox(first >> 3, offset, seed);
  if (ALIGNED || (first & 7) == 0) return a;
  const uint4 b = philox((first >> 3) + 1, offset, seed);
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = first & 4 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = first & 2 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = first & 1 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// What stays of eight elements, scaled.  A dropped element is zero whatever it held (NaN and infinities too).
// drop > 0; above = (drop << 16) - 1: a number is at least `drop` when, in a word's upper half, the word is greater than that.
__device__ __forceinline__ uint32_t dropout_above(uint32_t drop) { return (drop << 16) - 1; }
__device__ __forceinline__ void drop8(float* f, const uint4& bits, uint32_t above, float scale) {
  const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = w[i] << 16 > above ? f[2 * i] * scale : 0.f;
    f[2 * i + 1] = w[i] > above ? f[2 * i + 1] * scale : 0.f;
  }
}

}  // namespace tdb
