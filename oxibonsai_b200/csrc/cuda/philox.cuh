// Random bits from a counter: Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011).
//
// Dropout over rows of d values takes its bits from the counter (column / 8, 0, row, row >> 32) under the seed as key: 128 bits for eight
// neighbouring values, 16 for each (value j of the eight has bits 16 (j % 2) of word j / 2).  A value stays where its 16 bits are below
// `steps` of 65536, so that the probability has steps of 2^-16, and what stays is multiplied by 65536 / steps: the mean is kept exactly.  32
// bits for a value would take twice the instructions, which are what bounds the kernels that make masks (see dropout.cu).
#pragma once
#include <stdint.h>

namespace bonsai {

struct DropoutRule {
  unsigned long long seed;
  const long long* seed_dev;     // given: read in place of `seed` when the kernel runs
  unsigned limit;                // steps of 65536, below 65536, in the upper half
  float share;                   // 65536 / steps, 0 where nothing stays
};

inline DropoutRule dropout_rule(unsigned long long seed, const long long* seed_dev, int steps) {
  return {seed, seed_dev, steps < 65536 ? (unsigned)steps << 16 : 0u, steps > 0 ? 65536.0f / (float)steps : 0.0f};
}

__device__ __forceinline__ uint2 philox_key(const DropoutRule& rule) {
  const unsigned long long s = rule.seed_dev != nullptr ? (unsigned long long)*rule.seed_dev : rule.seed;
  return make_uint2((unsigned)s, (unsigned)(s >> 32));
}

__device__ __forceinline__ uint4 philox(uint4 c, uint2 k) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const unsigned long long x = (unsigned long long)0xD2511F53u * c.x, y = (unsigned long long)0xCD9E8D57u * c.z;
    c = make_uint4((unsigned)(y >> 32) ^ c.y ^ k.x, (unsigned)y, (unsigned)(x >> 32) ^ c.w ^ k.y, (unsigned)x);
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

// The random words of values 8 * group .. 8 * group + 7 of a row, and whether value j of them stays.
__device__ __forceinline__ uint4 dropout_words(unsigned group, unsigned long long row, uint2 key) {
  return philox(make_uint4(group, 0u, (unsigned)row, (unsigned)(row >> 32)), key);
}
__device__ __forceinline__ bool dropout_keeps(const uint4& words, int j, unsigned limit) {
  const unsigned w = j < 2 ? words.x : j < 4 ? words.y : j < 6 ? words.z : words.w;
  return (j & 1 ? w : w << 16) < limit;
}
// Two 16-bit values in a word, those that do not stay set to 0; `random`: their 32 bits.
__device__ __forceinline__ unsigned dropout_pair(unsigned two, unsigned random, unsigned limit) {
  two = random << 16 < limit ? two : two & 0xffff0000u;
  return random < limit ? two : two & 0xffffu;
}

}  // namespace bonsai
