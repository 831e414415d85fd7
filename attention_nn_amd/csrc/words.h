// Order-preserving words of numbers and ranges of them (internal; plain C++ on the host too).
//
// A number's word is its bits with the sign turned, all of them turned below zero: the larger
// number has the larger word.  No number here is -0 (it counts as 0, word 0x80000000), but a
// range may end at the word that -0 would have, 0x7fffffff.  As numbers -0 and 0 are
// equal: compared with the number of its upper end, 0 would lie in a range whose words
// all lie below 0's.  Whether a number lies in a range is therefore asked of its word.
#pragma once
#include <stdint.h>

#ifndef ANN_HD
#if defined(__HIPCC__)
#define ANN_HD __host__ __device__ __forceinline__
#else
#define ANN_HD inline
#endif
#endif

namespace ann {

// Of a number (no -0; a NaN's lies outside those of -infinity .. infinity).
ANN_HD uint32_t word_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
ANN_HD float word_value(uint32_t k) {
  return __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// The largest number with a word up to k.
ANN_HD float word_most(uint32_t k) { return word_value(k == 0x7fffffffu ? k - 1 : k); }

// The words lo .. hi (lo above -infinity's), cut into 2^11 equal parts at most.
struct WordRange {
  uint32_t lo, hi;
  ANN_HD int shift() const { return hi - lo >= 2048 ? 21 - __builtin_clz(hi - lo) : 0; }   // log2 of a part
  // Whether x, -0 too, lies inside; its part.
  ANN_HD bool has(float x, int shift, int& part) const {
    const uint32_t at = word_of(x + 0.f) - lo;
    part = (int)(at >> shift);
    return at <= hi - lo;
  }
  ANN_HD WordRange part(int i, int shift) const {
    const uint32_t a = lo + ((uint32_t)i << shift), b = a + ((1u << shift) - 1);
    return {a, b < hi ? b : hi};
  }
};

}  // namespace ann
