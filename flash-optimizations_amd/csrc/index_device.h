// Index records ("index"): geometry and the coding that the store and the scores share.
//
// A record is one key of 128 coordinates as E4M3 codes with one float32 scale, value =
// code * scale. A page holds 64 records: their code rows of 128 bytes, then their 64
// scales, 8,448 bytes, so that a wave reads 16 records' codes as 2 KiB in a row and a
// page's scales as 256 bytes. The store writes powers of two as scales, the smallest that
// holds the row (E4M3 is a floating format: a finer scale would gain nothing but the
// last binade, and the division would no longer be exact), NaN for a row with an infinity
// or NaN, which reads as 128 NaN.
#pragma once
#include "remnant_device.h"

namespace rm {

constexpr int kIndexDim = 128;
constexpr int kIndexRope = 64;  // the last 64 coordinates are rotated
constexpr int kIndexScalesAt = kPageRecords * kIndexDim;                // 8,192
constexpr int kIndexPageBytes = kIndexScalesAt + 4 * kPageRecords;      // 8,448

// The maximum of NaN-free magnitudes as BF16 bits of two values a dword.
__device__ __forceinline__ uint32_t top_of_pairs(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(
      uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a & 0x7fff7fffu),
                                          __builtin_bit_cast(u16x2, b & 0x7fff7fffu)));
}

// Four codes of a row whose scale is 2^e, from two pairs of BF16.
__device__ __forceinline__ uint32_t index_codes(uint32_t n0, uint32_t n1, float scale) {
  s16x2 c = {0, 0};
  c = fp8_pair<false>(c, __builtin_bit_cast(bf16x2, n0), scale);
  c = fp8_pair<true>(c, __builtin_bit_cast(bf16x2, n1), scale);
  return __builtin_bit_cast(uint32_t, c);
}

}  // namespace rm
