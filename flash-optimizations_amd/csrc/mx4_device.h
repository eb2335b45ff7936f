// 4-bit latent records ("mx4"): geometry and the device helpers that the store,
// the reader and the decode share.
//
// A record is 512 coordinates as E2M1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their
// negatives; coordinate 2i in the low half of byte i) with one UE8M0 scale byte
// for 32 coordinates: value = code * 2^(byte - 127). 256 + 16 bytes, 16-byte
// aligned, 64 to a page. The 64-coordinate RoPE tail is stored rotated, so a
// reader needs no position. A scale byte the store writes is 112..159, or 255 for
// a group with an infinity or NaN in it, which reads as 32 NaN.
#pragma once
#include "remnant_device.h"

namespace rm {

constexpr int kMx4Group = 32;
constexpr int kMx4CodeBytes = kHeadDim / 2;                        // 256
constexpr int kMx4ScaleBytes = kHeadDim / kMx4Group;               // 16
constexpr int kMx4RecordBytes = kMx4CodeBytes + kMx4ScaleBytes;    // 272
constexpr int kMx4MaxExponent = 32;  // largest scale the store writes: 2^32
constexpr int kMx4NanScale = 255;

// Scale exponent of a group whose largest magnitude is amax: the smallest e with
// max(amax, 1e-4) <= 6 * 2^e, at most 32 (values beyond 6 * 2^32 saturate).
// 6 * 2^e = 1.5 * 2^(e + 2).
__device__ __forceinline__ int mx4_exponent(float amax) {
  if (!(amax >= 1e-4f)) return -15;
  const uint32_t b = f2u(amax);
  const int e = (int)((b >> 23) & 0xffu) - 127 - 2 + ((b & 0x7fffffu) > 0x400000u ? 1 : 0);
  return e < kMx4MaxExponent ? e : kMx4MaxExponent;
}

// Two BF16 divided by a power-of-two scale -> E2M1, round to nearest even, ties to
// the even code, magnitudes above 6 to 6; into byte kByte of `acc`
// (v_cvt_scalef32_pk_fp4_bf16; the self-test library compares every finite BF16
// with the software rounding).
template <int kByte>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t acc, bf16x2 n, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(acc, n, scale, kByte);
}

// The two codes of byte kByte times a power-of-two scale -> two BF16 (exact;
// v_cvt_scalef32_pk_bf16_fp4, NaN for scale byte 255, whose float is infinite).
template <int kByte>
__device__ __forceinline__ uint32_t fp4_pair_to_bf16(uint32_t codes, float scale) {
  const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kByte);
  return __builtin_bit_cast(uint32_t, r);
}
// Eight codes (one dword) -> eight BF16.
__device__ __forceinline__ u32x4 fp4x8_to_bf16(uint32_t codes, float scale) {
  return u32x4{fp4_pair_to_bf16<0>(codes, scale), fp4_pair_to_bf16<1>(codes, scale),
               fp4_pair_to_bf16<2>(codes, scale), fp4_pair_to_bf16<3>(codes, scale)};
}

// The scale a byte stands for, as a float (byte 255: infinity, see above).
__device__ __forceinline__ float mx4_scale(uint32_t byte) { return u2f(byte << 23); }

}  // namespace rm
