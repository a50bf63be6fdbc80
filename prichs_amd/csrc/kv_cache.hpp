// kv_cache.hpp -- layout and number format of the paged 4-bit KV cache.
//
// A page holds kKvPage positions of every kv head; one head's part of a page:
//   K codes  [64 positions][64 bytes]             value 2c and 2c + 1 of a byte
//   V codes  [16 quads][16][4 positions][4 bytes] dword c of a position's 64
//            bytes (values 8c .. 8c + 7) next to dword c of its neighbours
//   K scales [64 positions][4 bytes], V scales [64 positions][4 bytes]
// A value is an e2m1 code (0 .5 1 1.5 2 3 4 6 and a sign bit) times the scale
// of its group of 32 along the head, 2^(byte - 127); byte 255 makes the whole
// group NaN.  Products of the two are exact in bf16.
#pragma once

#include "common.hpp"

namespace prichs {

constexpr int kKvHd = PRICHS_KV_HEAD_DIM;
constexpr int kKvPage = PRICHS_KV_PAGE;
constexpr int kKvK = 0;                           // byte offsets within a head's part
constexpr int kKvV = kKvPage * kKvHd / 2;
constexpr int kKvKScale = 2 * kKvV;
constexpr int kKvVScale = kKvKScale + 4 * kKvPage;
constexpr int kKvPart = kKvVScale + 4 * kKvPage;  // bytes of a (page, kv head)
static_assert(kKvPart == PRICHS_KV_PAGE_BYTES, "header and layout agree");

// Byte offset of dword c of position t in the V codes.
__device__ __forceinline__ int kv_v_off(int t, int c) {
  return kKvV + (t >> 2) * 256 + c * 16 + (t & 3) * 4;
}

// The scale byte of a group whose largest magnitude has the f32 bits `amax`:
// the least s in 1 .. 252 with amax <= 7 * 2^(s - 127), so that rounding 6 <
// x <= 7 down to the largest level is off by no more than rounding 5 is; 255
// for an infinity or NaN.  Adding 0x1fffff carries into the exponent exactly
// where the mantissa passes 1.75.  Past 252 the levels 4 and 6 would be
// infinite: magnitudes above 6 * 2^125 become that.
__device__ __forceinline__ uint32_t kv_scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255;
  const int s = (int)((amax + 0x1fffffu) >> 23) - 2;
  return (uint32_t)min(max(s, 1), 252);
}
// The scale as an f32 (NaN for byte 255).
__device__ __forceinline__ float kv_scale(uint32_t byte) {
  return byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

}  // namespace prichs
