// kv_cache.hpp -- layout and number format of the paged 4-bit KV cache.
//
// A page holds kKvPage positions of every kv head; one head's part of a page:
//   K codes   [64 positions][64 bytes]             values 2c and 2c + 1 of a byte
//   V codes   [16 quads][16][4 positions][4 bytes] dword c of a position's 64
//             bytes (values 8c .. 8c + 7) next to dword c of its neighbours
//   K scales  [4 groups][16][4]     position t at t % 16, t / 16
//   V scales  [4 groups][4][4][4]   position t at (t / 4) % 4, t / 16, t % 4
// The orders are those in which the attention's lanes hold them (kv_attention.hip):
// a lane takes 16 bytes of K of one position, dword c of 4 positions of V, and its
// scales of a whole page in one load each.
// A value is an e2m1 code (0 .5 1 1.5 2 3 4 6 and a sign bit) times the scale
// of its group of 32 along the head, 2^(byte - 127); byte 255 makes the whole
// group NaN.  Products of the two are exact in bf16, and the conversion of two
// codes with their scale is one instruction (which gives NaN for byte 255).
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

// Byte offsets of position t's scale of group r.
__device__ __forceinline__ int kv_k_scale_off(int t, int r) {
  return kKvKScale + r * kKvPage + (t & 15) * 4 + (t >> 4);
}
__device__ __forceinline__ int kv_v_scale_off(int t, int r) {
  return kKvVScale + r * kKvPage + ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3);
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
// The scale as an f32 (byte 255: an infinity, which the conversions make NaN).
__device__ __forceinline__ float kv_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Page of position pos of sequence b, or -1 where the table has none.
__device__ __forceinline__ int kv_page_of(const int32_t *table, int max_pages, int n_pages, int b,
                                          long long pos) {
  if (pos < 0 || pos >= (long long)max_pages * kKvPage) return -1;
  const int p = table[(long long)b * max_pages + (int)(pos / kKvPage)];
  return p >= 0 && p < n_pages ? p : -1;
}

}  // namespace prichs
