// A cache of keys and values in 8 bits: how a row is held and where its codes lie.
//
// A row x of a token's key (or value) is e4m3 codes times a power of two of its own, 2^e, the smallest with which the row's
// largest magnitude stays within 448, the format's largest number: e = ceil(log2(max |x| / 448)), at least -126.  The scale
// byte is e + 127 (the exponent field of the float 2^e).  e4m3 rounds relative to a number's own size, so a power of two
// loses nothing against a finer scale, and scaling and its undoing are exact.  A row that holds something that is no finite
// number is held as NaN throughout.
//
// Pages: codes [pages][kv heads][2][page_size * dh] bytes, scales [pages][kv heads][2][page_size].  Sixteen keys' codes lie
// together, in pieces of 64 elements (a kilobyte; a last piece of 32 elements where dh % 64 == 32), each piece in the order
// in which a wavefront's lanes (row r = lane % 16, group g = lane / 16) take it: lane after lane u codes, u = 16 (8 in a last
// piece of 32), so that every load is one contiguous piece of memory:
//   keys:   lane (r, g): key r, elements u g .. u g + u - 1 of the piece
//   values: lane (r, g): for each 16 elements of the piece, element r of them, keys 4 g .. 4 g + 3
#pragma once
#include "common.h"

namespace jle {

constexpr uint32_t kCodesNaN = 0x7f7f7f7fu;  // four codes that are no number
// of four codes, those that are no number: all bits of their bytes
__device__ __forceinline__ uint32_t codes_none(uint32_t w) { return ((((w & kCodesNaN) + 0x01010101u) & 0x80808080u) >> 7) * 255u; }

__host__ __device__ __forceinline__ int lane_codes(int d, int dh) { return dh - (d & ~63) >= 64 ? 16 : 8; }

// where element d of key j (of sixteen) lies among their 16 * dh codes
__device__ __forceinline__ int key_place(int d, int j, int dh) {
  const int u = lane_codes(d, dh), e = d & 63;
  return (d & ~63) * 16 + e / u * 16 * u + j * u + e % u;
}
__device__ __forceinline__ int value_place(int d, int j, int dh) {
  const int u = lane_codes(d, dh), e = d & 63;
  return (d & ~63) * 16 + (j >> 2) * 16 * u + (d & 15) * u + (e >> 4) * 4 + (j & 3);
}

// the scale byte of a row from the bits of its largest magnitude (255: not finite).  448 = 1.75 * 2^8: the carry into the
// exponent is a fraction beyond 1.75
__device__ __forceinline__ int scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  return max((int)((top + 0x1fffffu) >> 23) - 8, 1);
}
// the factor that turns numbers into codes' units: 2^-e
__device__ __forceinline__ float code_factor(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// four numbers within +-448 as four codes, rounded to nearest even
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// x / d for 0 <= x < 2^31 by a product: with floor(2^32 / d) (2^32 - 1 for one) the estimate is the quotient or one less.
// (A division of two numbers that are only known when the kernel runs is tens of instructions, and a short launch waits for
// every instruction that it meets for the first time.)
struct Divisor {
  uint32_t d, magic;
};
inline Divisor divisor(int d) { return {(uint32_t)d, d == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / (uint32_t)d)}; }
__device__ __forceinline__ int over(int x, Divisor by) {
  const uint32_t q = __umulhi((uint32_t)x, by.magic);
  return (int)(q + ((uint32_t)x - q * by.d >= by.d));
}

__host__ inline bool quantized_head_ok(int dh) { return dh == 32 || dh == 64 || dh == 96 || dh == 128 || dh == 256; }

}  // namespace jle
