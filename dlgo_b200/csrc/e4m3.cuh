// The 8-bit cache's rows: a key or a value of one head and position as e4m3 numbers with one power of two,
//
//   e = the smallest whole number with max |x| <= 448 * 2^e, kept within [-119, 119];  byte = e + 127
//   stored = x / 2^e, clamped to +-448, to the nearest e4m3 number (ties to even);     value = stored * 2^e
//
// A power of two costs nothing in a floating format (the row's largest number lies in the top octave either way), is found
// from the exponent of the maximum alone, and makes every value a product that float16, bfloat16 and fp32 hold exactly
// (within their exponents' range).  Infinities are stored as the largest number of their sign, a NaN as NaN; neither
// changes the row's scale beyond the limit above.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>
#include <string.h>

#include <utility>

namespace dlgo {

constexpr int E8_PAGE = 64;          // positions of a page

// scale byte of a row whose largest |x| is `most` (no NaN)
__device__ __forceinline__ int e4m3_scale_byte(float most) {
  const unsigned u = __float_as_uint(most);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);     // 448 = 1.75 * 2^8
  return min(max(e, 8), 246);
}
__device__ __forceinline__ float e4m3_scale(int byte) { return __uint_as_float((unsigned)byte << 23); }            // 2^e
__device__ __forceinline__ float e4m3_inverse(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }  // 2^-e

// two numbers to e4m3, the first in the low byte
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t e4m3_quad(float a, float b, float c, float d) {
  return e4m3_pair(a, b) | (e4m3_pair(c, d) << 16);
}
// the low or the high two e4m3 numbers of a word as float16 (exact)
__device__ __forceinline__ uint32_t e4m3_low_half2(uint32_t w) {
  uint32_t h;
  asm("{.reg .b16 l, u; mov.b32 {l, u}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ uint32_t e4m3_high_half2(uint32_t w) {
  uint32_t h;
  asm("{.reg .b16 l, u; mov.b32 {l, u}, %1; cvt.rn.f16x2.e4m3x2 %0, u;}" : "=r"(h) : "r"(w));
  return h;
}

// An entry point called with its arguments as one record of 8-byte fields, in their order: pointers and whole numbers as such,
// a float as a double.  (From Python one record takes 2 us less than two dozen arguments.)
template <typename T> struct RecordField {                   // a pointer
  static bool get(const long long* r, T& x) { x = (T)(uintptr_t)*r; return true; }
};
template <> struct RecordField<int> {
  static bool get(const long long* r, int& x) { x = (int)*r; return x == *r; }
};
template <> struct RecordField<float> {
  static bool get(const long long* r, float& x) {
    double d;
    memcpy(&d, r, 8);
    x = (float)d;
    return true;
  }
};
template <size_t I, typename T> struct RecordAt { T x; };
template <typename... A, size_t... I>
int call_record(int (*fn)(A...), const long long* r, std::index_sequence<I...>) {
  struct All : RecordAt<I, A>... {} all;
  const bool fit = (RecordField<A>::get(r + I, static_cast<RecordAt<I, A>&>(all).x) & ...);
  return fit ? fn(static_cast<RecordAt<I, A>&>(all).x...) : DLGO_ERR_SIZE;
}
template <typename... A> int call_record(int (*fn)(A...), const long long* r) {
  return call_record(fn, r, std::index_sequence_for<A...>());
}

}  // namespace dlgo
