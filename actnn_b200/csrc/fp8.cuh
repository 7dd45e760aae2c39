// 8-bit floating-point codes (e4m3) with power-of-two scales: what the product and its codes share.
//
// Of a block, e is the least integer, at least -126, with max |x| <= 448 * 2^e; a code is x * 2^-e rounded to e4m3, half to even, and
// stands for code * 2^e.  The scale is a power of two, so the only rounding is that of the code.  It is kept as the byte e + 127.
// Numbers that are not finite take no part in the maximum; their code is e4m3's NaN.
//
// Scales of rows lie in the order the tensor cores read them: [ceil(blocks / 4)][ceil(rows / 128)][512], of 128 rows and four
// blocks the byte of row r and block j at (r % 32) * 16 + (r / 32) * 4 + j.
#pragma once

#include "activation.cuh"
#include "load_one.cuh"

namespace actnn {

constexpr int kFpBlock = 128;

static inline int64_t fp8_row_bytes(int64_t K) { return (K + 15) / 16 * 16; }
static inline int64_t fp8_scale_bytes(int64_t rows, int64_t K) { return (K + 511) / 512 * ((rows + 127) / 128) * 512; }

#ifdef __CUDACC__
// Where the byte of (row, block) lies; `tiles`: ceil(rows / 128).
ACTNN_DEV size_t fp8_scale_at(int64_t row, int64_t block, int64_t tiles) {
  return ((size_t)(block >> 2) * tiles + (row >> 7)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (block & 3);
}
// The byte of a block whose largest magnitude has these bits (finite).  448 is 1.75 * 2^8: what is above it in its mantissa, 0x600001 on,
// carries into the exponent.
ACTNN_DEV uint32_t fp8_scale_byte(uint32_t bits) { return (uint32_t)max((int)((bits + 0x1fffffu) >> 23) - 8, 1); }
// 2^e and 2^-e of a byte e + 127, from 1 to 253.
ACTNN_DEV float fp8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
ACTNN_DEV float fp8_factor(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// Codes of lo and hi in the lower and upper byte.
ACTNN_DEV uint32_t fp8_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
ACTNN_DEV float2 fp8_unpack(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)pair));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
ACTNN_DEV bool not_finite(uint32_t bits) { return (bits & 0x7fffffffu) >= 0x7f800000u; }
// A word of elements (one of float32, two of a 16-bit type): zero, or NaN, in the place of what is not finite.
template <typename T> ACTNN_DEV uint32_t fp8_word(uint32_t w, uint32_t instead) {
  const float2 f = pair_to_float(w, T());
  return (not_finite(__float_as_uint(f.x)) ? instead & 0xffffu : w & 0xffffu) | (not_finite(__float_as_uint(f.y)) ? instead & 0xffff0000u : w & 0xffff0000u);
}
template <> ACTNN_DEV uint32_t fp8_word<float>(uint32_t w, uint32_t instead) { return not_finite(w) ? instead : w; }
template <typename T> ACTNN_DEV uint32_t fp8_word_finite(uint32_t w) { return fp8_word<T>(w, 0u); }
template <typename T> ACTNN_DEV uint32_t fp8_word_nan(uint32_t w) { return fp8_word<T>(w, sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu); }
// Their magnitudes, which compare as unsigned numbers do; whether one of them is not finite; the larger ones.
template <typename T> ACTNN_DEV uint32_t fp8_word_abs(uint32_t w) { return w & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu); }
template <typename T> ACTNN_DEV uint32_t fp8_word_max(uint32_t a, uint32_t b) { return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b); }
template <typename T> ACTNN_DEV bool fp8_word_bad(uint32_t magnitudes) {
  const float2 f = pair_to_float(magnitudes, T());
  return not_finite(__float_as_uint(f.x)) || not_finite(__float_as_uint(f.y));
}
template <> ACTNN_DEV bool fp8_word_bad<float>(uint32_t magnitudes) { return not_finite(magnitudes); }

// The codes of eight elements, which are finite or NaN.
template <typename T> ACTNN_DEV uint2 fp8_codes8(const Vec<T, 8>& v, float factor) {
  float2 f[4];
  unpack_vec(v, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f_mul(f[i], make_float2(factor, factor));
  return make_uint2(fp8_pair(f[0].x, f[0].y) | fp8_pair(f[1].x, f[1].y) << 16, fp8_pair(f[2].x, f[2].y) | fp8_pair(f[3].x, f[3].y) << 16);
}
// The largest magnitudes, as bits of float32, of two vectors over the half of the warp that the lane is in, given the largest of the words
// of each.  16-bit types go through the lanes side by side.
template <typename T> ACTNN_DEV void fp8_half_warp(uint32_t m, uint32_t n, uint32_t (&bits)[2]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t w = __vmaxu2(__byte_perm(m, n, 0x5410), __byte_perm(m, n, 0x7632));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) w = __vmaxu2(w, __shfl_xor_sync(kFull, w, o));
    const float2 f = pair_to_float(w, T());
    bits[0] = __float_as_uint(f.x), bits[1] = __float_as_uint(f.y);
  } else {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(kFull, m, o)), n = max(n, __shfl_xor_sync(kFull, n, o));
    bits[0] = m, bits[1] = n;
  }
}
template <typename T> ACTNN_DEV uint32_t fp8_words_most(const Vec<T, 8>& v) {
  uint32_t m = fp8_word_abs<T>(v.w[0]);
#pragma unroll
  for (int i = 1; i < (int)(sizeof(v.w) / 4); ++i) m = fp8_word_max<T>(m, fp8_word_abs<T>(v.w[i]));
  return m;
}
// The largest magnitudes of two vectors' blocks, which with a vector are half a warp.  What is not finite does not count, and is
// made NaN.
template <typename T> ACTNN_DEV void fp8_block_bits(Vec<T, 8>& a, Vec<T, 8>& b, uint32_t (&bits)[2]) {
  uint32_t m = fp8_words_most(a), n = fp8_words_most(b);
  if (__any_sync(kFull, fp8_word_bad<T>(fp8_word_max<T>(m, n)))) {
    m = n = 0;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(a.w) / 4); ++i) {
      m = fp8_word_max<T>(m, fp8_word_abs<T>(fp8_word_finite<T>(a.w[i])));
      n = fp8_word_max<T>(n, fp8_word_abs<T>(fp8_word_finite<T>(b.w[i])));
      a.w[i] = fp8_word_nan<T>(a.w[i]);
      b.w[i] = fp8_word_nan<T>(b.w[i]);
    }
  }
  fp8_half_warp<T>(m, n, bits);
}
// Eight elements from e on, zeros from `end` on.  VEC: whole aligned vectors.
template <typename T, bool VEC> ACTNN_DEV Vec<T, 8> fp8_load(const T* p, int64_t e, int64_t end) {
  if (VEC && e < end) return load_vec<T, 8>(p + e);
  Vec<T, 8> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(v.w)[i] = !VEC && e + i < end ? load_one(p + e + i) : from_float<T>(0.f);
  return v;
}
#endif

}  // namespace actnn
