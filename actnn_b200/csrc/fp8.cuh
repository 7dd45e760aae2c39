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

namespace actnn {

constexpr int kFpBlock = 128;

static inline int64_t fp8_row_bytes(int64_t K) { return (K + 15) / 16 * 16; }
static inline int64_t fp8_scale_bytes(int64_t rows, int64_t K) { return (K + 511) / 512 * ((rows + 127) / 128) * 512; }

#ifdef __CUDACC__
// Where the byte of (row, block) lies; `tiles`: ceil(rows / 128).
ACTNN_DEV size_t fp8_scale_at(int64_t row, int64_t block, int64_t tiles) {
  return ((size_t)(block >> 2) * tiles + (row >> 7)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (block & 3);
}
// The byte of a block whose largest magnitude has these bits (finite).  448 is 1.75 * 2^8.
ACTNN_DEV uint32_t fp8_scale_byte(uint32_t bits) {
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return (uint32_t)max(e, 1);
}
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
ACTNN_DEV float finite_or_nan(float v) { return not_finite(__float_as_uint(v)) ? __uint_as_float(0x7fffffffu) : v; }

// The largest magnitude of the finite elements, as bits; `bad`: whether there are others.
template <typename T> ACTNN_DEV uint32_t fp8_most(const Vec<T, 8>& v, bool& bad) {
  uint32_t most = most_of(v);
  bad = not_finite(most);
  if (bad) {
    most = 0;
    float2 f[4];
    unpack_vec(v, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = abs_bits(f[i].x), y = abs_bits(f[i].y);
      most = max(most, max(not_finite(x) ? 0u : x, not_finite(y) ? 0u : y));
    }
  }
  return most;
}
// The codes of eight elements.
template <typename T> ACTNN_DEV uint2 fp8_codes8(const Vec<T, 8>& v, float factor, bool bad) {
  float2 f[4];
  unpack_vec(v, f);
  if (bad) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(finite_or_nan(f[i].x), finite_or_nan(f[i].y));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f_mul(f[i], make_float2(factor, factor));
  return make_uint2(fp8_pair(f[0].x, f[0].y) | fp8_pair(f[1].x, f[1].y) << 16, fp8_pair(f[2].x, f[2].y) | fp8_pair(f[3].x, f[3].y) << 16);
}
// The largest over the half of the warp that the lane is in.
ACTNN_DEV uint32_t half_warp_max(uint32_t v) { return __reduce_max_sync((threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu, v); }
// Eight elements from e on, zeros from `end` on.  VEC: whole aligned vectors.
template <typename T, bool VEC> ACTNN_DEV Vec<T, 8> fp8_load(const T* p, int64_t e, int64_t end) {
  if (VEC && e < end) return load_vec<T, 8>(p + e);
  Vec<T, 8> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(v.w)[i] = !VEC && e + i < end ? __ldg(p + e + i) : from_float<T>(0.f);
  return v;
}
#endif

}  // namespace actnn
