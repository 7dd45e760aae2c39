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
// The largest magnitudes, as bits of float32, of two vectors over the half of the warp that the lane is in, which with a vector is a
// block; `bad`: whether the block holds what is not finite, which does not count.  16-bit types go through the lanes side by side.
template <typename T> ACTNN_DEV void fp8_block_bits(const Vec<T, 8>& a, const Vec<T, 8>& b, uint32_t (&bits)[2], bool (&bad)[2]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = a.w[0] & 0x7fff7fffu, n = b.w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __vmaxu2(m, a.w[i] & 0x7fff7fffu), n = __vmaxu2(n, b.w[i] & 0x7fff7fffu);
    uint32_t w = __vmaxu2(__byte_perm(m, n, 0x5410), __byte_perm(m, n, 0x7632));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) w = __vmaxu2(w, __shfl_xor_sync(kFull, w, o));
    bits[0] = __float_as_uint(pair_to_float(w, T()).x);
    bits[1] = __float_as_uint(pair_to_float(w, T()).y);
  } else {
    bits[0] = most_of(a), bits[1] = most_of(b);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      bits[0] = max(bits[0], __shfl_xor_sync(kFull, bits[0], o)), bits[1] = max(bits[1], __shfl_xor_sync(kFull, bits[1], o));
  }
  bad[0] = not_finite(bits[0]), bad[1] = not_finite(bits[1]);
  if (__any_sync(kFull, bad[0] || bad[1])) {
    bool mine;
    uint32_t x = fp8_most(a, mine), y = fp8_most(b, mine);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x = max(x, __shfl_xor_sync(kFull, x, o)), y = max(y, __shfl_xor_sync(kFull, y, o));
    bits[0] = x, bits[1] = y;
  }
}
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
