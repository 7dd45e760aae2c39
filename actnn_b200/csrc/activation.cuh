// Activation functions with their derivatives, and 8-bit codes: what the token operators share.
//
// A code stands for code * scale, |code| <= 127, half to even:  scale = a * (1 / 127),  code = rint(x * (127 * (1 / a))),  a the
// largest magnitude of what shares the scale, at least kTiny.  Every step is one rounded fp32 operation in this order, so codes
// are reproducible to the bit.  a is found on the bit patterns of |x|, where infinities and NaNs are above all numbers; it
// becomes a NaN then, and so does the scale: everything that shares it decodes to NaN.
#pragma once

#include "common.cuh"

namespace actnn {

constexpr float kTiny = 1e-30f;

enum ActKind { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4, kActKinds = 5 };

// n / d for 0 <= n < 2^31 by one multiplication; d from 1 to 2^31 - 1.
struct FastDiv {
  uint32_t d, m, s;
};
static inline FastDiv make_fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  while (f.s < 31 && (1u << f.s) < d) ++f.s;                       // the smallest s with 2^s >= d
  f.m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << f.s) - d)) / d + 1);
  return f;
}

#ifdef __CUDACC__
ACTNN_DEV uint32_t fast_div(uint32_t n, const FastDiv& f) { return (__umulhi(n, f.m) + n) >> f.s; }

// ------------------------------------------------------------------ vectors of V elements as floats
template <typename T> ACTNN_DEV float to_float(T v);
template <> ACTNN_DEV float to_float<float>(float v) { return v; }
template <> ACTNN_DEV float to_float<__half>(__half v) { return __half2float(v); }
template <> ACTNN_DEV float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> ACTNN_DEV T from_float(float v);
template <> ACTNN_DEV float from_float<float>(float v) { return v; }
template <> ACTNN_DEV __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> ACTNN_DEV __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

ACTNN_DEV float2 pair_to_float(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
ACTNN_DEV float2 pair_to_float(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
ACTNN_DEV uint32_t pair_from_float(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
ACTNN_DEV uint32_t pair_from_float(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// V elements at p as they sit in registers; p aligned to 16 bytes or to the vector, whichever is less.
template <typename T, int V> struct Vec { uint32_t w[V * sizeof(T) / 4]; };
template <typename T> struct Vec<T, 1> { T v; };

template <typename T, int V> ACTNN_DEV Vec<T, V> load_vec(const T* p) {
  Vec<T, V> r;
  if constexpr (V == 1) {
    r.v = __ldg(p);
  } else if constexpr (V * sizeof(T) == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
  } else if constexpr (V * sizeof(T) == 8) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i)
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(r.w[4 * i]), "=r"(r.w[4 * i + 1]), "=r"(r.w[4 * i + 2]), "=r"(r.w[4 * i + 3])
                   : "l"(reinterpret_cast<const char*>(p) + 16 * i));
  }
  return r;
}
template <typename T, int V> ACTNN_DEV void unpack_vec(const Vec<T, V>& r, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = to_float(r.v);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 p = pair_to_float(r.w[i], T());
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}
template <typename T, int V> ACTNN_DEV void store_vec(T* p, const float (&f)[V]) {
  if constexpr (V == 1) {
    *p = from_float<T>(f[0]);
  } else {
    uint32_t w[V * sizeof(T) / 4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = pair_from_float(f[2 * i], f[2 * i + 1], T());
    }
    if constexpr (V * sizeof(T) == 4) {
      asm volatile("st.global.u32 [%0], %1;" :: "l"(p), "r"(w[0]) : "memory");
    } else if constexpr (V * sizeof(T) == 8) {
      asm volatile("st.global.v2.u32 [%0], {%1,%2};" :: "l"(p), "r"(w[0]), "r"(w[1]) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i)
        asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};"
                     :: "l"(reinterpret_cast<char*>(p) + 16 * i), "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]),
                        "r"(w[4 * i + 3]) : "memory");
    }
  }
}

// ------------------------------------------------------------------ codes
// The largest magnitude from the bits of the largest absolute value: kTiny at least, a NaN where it is not finite.
ACTNN_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
ACTNN_DEV float largest(uint32_t bits) {
  return __uint_as_float(bits >= 0x7f800000u ? 0x7fffffffu : max(bits, __float_as_uint(kTiny)));
}

ACTNN_DEV float code_factor(float a) { return __fmul_rn(__frcp_rn(a), 127.f); }
ACTNN_DEV float code_step(float a) { return __fmul_rn(a, 1.f / 127.f); }
// rint(x * inv) as the low byte of the returned word: adding 1.5 * 2^23 leaves the integer, half to even, in the low bits.
ACTNN_DEV uint32_t code_bits(float x, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)); }
ACTNN_DEV uint32_t pack_codes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The four signed bytes of w as floats: with its sign flipped a byte is the offset from 2^23 of the float 0x4b0000bb.
ACTNN_DEV void unpack_codes4(uint32_t w, float (&f)[4]) {
  w ^= 0x80808080u;
  f[0] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)) - 8388736.f;
  f[1] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441)) - 8388736.f;
  f[2] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)) - 8388736.f;
  f[3] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)) - 8388736.f;
}

// V codes (V = 1, 2, 4 or 8) in and out of memory, and as floats
template <int V> struct Codes { uint32_t w[(V + 3) / 4]; };
template <int V> ACTNN_DEV Codes<V> load_codes(const int8_t* p) {
  Codes<V> r;
  if constexpr (V == 1) r.w[0] = (uint32_t)__ldg(reinterpret_cast<const uint8_t*>(p));
  else if constexpr (V == 2) r.w[0] = (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p));
  else if constexpr (V == 4) asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
  else asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
  return r;
}
template <int V> ACTNN_DEV void unpack_codes(const Codes<V>& r, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = (float)(int8_t)r.w[0];
  } else if constexpr (V == 2) {
    float q[4];
    unpack_codes4(r.w[0], q);
    f[0] = q[0];
    f[1] = q[1];
  } else {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      float q[4];
      unpack_codes4(r.w[i], q);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[4 * i + j] = q[j];
    }
  }
}
// c: words whose low bytes are the codes
template <int V> ACTNN_DEV void store_codes(int8_t* p, const uint32_t (&c)[V]) {
  if constexpr (V == 1) {
    *reinterpret_cast<uint8_t*>(p) = (uint8_t)c[0];
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)__byte_perm(c[0], c[1], 0x0040);
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint32_t*>(p) = pack_codes4(c[0], c[1], c[2], c[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_codes4(c[0], c[1], c[2], c[3]), pack_codes4(c[4], c[5], c[6], c[7]));
  }
}

// ------------------------------------------------------------------ functions
// PRECISE (float32 data): expf and a rounded division, errors of an ulp or two.  16-bit data: the hardware's exponential and
// reciprocal, whose relative errors (some 1e-6 in the range that matters) vanish in the rounding to 2^-9 or 2^-12.
template <bool PRECISE> ACTNN_DEV float logistic(float z) {
  if constexpr (PRECISE) return 1.f / (1.f + expf(-z));
  else return __fdividef(1.f, 1.f + __expf(-z));                   // 0 from 1 + exp(-z) = 2^126 on
}
template <bool PRECISE> ACTNN_DEV float exp_of(float z) {
  if constexpr (PRECISE) return expf(z);
  else return __expf(z);
}

template <int KIND, bool PRECISE> ACTNN_DEV float act_value(float z) {
  if constexpr (KIND == kActRelu) return z < 0.f ? 0.f : z;                       // a NaN stays one
  if constexpr (KIND == kActSilu) return z * logistic<PRECISE>(z);
  if constexpr (KIND == kActGelu) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if constexpr (KIND == kActGeluTanh)                                              // (1 + tanh(u)) / 2 = logistic(2 u)
    return z * logistic<PRECISE>(1.5957691216057308f * (z + 0.044715f * z * z * z));
  return z;
}
// value and derivative
template <int KIND, bool PRECISE> ACTNN_DEV float2 act_both(float z) {
  if constexpr (KIND == kActRelu) return make_float2(z < 0.f ? 0.f : z, z > 0.f ? 1.f : (z == z ? 0.f : z));
  if constexpr (KIND == kActSilu) {
    const float s = logistic<PRECISE>(z);
    return make_float2(z * s, s * (1.f + z * (1.f - s)));
  }
  if constexpr (KIND == kActGelu) {
    const float p = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    return make_float2(z * p, p + z * (0.3989422804014327f * exp_of<PRECISE>(-0.5f * z * z)));
  }
  if constexpr (KIND == kActGeluTanh) {
    const float z2 = z * z;
    const float s = logistic<PRECISE>(1.5957691216057308f * z * (1.f + 0.044715f * z2));
    const float t = s * (1.f - s);                                  // zero far out, where z2 may have overflowed
    return make_float2(z * s, t == 0.f ? s : s + z * t * (1.5957691216057308f * (1.f + 0.134145f * z2)));
  }
  return make_float2(z, 1.f);
}
#endif  // __CUDACC__

}  // namespace actnn
