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

// ------------------------------------------------------------------ pairs
// This GPU has fp32 additions, products and fused products of two numbers in one instruction, each rounded as the single ones
// are.  The arithmetic of the token operators is written for F = float2 (pairs) and F = float (vectors of one element).
ACTNN_DEV uint64_t bits_of(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
ACTNN_DEV float2 pair_of(uint64_t r) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
ACTNN_DEV float2 f_add(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
  return pair_of(r);
}
ACTNN_DEV float2 f_mul(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
  return pair_of(r);
}
ACTNN_DEV float2 f_fma(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
  return pair_of(r);
}
ACTNN_DEV float f_add(float a, float b) { return __fadd_rn(a, b); }
ACTNN_DEV float f_mul(float a, float b) { return __fmul_rn(a, b); }
ACTNN_DEV float f_fma(float a, float b, float c) { return __fmaf_rn(a, b, c); }
template <typename F> ACTNN_DEV F f_both(float v);
template <> ACTNN_DEV float f_both<float>(float v) { return v; }
template <> ACTNN_DEV float2 f_both<float2>(float v) { return make_float2(v, v); }
// op on each number
template <typename Op> ACTNN_DEV float f_each(float v, Op op) { return op(v); }
template <typename Op> ACTNN_DEV float2 f_each(float2 v, Op op) { return make_float2(op(v.x), op(v.y)); }
ACTNN_DEV float f_sum(float v) { return v; }
ACTNN_DEV float f_sum(float2 v) { return v.x + v.y; }

// V numbers of a thread: V / 2 pairs, or one.
template <int V> struct Many { using F = float2; static constexpr int N = V / 2; };
template <> struct Many<1> { using F = float; static constexpr int N = 1; };

// ------------------------------------------------------------------ vectors of V elements
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
ACTNN_DEV uint32_t pair_from_float(float2 v, __half) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
ACTNN_DEV uint32_t pair_from_float(float2 v, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// As they sit in registers; the address is a multiple of 16 bytes or of the vector, whichever is less.
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
template <typename T, int V> ACTNN_DEV void unpack_vec(const Vec<T, V>& r, typename Many<V>::F (&f)[Many<V>::N]) {
  if constexpr (V == 1) {
    f[0] = to_float(r.v);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (sizeof(T) == 4) f[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
      else f[i] = pair_to_float(r.w[i], T());
    }
  }
}
// STREAM: written once and not read soon (evict first).
template <typename T, int V, bool STREAM = false> ACTNN_DEV void store_vec(T* p, const typename Many<V>::F (&f)[Many<V>::N]) {
  if constexpr (V == 1) {
    *p = from_float<T>(f[0]);
  } else {
    uint32_t w[V * sizeof(T) / 4];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[2 * i] = __float_as_uint(f[i].x);
        w[2 * i + 1] = __float_as_uint(f[i].y);
      } else {
        w[i] = pair_from_float(f[i], T());
      }
    }
    if constexpr (V * sizeof(T) == 4) {
      asm volatile("st.global.u32 [%0], %1;" :: "l"(p), "r"(w[0]) : "memory");
    } else if constexpr (V * sizeof(T) == 8) {
      asm volatile("st.global.v2.u32 [%0], {%1,%2};" :: "l"(p), "r"(w[0]), "r"(w[1]) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i)
        if constexpr (STREAM) asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};"
                     :: "l"(reinterpret_cast<char*>(p) + 16 * i), "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]),
                        "r"(w[4 * i + 3]) : "memory");
        else asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};"
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
// The largest magnitude of a vector, as bits.  16-bit types compare their halves: the sign bit cleared, the order is that of
// unsigned numbers.
template <typename T, int V> ACTNN_DEV uint32_t most_of(const Vec<T, V>& r) {
  if constexpr (V == 1) {
    return abs_bits(to_float(r.v));
  } else if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, r.w[i] & 0x7fffffffu);
    return m;
  } else {
    uint32_t m = r.w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < V / 2; ++i) m = __vmaxu2(m, r.w[i] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    return abs_bits(pair_to_float(m, T()).x);
  }
}

ACTNN_DEV float code_factor(float a) { return __fmul_rn(__frcp_rn(a), 127.f); }
ACTNN_DEV float code_step(float a) { return __fmul_rn(a, 1.f / 127.f); }
// rint(x * inv) as the low byte of the float's bits: adding 1.5 * 2^23 leaves the integer, half to even, in the low bits.  The
// product is written as a fused one with zero: as a plain product of a pair the compiler fuses it with the addition, which
// skips a rounding and moves codes at ties.
template <typename F> ACTNN_DEV F code_bits(F x, F inv) { return f_add(f_fma(x, inv, f_both<F>(0.f)), f_both<F>(12582912.f)); }
ACTNN_DEV uint32_t pack_codes4(float2 a, float2 b) {
  return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                     __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}
// The four signed bytes of w as floats: with its sign flipped a byte is the offset from 2^23 of the float 0x4b0000bb.
ACTNN_DEV void unpack_codes4(uint32_t w, float2& a, float2& b) {
  w ^= 0x80808080u;
  const float2 off = make_float2(-8388736.f, -8388736.f);
  a = f_add(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441))), off);
  b = f_add(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443))), off);
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
template <int V> ACTNN_DEV void unpack_codes(const Codes<V>& r, typename Many<V>::F (&f)[Many<V>::N]) {
  if constexpr (V == 1) {
    f[0] = (float)(int8_t)r.w[0];
  } else if constexpr (V == 2) {
    float2 none;
    unpack_codes4(r.w[0], f[0], none);
  } else {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) unpack_codes4(r.w[i], f[2 * i], f[2 * i + 1]);
  }
}
// c: floats whose low bytes are the codes
template <int V> ACTNN_DEV void store_codes(int8_t* p, const typename Many<V>::F (&c)[Many<V>::N]) {
  if constexpr (V == 1) {
    *reinterpret_cast<uint8_t*>(p) = (uint8_t)__float_as_uint(c[0]);
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)__byte_perm(__float_as_uint(c[0].x), __float_as_uint(c[0].y), 0x0040);
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint32_t*>(p) = pack_codes4(c[0], c[1]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_codes4(c[0], c[1]), pack_codes4(c[2], c[3]));
  }
}

// ------------------------------------------------------------------ functions
// PRECISE (float32 data): expf, erff and rounded divisions, errors of an ulp or two.  16-bit data: the hardware's exponential
// and reciprocal, one instruction each, whose relative errors (some 1e-6 in the range that matters) vanish in the rounding to
// 2^-9 or 2^-12; with subnormal numbers flushed they need no scaling around them.
ACTNN_DEV float fast_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
ACTNN_DEV float fast_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + exp(-z * factor))
template <bool PRECISE, typename F> ACTNN_DEV F logistic(F z, float factor) {
  if constexpr (PRECISE) {
    return f_each(z, [=](float v) { return 1.f / (1.f + expf(-v * factor)); });
  } else {
    const F e = f_each(f_mul(z, f_both<F>(-kLog2e * factor)), [](float v) { return fast_exp2(v); });
    return f_each(f_add(e, f_both<F>(1.f)), [](float v) { return fast_rcp(v); });
  }
}

// The normal distribution's function and density at z.  Fast form: 1 - erf(x) = (a1 t + ... + a5 t^5) exp(-x^2) + e,
// t = 1 / (1 + p x), |e| < 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26), at x = |z| / sqrt(2);
// half of it is the distribution's tail, and exp(-x^2) is the density's exponential.  Far out the tail's own relative error is what
// counts: 0.0016 of it down to z = -5, 0.0036 to -6, 0.010 to -8.  Precise form: the sum of one and erf, errors of 2^-24 of one; erfc, whose errors are of the tail
// itself, made 8192 x 4096 float32 elements 72 us forward and 73 back instead of 58 and 62.
template <bool PRECISE, bool DENSITY, typename F> ACTNN_DEV void normal(F z, F& below, F& density) {
  if constexpr (PRECISE) {
    below = f_each(z, [](float v) { return 0.5f * (1.f + erff(v * 0.70710678118654752f)); });
    if constexpr (DENSITY) density = f_each(z, [](float v) { return 0.3989422804014327f * expf(-0.5f * v * v); });
  } else {
    const F x = f_each(z, [](float v) { return fabsf(v); });
    const F t = f_each(f_fma(x, f_both<F>(0.3275911f * 0.70710678118654752f), f_both<F>(1.f)), [](float v) { return fast_rcp(v); });
    const F e = f_each(f_mul(f_mul(z, z), f_both<F>(-0.5f * kLog2e)), [](float v) { return fast_exp2(v); });
    F p = f_fma(t, f_both<F>(0.5f * 1.061405429f), f_both<F>(0.5f * -1.453152027f));
    p = f_fma(p, t, f_both<F>(0.5f * 1.421413741f));
    p = f_fma(p, t, f_both<F>(0.5f * -0.284496736f));
    p = f_fma(p, t, f_both<F>(0.5f * 0.254829592f));
    const F tail = f_mul(f_mul(p, t), e);
    // The tail as it is below zero, 1 - tail above, by the sign m of -z: m * tail + (1 - m) / 2.  (Half plus or minus half less the
    // tail would be gone at -6.)
    const F m = f_each(z, [](float v) { return __uint_as_float((~__float_as_uint(v) & 0x80000000u) | 0x3f800000u); });
    below = f_fma(tail, m, f_fma(m, f_both<F>(-0.5f), f_both<F>(0.5f)));
    if constexpr (DENSITY) density = f_mul(e, f_both<F>(0.3989422804014327f));
  }
}

template <int KIND, bool PRECISE, typename F> ACTNN_DEV F act_value(F z) {
  if constexpr (KIND == kActRelu) return f_each(z, [](float v) { return v < 0.f ? 0.f : v; });       // a NaN stays one
  if constexpr (KIND == kActSilu) return f_mul(z, logistic<PRECISE>(z, 1.f));
  if constexpr (KIND == kActGelu) {
    F below, none;
    normal<PRECISE, false>(z, below, none);
    return f_mul(z, below);
  }
  if constexpr (KIND == kActGeluTanh) {                             // (1 + tanh(u)) / 2 = logistic(2 u)
    const F z2 = f_each(f_mul(z, z), [](float v) { return fminf(v, 1e4f); });
    return f_mul(z, logistic<PRECISE>(f_mul(z, f_fma(z2, f_both<F>(0.044715f), f_both<F>(1.f))), 1.5957691216057308f));
  }
  return z;
}
// derivative, and the value on request
template <int KIND, bool PRECISE, typename F> ACTNN_DEV F act_slope(F z, F* value = nullptr) {
  const F one = f_both<F>(1.f), minus = f_both<F>(-1.f);
  if constexpr (KIND == kActRelu) {
    if (value) *value = act_value<kActRelu, PRECISE>(z);
    return f_each(z, [](float v) { return v > 0.f ? 1.f : (v == v ? 0.f : v); });
  } else if constexpr (KIND == kActSilu) {
    const F s = logistic<PRECISE>(z, 1.f);
    if (value) *value = f_mul(z, s);
    return f_mul(s, f_fma(z, f_fma(s, minus, one), one));
  } else if constexpr (KIND == kActGelu) {
    F below, density;
    normal<PRECISE, true>(z, below, density);
    if (value) *value = f_mul(z, below);
    return f_fma(z, density, below);
  } else if constexpr (KIND == kActGeluTanh) {
    // far out, where z * z may have overflowed, s (1 - s) is zero: the square is held at 1e4
    const F z2 = f_each(f_mul(z, z), [](float v) { return fminf(v, 1e4f); });
    const F s = logistic<PRECISE>(f_mul(z, f_fma(z2, f_both<F>(0.044715f), one)), 1.5957691216057308f);
    if (value) *value = f_mul(z, s);
    const F t = f_mul(s, f_fma(s, minus, one));
    return f_fma(f_mul(z, t), f_fma(z2, f_both<F>(1.5957691216057308f * 0.134145f), f_both<F>(1.5957691216057308f)), s);
  } else {
    if (value) *value = z;
    return one;
  }
}
#endif  // __CUDACC__

}  // namespace actnn
