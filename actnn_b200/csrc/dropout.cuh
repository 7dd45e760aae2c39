// Dropout decided by a counter-based generator: what an element's place and a key say, wherever and whenever they are asked.
//
// Element e of a tensor has the 16-bit field e % 8 (words and their halves upwards) of the Philox4x32-10 output for counter e / 8 and
// key (seed, offset), the fields that the dropout with a stored mask compares.  It is kept where field + 1 > 65536 p, which in
// integers is field >= floor(65536 p), and multiplied by 1 / (1 - p).
#pragma once

#include "activation.cuh"
#include "load_one.cuh"

namespace actnn {

// A key on the host, or, where a launch is replayed with another one every time, on the device.
struct DropKey {
  NoiseKey key;
  const int64_t* state;        // (seed, offset) on the device, or NULL: `key`
  uint32_t least;              // the least field that is kept, in the upper half of a word
  float inv;                   // 1 / (1 - p)
};
static inline DropKey make_drop_key(float p, uint64_t seed, uint64_t offset, const int64_t* state) {
  return DropKey{make_noise_key(seed, offset), state, (uint32_t)((double)p * 65536.) << 16, (float)(1.0 / (1.0 - (double)p))};
}

#ifdef __CUDACC__
// The key of a launch.  From the device the round keys cost twenty additions a thread.
ACTNN_DEV NoiseKey drop_key(const DropKey& d) {
  if (!d.state) return d.key;
  uint64_t seed, offset;
  asm volatile("ld.global.v2.u64 {%0,%1}, [%2];" : "=l"(seed), "=l"(offset) : "l"(d.state));
  NoiseKey k;
  uint32_t a = (uint32_t)seed, b = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    k.k0[r] = a; k.k1[r] = b;
    a += 0x9E3779B9u; b += 0xBB67AE85u;
  }
  k.o0 = (uint32_t)offset; k.o1 = (uint32_t)(offset >> 32);
  return k;
}
// What an element is multiplied by, for the eight of a call: inv or zero.
ACTNN_DEV void drop_factors(const Philox4& r, uint32_t least, float inv, float2 (&m)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = make_float2((r.v[i] << 16) >= least ? inv : 0.f, r.v[i] >= least ? inv : 0.f);
}
// The eight elements of a call: kept ones times inv, others zero whatever they were.  (A field's lower neighbour does not reach the
// comparison of the upper one: least has no bits there.)
ACTNN_DEV void drop_oct(float2 (&f)[4], const Philox4& r, uint32_t least, float inv) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = f_mul(f[i], make_float2(inv, inv));
    f[i] = make_float2((r.v[i] << 16) >= least ? y.x : 0.f, r.v[i] >= least ? y.y : 0.f);
  }
}
#endif

}  // namespace actnn
