// Loads of one element that stay behind the condition they stand under.  The toolkit's own load of a 16-bit type is assembly without
// effects to the compiler, which may move it before a branch: a pointer that may be NULL, or a row that is not there, was then read.
#pragma once

#include "common.cuh"

namespace actnn {
#ifdef __CUDACC__
ACTNN_DEV float load_one(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
ACTNN_DEV __half load_one(const __half* p) {
  uint16_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return __ushort_as_half(v);
}
ACTNN_DEV __nv_bfloat16 load_one(const __nv_bfloat16* p) {
  uint16_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return __ushort_as_bfloat16(v);
}
ACTNN_DEV uint32_t load_one(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
#endif
}  // namespace actnn
