// The norms before and after a block with its gate and residual scale, on rows of C channels:
//
//   u = (f - m1) p1 w1 + b1        the block's output f, normalised (or as it is)
//   d = keep u / (1 - p)           dropout (dropout.cuh)
//   r = s x + g d                  the residual stream x, scaled, and what passes the gate
//   h = (r - m2) p2 w2 + b2        what the next block reads
//
// m, p: mean and reciprocal deviation of the row, sqrt(mean((v - m)^2) + eps); the rms kind has m = 0.  What the backward pass
// keeps are the inputs x and f in 8 bits, a scale for 256 channels of a row, and the four statistics: codes of inputs follow from
// exact numbers, those of r would move with the last bit of a sum.  With n1, n2 the normalised values made of the decoded inputs:
//
//   dn2 = dh w2      c = dr + p2 dn2      t = c - p2 (mean dn2 + n2 mean(dn2 n2))      dx = s t      dg = sum t d
//   du = keep g t / (1 - p)      dn1 = du w1      df = p1 (dn1 - mean dn1 - n1 mean(dn1 n1))
//   dw2 = sum dh n2, db2 = sum dh, dw1 = sum du n1, db1 = sum du   over the rows
//
// With a = keep g w1 / (1 - p), dn1 is a t, so that the means of the second norm's gradient follow from sums that do not wait for
// those of the first: mean(dn1 n1) = (sum a c n1 - p2 mean dn2 sum a n1 - p2 mean(dn2 n2) sum a n1 n2) / C.  A row takes one
// joint reduction, not two.
//
// What is not finite goes where these formulas take it.  A mean that is not finite, or a NaN, makes a row's normalised values NaN; an infinity without
// a mean (rms) has p = 0, so that its own channel is NaN and the row's others are zero.  The gradients of such a row are NaN, and no other row's are
// touched.
//
// 8192 x 4096 bf16 with dropout: forward 80 us, backward 102, the join 6 (51 and 51 at the copy rate); 16384 x 8192 f16 without: 251, 355, 8
// (205 each); 12608 x 768 float32, layer kind: 32, 37, 6 (27 each).  Forward is bound by instructions (issue slots 71 % busy); backward by
// some 470 of them a warp's 256 channels, of which dropout's generator takes 70, and by a row's barrier: registers allow one block of 16 warps an
// SM, which stand at it together (issue slots 56 % busy).
#pragma once

#include <algorithm>
#include <type_traits>

#include "cluster.cuh"
#include "dropout.cuh"

namespace actnn {

constexpr int kRnBlock = 256;                          // channels that share a scale
constexpr int kRnMostC = 32768;
constexpr int kRnThreads = 256;                        // of the kernels that give a warp a row
constexpr int kRnMostThreads = 512, kRnMostCluster = 8;          // of the backward pass: eight channels a thread

// A tensor of one of the three types, that of `dtype`; -1: not given, ones or zeros (then `p` can be read all the same).
struct RnParameter {
  const void* p;
  int dtype;
#ifdef __CUDACC__
  ACTNN_DEV bool given() const { return dtype >= 0; }
#endif
};
struct RnArgs {
  const void *x, *f;                                   // forward; backward where no codes were kept
  const void *dr, *dh;                                 // gradients, NULL: zero
  RnParameter w1, b1, w2, b2, gate;
  void *r, *h, *dx, *df;                               // dx, df NULL: not wanted
  int8_t *cx, *cf;                                     // codes [rows, C], NULL: none
  float *sx, *sf;                                      // their scales [rows, ceil(C / 256)]
  float4* stats;                                       // [rows]: m1, p1, m2, p2
  float* parts;                                        // [runs][slots][C], backward: partial sums of the parameters' gradients
  void *dw2, *db2, *dw1, *db1, *dgate;                 // the parameters' gradients
  uint32_t rows;
  int C, blocks;                                       // blocks: scales a row
  float scale, eps, inv_c;
  int pdtype, gdtype;                                  // types of their gradients
  bool layer, post, dropped;
  FastDiv by_gate;                                     // rows of a gate
  DropKey drop;
  // the runs of rows of the backward pass
  int cluster;                                                  // blocks that share a row
  int slots, slot_w2, slot_b2, slot_w1, slot_b1, slot_gate;     // -1: not wanted
  uint32_t unit_rows, units;                                    // rows whose sums belong together: those of a gate where its gradient is wanted, else all
  uint32_t runs_of_unit, units_of_run, runs;                    // units_of_run > 0: a run is so many whole units, else a part of one
  bool coded;                                                   // backward: of codes, else of x and f
  cudaStream_t stream;
};
int rn_blocks_per_sm(const void* kernel, int threads, int smem);           // resident at a time; raises the kernel's limit of shared memory
enum RnWhat { kRnForward, kRnBackward };
int rn_run_f32(const RnArgs& a, RnWhat what, bool vec);
int rn_run_f16(const RnArgs& a, RnWhat what, bool vec);
int rn_run_bf16(const RnArgs& a, RnWhat what, bool vec);

#ifdef __CUDACC__
// Loads that stay where they stand (load_one.cuh).
ACTNN_DEV float rn_ld(const float* p) { return load_one(p); }
ACTNN_DEV float2 rn_ld(const float2* p) {
  float2 v;
  asm volatile("ld.global.nc.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
ACTNN_DEV float4 rn_ld(const float4* p) {
  float4 v;
  asm volatile("ld.global.nc.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
ACTNN_DEV uint4 rn_ld(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// ------------------------------------------------------------------ eight channels of a thread
// Element `c` of a row that all threads have in common, by a 32-bit offset.
template <typename T> ACTNN_DEV T* rn_at(T* row, int c) {
  return (T*)((std::conditional_t<std::is_const_v<T>, const char, char>*)row + (uint32_t)c * (uint32_t)sizeof(T));
}
// Elements from `c` on, zero behind C.
template <typename T, bool VEC> ACTNN_DEV Vec<T, 8> rn_load(const T* row, int c, int C) {
  Vec<T, 8> v;
  if (VEC && c < C) return load_vec<T, 8>(rn_at(row, c));
#pragma unroll
  for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(v.w)[i] = !VEC && c + i < C ? load_one(row + c + i) : from_float<T>(0.f);
  return v;
}
template <typename T, bool VEC> ACTNN_DEV void rn_store(T* row, int c, int C, const float2 (&f)[4]) {
  if constexpr (VEC) {
    if (c < C) store_vec<T, 8>(rn_at(row, c), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < C) row[c + i] = from_float<T>(i & 1 ? f[i / 2].y : f[i / 2].x);
  }
}
template <bool VEC> ACTNN_DEV Codes<8> rn_load_codes(const int8_t* row, int c, int C) {
  Codes<8> r;
  r.w[0] = r.w[1] = 0;
  if constexpr (VEC) {
    if (c < C) r = load_codes<8>(rn_at(row, c));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < C) r.w[i / 4] |= load_one(reinterpret_cast<const uint8_t*>(row) + c + i) << (8 * (i % 4));
  }
  return r;
}
template <bool VEC> ACTNN_DEV void rn_store_codes(int8_t* row, int c, int C, const float2 (&f)[4]) {
  if constexpr (VEC) {
    if (c < C) store_codes<8>(rn_at(row, c), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < C) row[c + i] = (int8_t)__float_as_uint(i & 1 ? f[i / 2].y : f[i / 2].x);
  }
}
// A parameter's values, of any of the three types; through the L1, every row reads them again.
template <bool VEC, typename P> ACTNN_DEV void rn_values(const P* p, int c, int C, float2 (&f)[4]) {
  if constexpr (VEC) {
    Vec<P, 8> v;
#pragma unroll
    for (int i = 0; i < (int)sizeof(P) / 2; ++i) {
      const uint4 q = c < C ? rn_ld(reinterpret_cast<const uint4*>(p + c) + i) : make_uint4(0, 0, 0, 0);
      v.w[4 * i] = q.x, v.w[4 * i + 1] = q.y, v.w[4 * i + 2] = q.z, v.w[4 * i + 3] = q.w;
    }
    unpack_vec(v, f);
  } else {
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c + i < C ? to_float(load_one(p + c + i)) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(e[2 * i], e[2 * i + 1]);
  }
}
template <bool VEC> ACTNN_DEV void rn_parameter(const RnParameter& q, int c, int C, float none, float2 (&f)[4]) {
  if (!q.given()) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(none, none);
  } else if (q.dtype == ACTNN_F32) {
    rn_values<VEC>((const float*)q.p, c, C, f);
  } else if (q.dtype == ACTNN_F16) {
    rn_values<VEC>((const __half*)q.p, c, C, f);
  } else {
    rn_values<VEC>((const __nv_bfloat16*)q.p, c, C, f);
  }
}
ACTNN_DEV RnParameter rn_gate_row(const RnArgs& a, uint32_t row) {
  if (!a.gate.given()) return a.gate;
  return RnParameter{(const char*)a.gate.p + (size_t)fast_div(row, a.by_gate) * a.C * (a.gate.dtype == ACTNN_F32 ? 4 : 2), a.gate.dtype};
}
// The fields that decide over the eight channels from `c` of a row, two a word.  Where C is no multiple of eight they belong to two calls.
// (Both directions multiply by factors: an element that is not finite is NaN where it is dropped.)
template <bool VEC> ACTNN_DEV Philox4 rn_fields(const RnArgs& a, const NoiseKey& key, uint32_t row, int c) {
  const uint64_t e = (uint64_t)row * a.C + c;
  Philox4 r = noise_call(key, e >> 3);
  if (VEC) return r;
  const Philox4 q = noise_call(key, (e >> 3) + 1);
  const uint32_t at = (uint32_t)e & 7;                  // fields to leave out: four, two and one
  uint32_t w[8] = {r.v[0], r.v[1], r.v[2], r.v[3], q.v[0], q.v[1], q.v[2], q.v[3]};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = at & 4 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = at & 2 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = __funnelshift_r(w[i], w[i + 1], at & 1 ? 16 : 0);
  return r;
}
// ------------------------------------------------------------------ forward
// The sum over the threads of a row: a warp's, or a block's, whose reductions take two places in turn (two are never under way at a time).
// Places of warps that are not there hold zero.
struct RnPlaces { float part[2][kRnMostThreads / 32]; };
template <bool WARP> ACTNN_DEV float rn_sum(float v, RnPlaces& s, int& place) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  if constexpr (!WARP) {
    constexpr int kWarps = kRnMostThreads / 32;
    const int lane = threadIdx.x & 31;
    if (lane == 0) s.part[place][threadIdx.x >> 5] = v;
    __syncthreads();
    v = s.part[place][lane & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    place ^= 1;
  }
  return v;
}
// Mean (of the layer kind) and reciprocal deviation of a row.  Values behind C are zero.
template <int V, bool WARP, bool LAYER> ACTNN_DEV float2 rn_statistics(const float2 (&v)[V][4], int c0, int step, const RnArgs& a, RnPlaces& places, int& place) {
  float mean = 0.f;
  float2 s = make_float2(0.f, 0.f);
  if constexpr (LAYER) {
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = f_add(s, v[k][i]);
    mean = rn_sum<WARP>(f_sum(s), places, place) * a.inv_c;
    s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = c0 + k * step;
      if (c + 8 <= a.C) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = f_add(v[k][i], make_float2(-mean, -mean));
          s = f_fma(e, e, s);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 e = make_float2(c + 2 * i < a.C ? v[k][i].x - mean : 0.f, c + 2 * i + 1 < a.C ? v[k][i].y - mean : 0.f);
          s = f_fma(e, e, s);
        }
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = f_fma(v[k][i], v[k][i], s);
  }
  return make_float2(mean, rsqrtf(rn_sum<WARP>(f_sum(s), places, place) * a.inv_c + a.eps));
}

// The parameters of a thread's channels in shared memory, as float32: what every row reads again takes two loads and no conversion.
// Sets of two halves, [set][half][vector * threads + thread].
ACTNN_DEV void rn_put(float4* at, int width, const float2 (&v)[4]) {
  at[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
  at[width] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
}
ACTNN_DEV void rn_get(const float4* at, int width, float2 (&v)[4]) {
  const float4 p = at[0], q = at[width];
  v[0] = make_float2(p.x, p.y), v[1] = make_float2(p.z, p.w), v[2] = make_float2(q.x, q.y), v[3] = make_float2(q.z, q.w);
}
enum RnSet { kRnGw, kRnW2, kRnGb, kRnB2 };             // w1 and b1 times the gate
template <bool LAYER> constexpr int rn_sets() { return LAYER ? 4 : 2; }

// A warp, or a block, goes through rows; a thread has V vectors of eight channels of each.  The next row's inputs are requested as soon
// as this row's are unpacked (unless V is so large that registers are short), so that the two or four reductions of a row do
// not wait for memory.
template <typename T, int V, bool WARP, bool VEC, bool LAYER>
__global__ void __launch_bounds__(WARP ? kRnThreads : kRnMostThreads, V == 1 && !WARP ? 2 : 1) rn_forward_kernel(const __grid_constant__ RnArgs a) {
  constexpr bool kAhead = V <= 4, kShared = V <= 2;     // parameters in shared memory, or read from the L1
  extern __shared__ float4 parameters_s[];
  __shared__ RnPlaces places;
  const int lanes = WARP ? 32 : blockDim.x, lane = WARP ? threadIdx.x & 31 : threadIdx.x, c0 = lane * 8, step = lanes * 8;
  const int width = V * blockDim.x;
  const uint32_t rows_step = WARP ? gridDim.x * (kRnThreads / 32) : gridDim.x;
  uint32_t row = WARP ? blockIdx.x * (kRnThreads / 32) + (threadIdx.x >> 5) : blockIdx.x, gate_of = 0;
  Vec<T, 8> xv[V], fv[V];
  auto load = [&](uint32_t r) {
    const size_t at = (size_t)r * a.C;
    const T *f = (const T*)a.f + at, *x = (const T*)a.x + at;
#pragma unroll
    for (int k = 0; k < V; ++k) fv[k] = rn_load<T, VEC>(f, c0 + k * step, a.C);
#pragma unroll
    for (int k = 0; k < V; ++k) xv[k] = rn_load<T, VEC>(x, c0 + k * step, a.C);
  };
  if (kAhead && row < a.rows) load(row);
  auto slot = [&](int set, int k) { return parameters_s + 2 * set * width + k * blockDim.x + threadIdx.x; };
  auto read = [&](const RnParameter& p, float none, int k, float2 (&v)[4]) { rn_parameter<VEC>(p, c0 + k * step, a.C, none, v); };
  // w1 or b1 times the gate of a row.
  auto product = [&](const RnParameter& p, float none, const RnParameter& gate, int k, float2 (&v)[4]) {
    read(p, none, k, v);
    if (!gate.given()) return;
    float2 q[4];
    read(gate, 1.f, k, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f_mul(v[i], q[i]);
  };
  auto put_products = [&](const RnParameter& gate) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float2 v[4];
      product(a.w1, 1.f, gate, k, v);
      rn_put(slot(kRnGw, k), width, v);
      if (LAYER) {
        product(a.b1, 0.f, gate, k, v);
        rn_put(slot(kRnGb, k), width, v);
      }
    }
  };
  if (!WARP && threadIdx.x < sizeof(places) / 4) (&places.part[0][0])[threadIdx.x] = 0.f;
  if constexpr (kShared) {
    if (a.gate.given()) gate_of = fast_div(row, a.by_gate);
    if (row < a.rows) put_products(rn_gate_row(a, row));
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float2 v[4];
      read(a.w2, 1.f, k, v);
      rn_put(slot(kRnW2, k), width, v);
      if (LAYER) {
        read(a.b2, 0.f, k, v);
        rn_put(slot(kRnB2, k), width, v);
      }
    }
  }
  if (!WARP) __syncthreads();
  const bool scaled = a.post || a.gate.given();
  NoiseKey key;
  if (a.dropped) key = drop_key(a.drop);
  for (int place = 0; row < a.rows; row += rows_step) {
    const size_t at = (size_t)row * a.C;
    if (!kAhead) load(row);
    if (a.cx) {
      // A warp's vectors are 256 channels that share a scale; the factors of both inputs are made at once, one in each half of the warp.
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = c0 + k * step, first = c & ~(kRnBlock - 1);
        if (V > 1 && first >= a.C) continue;
        const uint32_t mf = __reduce_max_sync(kFull, most_of(fv[k])), mx = __reduce_max_sync(kFull, most_of(xv[k]));
        const bool upper = threadIdx.x & 16;
        const float most = largest(upper ? mx : mf), factor = code_factor(most);
        auto code = [&](const Vec<T, 8>& v, int8_t* codes, float by) {
          float2 q[4];
          unpack_vec(v, q);
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = code_bits(q[i], make_float2(by, by));
          rn_store_codes<VEC>(codes + at, c, a.C, q);
        };
        code(fv[k], a.cf, __shfl_sync(kFull, factor, 0));
        code(xv[k], a.cx, __shfl_sync(kFull, factor, 16));
        if ((threadIdx.x & 15) == 0) *rn_at((upper ? a.sx : a.sf) + (size_t)row * a.blocks, first / kRnBlock) = code_step(most);
      }
    }
    float2 u[V][4], x[V][4];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      unpack_vec(fv[k], u[k]);
      unpack_vec(xv[k], x[k]);
    }
    if (kAhead && row + rows_step < a.rows) load(row + rows_step);
    const float2 one = a.post ? rn_statistics<V, WARP, LAYER>(u, c0, step, a, places, place) : make_float2(0.f, 1.f);
    RnParameter gate = a.gate;
    if (a.gate.given()) {
      if (const uint32_t g = fast_div(row, a.by_gate); !kShared || g != gate_of) {
        gate = rn_gate_row(a, row);
        if (kShared) put_products(gate);
        gate_of = g;
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = c0 + k * step;
      float2 p[4];
      if (a.post) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (LAYER) u[k][i] = f_add(u[k][i], make_float2(-one.x, -one.x));
          u[k][i] = f_mul(u[k][i], make_float2(one.y, one.y));
        }
      }
      if (scaled) {
        if constexpr (kShared) rn_get(slot(kRnGw, k), width, p);
        else product(a.w1, 1.f, gate, k, p);
        if constexpr (LAYER) {
          float2 b[4];
          if constexpr (kShared) rn_get(slot(kRnGb, k), width, b);
          else product(a.b1, 0.f, gate, k, b);
#pragma unroll
          for (int i = 0; i < 4; ++i) u[k][i] = f_fma(u[k][i], p[i], b[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) u[k][i] = f_mul(u[k][i], p[i]);
        }
      }
      if (a.dropped) {
        drop_factors(rn_fields<VEC>(a, key, row, c), a.drop.least, a.drop.inv, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[k][i] = f_mul(u[k][i], p[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) u[k][i] = f_fma(x[k][i], make_float2(a.scale, a.scale), u[k][i]);
      rn_store<T, VEC>((T*)a.r + at, c, a.C, u[k]);
      if ((LAYER || !VEC) && c + 8 > a.C) {             // nothing behind C enters the sums
#pragma unroll
        for (int i = 0; i < 4; ++i) u[k][i] = make_float2(c + 2 * i < a.C ? u[k][i].x : 0.f, c + 2 * i + 1 < a.C ? u[k][i].y : 0.f);
      }
    }
    const float2 two = rn_statistics<V, WARP, LAYER>(u, c0, step, a, places, place);
    if (a.stats && lane == 0) a.stats[row] = make_float4(one.x, one.y, two.x, two.y);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = c0 + k * step;
      float2 p[4];
      if constexpr (kShared) rn_get(slot(kRnW2, k), width, p);
      else read(a.w2, 1.f, k, p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (LAYER) u[k][i] = f_add(u[k][i], make_float2(-two.x, -two.x));
        u[k][i] = f_mul(f_mul(u[k][i], make_float2(two.y, two.y)), p[i]);
      }
      if constexpr (LAYER) {
        if constexpr (kShared) rn_get(slot(kRnB2, k), width, p);
        else read(a.b2, 0.f, k, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[k][i] = f_add(u[k][i], p[i]);
      }
      rn_store<T, VEC>((T*)a.h + at, c, a.C, u[k]);
    }
  }
}

// ------------------------------------------------------------------ backward
// What the backward pass reads of eight channels of a row, as it lies in memory.
template <typename T, bool CODED> struct RnRaw {
  Vec<T, 8> dr, dh, x, f;
};
template <typename T> struct RnRaw<T, true> {
  Vec<T, 8> dr, dh;
  Codes<8> x, f;
  float sx, sf;
};
template <typename T, bool CODED, bool VEC> ACTNN_DEV void rn_load_raw(RnRaw<T, CODED>& v, const RnArgs& a, uint32_t row, int c) {
  const size_t at = (size_t)row * a.C;
  const int C = a.C;
  v.dr = rn_load<T, VEC>((const T*)a.dr + at, a.dr ? c : C, C);
  v.dh = rn_load<T, VEC>((const T*)a.dh + at, a.dh ? c : C, C);
  if constexpr (CODED) {
    v.x = rn_load_codes<VEC>(a.cx + at, c, C);
    v.f = rn_load_codes<VEC>(a.cf + at, c, C);
    v.sx = v.sf = 0.f;
    if (c < C) {
      const size_t s = (size_t)row * a.blocks;
      v.sx = rn_ld(rn_at((const float*)a.sx + s, c / kRnBlock));
      v.sf = rn_ld(rn_at((const float*)a.sf + s, c / kRnBlock));
    }
  } else {
    v.x = rn_load<T, VEC>((const T*)a.x + at, c, C);
    v.f = rn_load<T, VEC>((const T*)a.f + at, c, C);
  }
}
// p2 (scale x - m2), and n1 = (f - m1) p1.
template <typename T, bool CODED, bool LAYER>
ACTNN_DEV void rn_inputs(const RnRaw<T, CODED>& v, const RnArgs& a, const float4& st, float2 (&x)[4], float2 (&n1)[4]) {
  float by_x = a.scale * st.w, by_f = st.y;
  if constexpr (CODED) {
    unpack_codes(v.x, x);
    unpack_codes(v.f, n1);
    by_x *= v.sx;
    if (!LAYER) by_f *= v.sf;
    if (LAYER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) n1[i] = f_fma(n1[i], make_float2(v.sf, v.sf), make_float2(-st.x, -st.x));
    }
  } else {
    unpack_vec(v.x, x);
    unpack_vec(v.f, n1);
    if (LAYER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) n1[i] = f_add(n1[i], make_float2(-st.x, -st.x));
    }
  }
  const float m = -st.z * st.w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = LAYER ? f_fma(x[i], make_float2(by_x, by_x), make_float2(m, m)) : f_mul(x[i], make_float2(by_x, by_x));
    n1[i] = f_mul(n1[i], make_float2(by_f, by_f));
  }
}
ACTNN_DEV void rn_store_any(void* p, int dtype, size_t at, float v) {
  if (dtype == ACTNN_F32) ((float*)p)[at] = v;
  else if (dtype == ACTNN_F16) ((__half*)p)[at] = __float2half_rn(v);
  else ((__nv_bfloat16*)p)[at] = __float2bfloat16_rn(v);
}
ACTNN_DEV void rn_store_eight(void* p, int dtype, size_t row, int c, int C, const float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + 2 * i < C) rn_store_any(p, dtype, row + c + 2 * i, v[i].x);
    if (c + 2 * i + 1 < C) rn_store_any(p, dtype, row + c + 2 * i + 1, v[i].y);
  }
}

// N sums (4 or 8) over the lanes of a warp: halves of the sums are exchanged with halves of the lanes, so that 4 take 6 shuffles and
// 8 take 9.  Returned is the sum whose number the lane's upper bits are.
template <int N> ACTNN_DEV float rn_warp_sums(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int o = 16;
#pragma unroll
  for (int n = N / 2; n >= 1; n /= 2, o /= 2) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = upper ? v[i] : v[n + i], keep = upper ? v[n + i] : v[i];
      v[i] = keep + __shfl_xor_sync(kFull, give, o);
    }
  }
  float s = v[0];
#pragma unroll
  for (; o >= 1; o /= 2) s += __shfl_xor_sync(kFull, s, o);
  return s;
}

// After a wait that ran out, when all blocks have sent what they send: until the phase under way at each of the two barriers is over, or a
// limit outlasts the sums on their way here.  (Of the two parities that of the phase before is over at once.)
ACTNN_DEV void rn_outlast(const uint64_t* bars) {
  for (int i = 0; i < 4; ++i) mbar_wait(smem_addr(&bars[i >> 1]), i & 1);
}

// A run of rows by a block, or by a cluster of blocks of 4096 channels each.  A thread has eight channels of every row and keeps the sums of
// their parameters' gradients; the next row's values are requested as soon as this row's are unpacked.  The warps' sums of a row go to
// shared memory in two places in turn, so that one barrier a row is enough, and each warp joins them for itself.  The blocks of a
// cluster send theirs to one another, counted as they arrive by a barrier in memory: a barrier of the cluster would wait for
// the results of the row before to reach the L2 as well.  A warp whose wait runs out is counted, writes NaN for that row and those behind it,
// and sends nothing more, so that the other warps' waits for the next row run out too: had it gone on, its later sums would be
// counted and read as those of rows that others have not done with.
//
// Fewer instructions: the gate g and w1 enter as their product, and what
// depends on the rows of one gate alone is summed once: with S = sum m t n1 and S' = sum m t, dw1 = g S, db1 = g S', dg = w1 S + b1 S'.
// These products, in shared memory as float32, are a thread's own: g w1, g b1 and w2, and dw1 and db1 over the gates.
// (With gate, w1 and each gradient's sums apart: 8192 x 4096 116 us where 102 are taken now, 16384 x 8192 500 (355).  The second half of a row's
// work done after the next row's first half, past the barrier: 138 us, what it holds in registers and copies costs more.)
template <typename T, bool VEC, bool CODED, bool LAYER>
__global__ void __launch_bounds__(kRnMostThreads, 1) rn_backward_kernel(const __grid_constant__ RnArgs a, unsigned* gave_up) {
  constexpr int N = LAYER ? 8 : 4, kWarps = kRnMostThreads / 32;
  enum { kW2, kDw1, kGw, kGb, kDb1 };
  extern __shared__ float4 parameters_s[];
  __shared__ __align__(16) float part_s[2][kRnMostCluster * kWarps][N];
  __shared__ uint64_t there_s[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, threads = blockDim.x, warps = threads >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(smem_addr(&there_s[i]), 1);
    mbar_init_fence();
  }
  const uint32_t rank = a.cluster > 1 ? cluster_rank() : 0, run = blockIdx.x / a.cluster;
  const int c = ((int)rank * threads + (int)threadIdx.x) * 8, C = a.C, entries = a.cluster * warps;
  uint32_t first, end;
  if (a.units_of_run) {
    const uint32_t unit = run * a.units_of_run;
    first = unit * a.unit_rows;
    end = min(a.units, unit + a.units_of_run) * a.unit_rows;
  } else {
    const uint32_t u = run / a.runs_of_unit, k = run - u * a.runs_of_unit;
    first = u * a.unit_rows + (uint32_t)((uint64_t)k * a.unit_rows / a.runs_of_unit);
    end = u * a.unit_rows + (uint32_t)((uint64_t)(k + 1) * a.unit_rows / a.runs_of_unit);
  }
  // Behind C they are zero: with w2 and the gate's products so, nothing there enters a sum.
  auto put = [&](int set, float2 (&v)[4]) {
    if (c + 8 > C) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = make_float2(c + 2 * i < C ? v[i].x : 0.f, c + 2 * i + 1 < C ? v[i].y : 0.f);
    }
    rn_put(parameters_s + 2 * set * threads + threadIdx.x, threads, v);
  };
  auto get = [&](int set, float2 (&v)[4]) { rn_get(parameters_s + 2 * set * threads + threadIdx.x, threads, v); };
  float2 none[4] = {}, w2[4];
  rn_parameter<VEC>(a.w2, c, C, 1.f, w2);
  put(kW2, w2);
  put(kDw1, none);
  if (LAYER) put(kDb1, none);
  if (a.cluster > 1) cluster_sync();                    // the others' barriers are there
  NoiseKey key;
  if (a.dropped) key = drop_key(a.drop);
  float2 dw2[4] = {}, sum[4] = {}, db2[4] = {}, sum_b[4] = {};
  RnRaw<T, CODED> raw;
  float4 next_st = make_float4(0.f, 0.f, 0.f, 0.f);
  if (first < end) {
    rn_load_raw<T, CODED, VEC>(raw, a, first, c);
    next_st = rn_ld(a.stats + first);
  }
  uint32_t gate = fast_div(first, a.by_gate), gate_left = (gate + 1) * a.by_gate.d - first;        // rows that the gate still has
  bool ok = true, other = true;                         // other: the next row has another gate
  // dw1, db1 and what the gate's gradient is, of the rows of a gate that are over.
  auto turn = [&](uint32_t row) {
    const uint32_t g = fast_div(row, a.by_gate);
    float2 q[4], v[4], d[4];
    rn_parameter<VEC>(rn_gate_row(a, row), c, C, 1.f, q);
    get(kDw1, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = f_fma(q[i], sum[i], d[i]);
    put(kDw1, d);
    if (LAYER) {
      get(kDb1, d);
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = f_fma(q[i], sum_b[i], d[i]);
      put(kDb1, d);
    }
    if (a.dgate) {
      rn_parameter<VEC>(a.w1, c, C, 1.f, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = f_mul(v[i], sum[i]);
      if (LAYER) {
        rn_parameter<VEC>(a.b1, c, C, 0.f, d);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = f_fma(d[i], sum_b[i], v[i]);
      }
      if (a.units_of_run) rn_store_eight(a.dgate, a.gdtype, (size_t)g * C, c, C, v);
      else rn_store_eight(a.parts, ACTNN_F32, ((size_t)run * a.slots + a.slot_gate) * C, c, C, v);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = sum_b[i] = make_float2(0.f, 0.f);
  };
  uint32_t phase = 0;
  for (int place = 0; first < end; ++first, place ^= 1) {
    if (other) {
      float2 q[4], w[4];
      rn_parameter<VEC>(rn_gate_row(a, first), c, C, 1.f, q);
      rn_parameter<VEC>(a.w1, c, C, 1.f, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = f_mul(w[i], q[i]);
      put(kGw, w);
      if (LAYER) {
        rn_parameter<VEC>(a.b1, c, C, 0.f, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = f_mul(w[i], q[i]);
        put(kGb, w);
      }
    }
    other = --gate_left == 0;
    if (other) gate_left = a.by_gate.d;
    const float4 st = next_st;
    float2 n1[4], n2[4], cc[4], m[4];                   // m: the dropout's factors
    {
      float2 dh[4], p[4];
      rn_inputs<T, CODED, LAYER>(raw, a, st, n2, n1);
      unpack_vec(raw.dr, cc);
      unpack_vec(raw.dh, dh);
      if (first + 1 < end) {
        rn_load_raw<T, CODED, VEC>(raw, a, first + 1, c);
        next_st = rn_ld(a.stats + first + 1);
      }
      if (a.dropped) drop_factors(rn_fields<VEC>(a, key, first, c), a.drop.least, a.drop.inv, m);
      const float2 p2 = make_float2(st.w, st.w);
      if constexpr (LAYER) {
        get(kGb, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (a.dropped) p[i] = f_mul(p[i], m[i]);
          n2[i] = f_fma(p[i], p2, n2[i]);
        }
      }
      float2 s0{}, s1{}, s2{}, s3{}, s4{}, s5{}, s6{}, s7{};
      get(kGw, p);
      get(kW2, w2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (a.dropped) p[i] = f_mul(p[i], m[i]);
        const float2 gn = f_mul(p[i], n1[i]);
        n2[i] = f_fma(gn, p2, n2[i]);
        const float2 dn2 = f_mul(dh[i], w2[i]);
        cc[i] = f_fma(p2, dn2, cc[i]);
        dw2[i] = f_fma(dh[i], n2[i], dw2[i]);
        if (LAYER) db2[i] = f_add(db2[i], dh[i]);
        s0 = f_fma(dn2, n2[i], s0);
        s1 = f_fma(gn, cc[i], s1);
        s2 = f_fma(gn, n2[i], s2);
        if (LAYER) s3 = f_add(s3, dn2), s4 = f_add(s4, gn), s5 = f_fma(p[i], cc[i], s5), s6 = f_add(s6, p[i]), s7 = f_fma(p[i], n2[i], s7);
      }
      float v[N];
      v[0] = f_sum(s0), v[1] = f_sum(s1), v[2] = f_sum(s2), v[3] = f_sum(s3);
      if constexpr (LAYER) v[4] = f_sum(s4), v[5] = f_sum(s5), v[6] = f_sum(s6), v[7] = f_sum(s7);
      const float mine = rn_warp_sums<N>(v);
      if (a.cluster > 1) {                              // all have read the place's sums of two rows ago: they have sent those of the last one since
        const uint32_t bar = smem_addr(&there_s[place]), at = smem_addr(part_s[place][rank * warps + warp]);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __shfl_sync(kFull, mine, i * (32 / N));
        if (ok && threadIdx.x == 0) mbar_expect_tx(bar, entries * N * (int)sizeof(float));
        if (ok && lane < a.cluster) {
#pragma unroll
          for (int i = 0; i < N; i += 4) peer_send4(at + 4 * i, bar, lane, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
        }
        if (ok) {
          ok = __all_sync(kFull, mbar_wait(bar, phase >> place & 1));
          if (!ok && lane == 0) atomicAdd(gave_up, 1u);
        }
        phase ^= 1u << place;
      } else {
        if (lane % (32 / N) == 0) part_s[place][warp][lane / (32 / N)] = mine;
        if (warps > 1) __syncthreads();
        else __syncwarp();
      }
    }
    float total[N];
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 q = lane < entries ? *reinterpret_cast<const float4*>(&part_s[place][lane][i]) : make_float4(0.f, 0.f, 0.f, 0.f);
      total[i] = q.x, total[i + 1] = q.y, total[i + 2] = q.z, total[i + 3] = q.w;
    }
    for (int e = lane + 32; e < entries; e += 32) {
#pragma unroll
      for (int i = 0; i < N; ++i) total[i] += part_s[place][e][i];
    }
    float joined = rn_warp_sums<N>(total);
    if (!ok) joined = __int_as_float(0x7fffffff);
#pragma unroll
    for (int i = 0; i < N; ++i) total[i] = __shfl_sync(kFull, joined, i * (32 / N)) * a.inv_c;
    float M = 0.f, mean1 = 0.f;                         // p2 mean dn2; p1 times the mean of dn1
    const float m2 = st.w * total[0];                   // p2 mean(dn2 n2)
    float dot1 = total[1] - m2 * total[2];              // mean(dn1 n1)
    if constexpr (LAYER) {
      M = st.w * total[3];
      dot1 -= M * total[4];
      mean1 = (total[5] - M * total[6] - m2 * total[7]) * st.y;
    }
    dot1 *= st.y;
    float2 p[4], dx[4];
    get(kGw, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 t = f_fma(n2[i], make_float2(-m2, -m2), cc[i]);
      if (LAYER) t = f_add(t, make_float2(-M, -M));
      dx[i] = f_mul(t, make_float2(a.scale, a.scale));
      if (a.dropped) t = f_mul(t, m[i]);                // what passes the dropout
      sum[i] = f_fma(t, n1[i], sum[i]);
      if (LAYER) sum_b[i] = f_add(sum_b[i], t);
      t = f_mul(t, p[i]);
      if (a.post) {
        n1[i] = LAYER ? f_fma(n1[i], make_float2(-dot1, -dot1), make_float2(-mean1, -mean1)) : f_mul(n1[i], make_float2(-dot1, -dot1));
        t = f_fma(t, make_float2(st.y, st.y), n1[i]);
      }
      n1[i] = t;
    }
    if (a.dx) rn_store<T, VEC>((T*)a.dx + (size_t)first * C, c, C, dx);
    if (a.df) rn_store<T, VEC>((T*)a.df + (size_t)first * C, c, C, n1);
    if (other || first + 1 == end) turn(first);
  }
  if (a.cluster > 1) cluster_sync();                    // nobody leaves while sums are on their way to it
  if (!ok) rn_outlast(there_s);
  auto leave = [&](const float2 (&v)[4], int slot) {
    if (slot >= 0) rn_store_eight(a.parts, ACTNN_F32, ((size_t)run * a.slots + slot) * C, c, C, v);
  };
  leave(dw2, a.slot_w2);
  get(kDw1, w2);
  leave(w2, a.slot_w1);
  if (LAYER) {
    leave(db2, a.slot_b2);
    get(kDb1, w2);
    leave(w2, a.slot_b1);
  }
}

// The partial sums of the runs, added in order: a block has 32 columns of one sum, 32 threads a column.
template <typename T>
__global__ void __launch_bounds__(1024) rn_join_kernel(const __grid_constant__ RnArgs a) {
  constexpr int kWays = 32;
  __shared__ float part_s[kWays][32];
  const uint32_t blocks = (a.C + 31) / 32, which = blockIdx.x / blocks;
  const int way = threadIdx.x >> 5, column = (blockIdx.x - which * blocks) * 32 + (threadIdx.x & 31);
  // slots in their order, the gate's last, which has a sum for each unit
  const bool gate = a.slot_gate >= 0 && which >= (uint32_t)a.slot_gate;
  const uint32_t slot = gate ? a.slot_gate : which, unit = which - slot;
  const uint32_t first = gate ? unit * a.runs_of_unit : 0, count = gate ? a.runs_of_unit : a.runs;
  float s = 0.f;
  if (column < a.C) {
#pragma unroll 4
    for (uint32_t k = way; k < count; k += kWays) s += rn_ld(a.parts + ((size_t)(first + k) * a.slots + slot) * a.C + column);
  }
  part_s[way][threadIdx.x & 31] = s;
  __syncthreads();
  if (way == 0 && column < a.C) {
#pragma unroll
    for (int w = 1; w < kWays; ++w) s += part_s[w][threadIdx.x];
    void* to = gate ? a.dgate : (int)slot == a.slot_w2 ? a.dw2 : (int)slot == a.slot_b2 ? a.db2 : (int)slot == a.slot_w1 ? a.dw1 : a.db1;
    rn_store_any(to, gate ? a.gdtype : a.pdtype, (size_t)unit * a.C + column, s);
  }
}

// ------------------------------------------------------------------ host
// A warp has rows of up to 256 channels, a block longer ones; as few vectors a thread as 512 threads need.  As many blocks as are resident.
template <typename T, bool VEC, bool LAYER> int rn_forward(const RnArgs& a) {
  auto run = [&](auto kernel, bool warp, int V) {
    const int threads = warp ? kRnThreads : (a.C + V * 256 - 1) / (V * 256) * 32;
    const int smem = V <= 2 ? rn_sets<LAYER>() * 2 * V * threads * (int)sizeof(float4) : 0;
    const int64_t wanted = warp ? ((int64_t)a.rows + kRnThreads / 32 - 1) / (kRnThreads / 32) : a.rows;
    const int64_t resident = (int64_t)device_info().sm_count * rn_blocks_per_sm((const void*)kernel, threads, smem);
    kernel<<<(unsigned)std::min(wanted, resident), threads, smem, a.stream>>>(a);
    return check_launch();
  };
  if (a.C <= 256) return run(rn_forward_kernel<T, 1, true, VEC, LAYER>, true, 1);
  if (a.C <= 4096) return run(rn_forward_kernel<T, 1, false, VEC, LAYER>, false, 1);
  if (a.C <= 8192) return run(rn_forward_kernel<T, 2, false, VEC, LAYER>, false, 2);
  if (a.C <= 16384) return run(rn_forward_kernel<T, 4, false, VEC, LAYER>, false, 4);
  return run(rn_forward_kernel<T, 8, false, VEC, LAYER>, false, 8);
}
template <typename T, bool VEC, bool CODED, bool LAYER> int rn_backward(const RnArgs& a) {
  auto* kernel = rn_backward_kernel<T, VEC, CODED, LAYER>;
  unsigned* gave_up = bulk_wait_counter();
  if (!gave_up) return ACTNN_ERR_LAUNCH;
  const int threads = a.cluster > 1 ? kRnMostThreads : (a.C + 255) / 256 * 32;
  const int smem = (LAYER ? 5 : 3) * 2 * threads * (int)sizeof(float4);
  rn_blocks_per_sm((const void*)kernel, threads, smem);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.runs * a.cluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = a.stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, a, gave_up) != cudaSuccess) return cudaGetLastError(), ACTNN_ERR_LAUNCH;
  if (int st = check_launch()) return st;
  if (a.slots == 0) return ACTNN_OK;
  const int sums = a.slot_gate >= 0 ? a.slots - 1 + (int)a.units : a.slots;
  rn_join_kernel<T><<<(unsigned)((a.C + 31) / 32 * sums), 1024, 0, a.stream>>>(a);
  return check_launch();
}
template <typename T, bool VEC> int rn_run_typed(const RnArgs& a, RnWhat what) {
  if (what == kRnForward) return a.layer ? rn_forward<T, VEC, true>(a) : rn_forward<T, VEC, false>(a);
  if (a.coded) return a.layer ? rn_backward<T, VEC, true, true>(a) : rn_backward<T, VEC, true, false>(a);
  return a.layer ? rn_backward<T, VEC, false, true>(a) : rn_backward<T, VEC, false, false>(a);
}
template <typename T> int rn_run(const RnArgs& a, RnWhat what, bool vec) {
  return vec ? rn_run_typed<T, true>(a, what) : rn_run_typed<T, false>(a, what);
}
#endif

}  // namespace actnn
