// Group norm with an activation on channels-last activations [N, S, C], S positions of C channels, G groups of C / G channels.
//
//   forward   mean, var over the S * C / G elements of a (sample, group);  z = (x - mean) * rstd * gamma + beta;  y = f(z)
//             codes: (x - mid) in 127 steps either way of half the group's range, mid the middle of the range
//   backward  x^ = mid + code * step,  h = (x^ - mean) * rstd,  dz = dy * f'(h * gamma + beta)
//             dgamma = sum dz * h,  dbeta = sum dz   (over samples and positions)
//             dx = rstd * (dz * gamma - A - h * B),  A, B = means over the group of dz * gamma and dz * gamma * h
//
// Two passes over the data each way, because every output needs a sum over its group: the first leaves partial results of
// `chunks` runs of positions, the second joins those it needs before it starts (in a fixed order: results are reproducible) and
// writes.  A thread keeps V consecutive channels and walks down the positions, so everything that belongs to a channel or group
// stays in registers, folded into as few constants as the formulas leave: z = za * code + zb and dx = k1 * dz + k2 * code + k3
// take three a channel and two a group (one set of these for the thread where V divides a group's channels).  What a thread
// will read next is on its way to a ring of its own in shared memory (cp.async), so that neither registers nor barriers limit
// how many bytes are under way.
//
// The range, and with it the codes, follow from exact minima and maxima by single fp32 operations: reproducible to the bit.
// The variance is joined from sums about a value of each thread's own (its first one), which loses nothing to cancellation
// however far the mean is from zero: the sum of squares about one of n values exceeds the one about their mean n-fold at most.
#pragma once

#include "activation.cuh"

namespace actnn {

// How the channels are cut: `tiles` runs of `tile` channels, at most kGnThreads vectors each.  A run holds whole groups, or is a
// part of one (`parts` of them a group).
struct GnShape {
  int64_t S;
  int C, G, cpg;                        // channels, groups, channels of a group
  int V;                                // channels of a thread: 8, 4, 2 or 1, a divisor of C
  int tile, tiles, parts;
  int chunks;                           // runs of positions, `rows` each but the last
  int64_t rows;
  float eps;
};
struct GnCall {
  const void *x, *dy;
  const float *gamma, *beta;
  void* out;
  int8_t* codes;
  float *stats, *dgamma, *dbeta;
  void* workspace;
  int64_t N;
  int kind;
  cudaStream_t stream;
};
// One partial result of the statistics.
struct Part { float mean, m2, lo, hi; };

// group_norm.cu, group_norm_f16.cu, group_norm_bf16.cu
int gn_run_f32(const GnCall& c, const GnShape& g, bool forward);
int gn_run_f16(const GnCall& c, const GnShape& g, bool forward);
int gn_run_bf16(const GnCall& c, const GnShape& g, bool forward);

namespace {

constexpr int kGnThreads = 256;
template <typename T> constexpr int kGnResident = sizeof(T) == 2 ? 3 : 2;      // blocks of an SM that the registers have to allow
constexpr int kGnDepth = 4;                     // positions of a ring

ACTNN_DEV int tile_first(const GnShape& g, int t) {
  return g.parts == 1 ? t * g.tile : t / g.parts * g.cpg + t % g.parts * g.tile;
}
ACTNN_DEV int tile_end(const GnShape& g, int t) {
  return g.parts == 1 ? min(g.C, (t + 1) * g.tile) : min((t / g.parts + 1) * g.cpg, tile_first(g, t) + g.tile);
}
// The block's place: sample, run of positions, run of channels.
struct BlockAt { int64_t n; int chunk, tile; };
ACTNN_DEV BlockAt block_at(const GnShape& g) {
  const uint32_t k = blockIdx.x / (uint32_t)g.tiles, n = k / (uint32_t)g.chunks;
  return BlockAt{(int64_t)n, (int)(k - n * (uint32_t)g.chunks), (int)(blockIdx.x - k * (uint32_t)g.tiles)};
}

// 16-byte places in front of the rings that hold a value for each group of the tile.
ACTNN_HD int gn_table(const GnShape& g) { return g.parts == 1 ? g.tile / g.cpg : 1; }

// Minimum and maximum that let a NaN through.
ACTNN_DEV float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
ACTNN_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Over the L lanes (a power of two) that share a group; every lane of the warp takes part.
ACTNN_DEV float lanes_sum(float v, int L) {
  for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
ACTNN_DEV float lanes_min(float v, int L) {
  for (int o = L >> 1; o > 0; o >>= 1) v = min_nan(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
ACTNN_DEV float lanes_max(float v, int L) {
  for (int o = L >> 1; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
ACTNN_DEV int lanes_for(int entries) { return entries >= 32 ? 32 : entries <= 1 ? 1 : 1 << (32 - __clz(entries - 1)); }

constexpr float kInf = __builtin_huge_valf();

// The next positions of a thread: A bytes each of one array and B of another (0: none), kGnDepth - 1 positions ahead.  Sizes that the
// asynchronous copy does not know (below 4 bytes) are loaded when they are needed.
template <int BYTES> ACTNN_DEV void copy_async(uint32_t dst, const char* src) {
  if constexpr (BYTES == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(dst), "l"(src) : "memory");
  else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" :: "r"(dst), "l"(src) : "memory");
  else
#pragma unroll
    for (int i = 0; i < BYTES; i += 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst + i), "l"(src + i) : "memory");
}
template <int BYTES> ACTNN_DEV void from_shared(uint32_t src, uint32_t* w) {
  if constexpr (BYTES == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(src) : "memory");
  else if constexpr (BYTES == 8) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(src) : "memory");
  else
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                   : "r"(src + 16 * i) : "memory");
}
template <int A, int B> struct Ring {
  static constexpr bool kAsync = A >= 4 && (B == 0 || B >= 4);
  static constexpr int kBytes = kAsync ? kGnDepth * kGnThreads * (A + B) : 0;
};
// Calls take(words of a, words of b) for `count` positions, `step` bytes apart in each array.
template <int A, int B, typename Take>
ACTNN_DEV void through_ring(uint32_t ring, const char* a, const char* b, int64_t step_a, int64_t step_b, int count, Take take) {
  const uint32_t ra = ring + threadIdx.x * A, rb = ring + kGnDepth * kGnThreads * A + threadIdx.x * B;
  auto ask = [&](int place, bool wanted) {
    if (wanted) {
      copy_async<A>(ra + place * (kGnThreads * A), a);
      a += step_a;
      if constexpr (B > 0) {
        copy_async<B>(rb + place * (kGnThreads * B), b);
        b += step_b;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kGnDepth - 1; ++i) ask(i, i < count);
  for (int base = 0; base < count; base += kGnDepth) {
#pragma unroll
    for (int s = 0; s < kGnDepth; ++s) {
      if (base + s < count) {
        asm volatile("cp.async.wait_group %0;" :: "n"(kGnDepth - 2) : "memory");
        uint32_t wa[A / 4], wb[B > 0 ? B / 4 : 1];
        from_shared<A>(ra + s * (kGnThreads * A), wa);
        if constexpr (B > 0) from_shared<B>(rb + s * (kGnThreads * B), wb);
        ask((s + kGnDepth - 1) % kGnDepth, base + s + kGnDepth - 1 < count);      // the place the position before has left
        take(wa, wb);
      }
    }
  }
}

// A constant for each channel of a thread.
template <int V> struct Row {
  typename Many<V>::F f[Many<V>::N];
  ACTNN_DEV void set(int i, float v) {
    if constexpr (V == 1) f[0] = v;
    else if (i & 1) f[i / 2].y = v;
    else f[i / 2].x = v;
  }
  ACTNN_DEV float get(int i) const {
    if constexpr (V == 1) return f[0];
    else return i & 1 ? f[i / 2].y : f[i / 2].x;
  }
};
// A constant of the group of each channel of a thread: one where all are of one group (ONE).
template <int V, bool ONE> struct GroupRow {
  using F = typename Many<V>::F;
  Row<V> r;
  F one;
  ACTNN_DEV void set(int i, float v) {
    if constexpr (ONE) one = f_both<F>(v);
    else r.set(i, v);
  }
  ACTNN_DEV F at(int i) const { return ONE ? one : r.f[i]; }       // of pair i
  ACTNN_DEV float get(int i) const {                               // of channel i
    if constexpr (!ONE) return r.get(i);
    else if constexpr (V == 1) return one;
    else return one.x;
  }
};

// Minimum and maximum of V channels over positions, NaNs let through: M = 1 over all, M = V for each channel.  Pairs of a
// 16-bit type are compared as they are.
ACTNN_DEV uint32_t min2_nan(uint32_t a, uint32_t b, __half) {
  uint32_t r;
  asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
ACTNN_DEV uint32_t max2_nan(uint32_t a, uint32_t b, __half) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
ACTNN_DEV uint32_t min2_nan(uint32_t a, uint32_t b, __nv_bfloat16) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
ACTNN_DEV uint32_t max2_nan(uint32_t a, uint32_t b, __nv_bfloat16) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T, int V, int M> struct Extremes {
  static constexpr bool kPairs = sizeof(T) == 2 && V > 1;
  static constexpr int N = kPairs ? (M == 1 ? 1 : V / 2) : M;
  uint32_t lo[N], hi[N];
  ACTNN_DEV Extremes() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kPairs) {
        lo[i] = pair_from_float(make_float2(kInf, kInf), T());
        hi[i] = lo[i] | 0x80008000u;
      } else {
        lo[i] = __float_as_uint(kInf);
        hi[i] = __float_as_uint(-kInf);
      }
    }
  }
  ACTNN_DEV void take(const Vec<T, V>& v, const typename Many<V>::F (&f)[Many<V>::N]) {
    if constexpr (kPairs) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        lo[M == 1 ? 0 : i] = min2_nan(lo[M == 1 ? 0 : i], v.w[i], T());
        hi[M == 1 ? 0 : i] = max2_nan(hi[M == 1 ? 0 : i], v.w[i], T());
      }
    } else {
      int i = 0;
#pragma unroll
      for (int k = 0; k < Many<V>::N; ++k)
        f_each(f[k], [&](float e) {
          const int at = M == 1 ? 0 : i++;
          lo[at] = __float_as_uint(min_nan(__uint_as_float(lo[at]), e));
          hi[at] = __float_as_uint(max_nan(__uint_as_float(hi[at]), e));
          return e;
        });
    }
  }
  ACTNN_DEV float2 get(int i) const {                   // of channel i; of all with M = 1
    if constexpr (kPairs) {
      const float2 l = pair_to_float(lo[M == 1 ? 0 : i / 2], T()), h = pair_to_float(hi[M == 1 ? 0 : i / 2], T());
      if constexpr (M == 1) return make_float2(min_nan(l.x, l.y), max_nan(h.x, h.y));
      else return i & 1 ? make_float2(l.y, h.y) : make_float2(l.x, h.x);
    } else {
      return make_float2(__uint_as_float(lo[i]), __uint_as_float(hi[i]));
    }
  }
};

// ------------------------------------------------------------------ statistics
// A block per sample, run of positions and run of channels.  ONE: V divides cpg, a thread has one value of each kind, else one a
// channel.  out[((n * G + group) * chunks + chunk) * parts + part].
template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_stats_kernel(const T* __restrict__ x, Part* __restrict__ out, const GnShape g) {
  using F = typename Many<V>::F;
  constexpr int N = Many<V>::N, M = ONE ? 1 : V;               // values of a thread
  extern __shared__ float4 dynamic_s[];
  __shared__ float4 part_s[kGnThreads * M];
  const BlockAt at = block_at(g);
  const int c0 = tile_first(g, at.tile), width = tile_end(g, at.tile) - c0;
  const int vecs = width / V, R = blockDim.x / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  const int64_t first = at.chunk * g.rows, end = min(g.S, first + g.rows);
  const int64_t step = (int64_t)R * g.C;
  if (r < R) {
    const int count = first + r < end ? (int)((end - first - r + R - 1) / R) : 0;
    if (count > 0) {
      const T* p = x + (at.n * g.S + first + r) * g.C + c0 + v * V;
      Row<V> shift;                                            // less it
      F s2[N], q2[N];
      Extremes<T, V, M> ex;
#pragma unroll
      for (int i = 0; i < V; ++i) shift.set(i, -to_float(p[ONE ? 0 : i]));
#pragma unroll
      for (int i = 0; i < N; ++i) s2[i] = q2[i] = f_both<F>(0.f);
      auto take = [&](const Vec<T, V>& w) {
        F f[N];
        unpack_vec(w, f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int to = ONE ? 0 : i;
          const F d = f_add(f[i], shift.f[ONE ? 0 : i]);
          s2[to] = f_add(s2[to], d);
          q2[to] = f_fma(d, d, q2[to]);
        }
        ex.take(w, f);
      };
      if constexpr (V > 1 && Ring<V * sizeof(T), 0>::kAsync) {
        through_ring<V * sizeof(T), 0>(smem_addr(dynamic_s), (const char*)p, nullptr, step * sizeof(T), 0, count,
                                       [&](const uint32_t* wa, const uint32_t*) {
                                         Vec<T, V> w;
#pragma unroll
                                         for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) w.w[i] = wa[i];
                                         take(w);
                                       });
      } else {
#pragma unroll 8
        for (int k = 0; k < count; ++k) take(load_vec<T, V>(p + k * step));
      }
      const float items = (float)(count * (V / M));
#pragma unroll
      for (int i = 0; i < M; ++i) {
        float s, q;
        if constexpr (ONE) s = f_sum(s2[0]), q = f_sum(q2[0]);
        else if constexpr (V == 1) s = s2[0], q = q2[0];
        else s = i & 1 ? s2[i / 2].y : s2[i / 2].x, q = i & 1 ? q2[i / 2].y : q2[i / 2].x;
        const float2 e = ex.get(i);
        part_s[(r * vecs + v) * M + i] = make_float4(fmaf(items, -shift.get(i), s), q - s * (s / items), e.x, e.y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < M; ++i) part_s[(r * vecs + v) * M + i] = make_float4(0.f, 0.f, kInf, -kInf);
    }
  }
  __syncthreads();
  // Lanes that share a group of the tile: its sum, then the squares about its mean.
  const int cells = vecs * M, groups = g.parts == 1 ? width / g.cpg : 1, cpg = cells / groups, entries = R * cpg, L = lanes_for(entries);
  const int member = threadIdx.x & (L - 1), per = blockDim.x / L;
  for (int j0 = 0; j0 < groups; j0 += per) {
    const int j = j0 + threadIdx.x / L;
    float sum = 0.f, lo = kInf, hi = -kInf, m2 = 0.f;
    const bool in = j < groups;
    for (int e = member; in && e < entries; e += L) {
      const int er = e / cpg;
      const float4 q = part_s[er * cells + j * cpg + (e - er * cpg)];
      sum += q.x;
      lo = min_nan(lo, q.z);
      hi = max_nan(hi, q.w);
    }
    sum = lanes_sum(sum, L);
    const float mean = sum / ((float)(end - first) * (float)(cpg * (V / M)));
    for (int e = member; in && e < entries; e += L) {
      const int er = e / cpg;
      const float4 q = part_s[er * cells + j * cpg + (e - er * cpg)];
      if (first + er < end) {
        const float items = (float)((end - first - er + R - 1) / R * (V / M)), d = q.x / items - mean;
        m2 += fmaf(items * d, d, q.y);
      }
    }
    m2 = lanes_sum(m2, L);
    lo = lanes_min(lo, L);
    hi = lanes_max(hi, L);
    if (in && member == 0) {
      const int group = c0 / g.cpg + j, part = g.parts == 1 ? 0 : at.tile % g.parts;
      out[((at.n * g.G + group) * g.chunks + at.chunk) * g.parts + part] = Part{mean, m2, lo, hi};
    }
  }
}

// Joins the partial results of one (sample, group) over L lanes; every one of them gets mean, rstd, mid and half of the range.
ACTNN_DEV float4 join_stats(const Part* __restrict__ p, bool in, const GnShape& g, int member, int L) {
  const int count = in ? g.chunks * g.parts : 0;
  auto items = [&](int i) {
    const int chunk = i / g.parts, part = i - chunk * g.parts;
    return (float)(min(g.S, (chunk + 1) * g.rows) - chunk * g.rows) *
           (float)(g.parts == 1 ? g.cpg : min(g.cpg, (part + 1) * g.tile) - part * g.tile);
  };
  float sum = 0.f, lo = kInf, hi = -kInf, m2 = 0.f;
  for (int i = member; i < count; i += L) {
    const Part q = p[i];
    sum = fmaf(items(i), q.mean, sum);
    lo = min_nan(lo, q.lo);
    hi = max_nan(hi, q.hi);
  }
  const float m = (float)g.S * (float)g.cpg;
  const float mean = lanes_sum(sum, L) / m;
  for (int i = member; i < count; i += L) {
    const Part q = p[i];
    const float d = q.mean - mean;
    m2 += fmaf(items(i) * d, d, q.m2);
  }
  const float var = lanes_sum(m2, L) / m;
  lo = lanes_min(lo, L);
  hi = lanes_max(hi, L);
  const float mid = __fadd_rn(__fmul_rn(0.5f, hi), __fmul_rn(0.5f, lo));
  float half = __fsub_rn(__fmul_rn(0.5f, hi), __fmul_rn(0.5f, lo));
  half = half < kTiny ? kTiny : half;                                      // a NaN stays one
  return make_float4(mean, 1.f / sqrtf(var + g.eps), mid, half);
}

// ------------------------------------------------------------------ output and codes
template <typename T, int V, bool ONE, int KIND, bool SAVE>
ACTNN_DEV void gn_apply(uint32_t ring, const T* __restrict__ p, T* __restrict__ y, int8_t* __restrict__ codes, int count, int64_t step,
                        const Row<V>& a, const Row<V>& b, const GroupRow<V, ONE>& mid, const GroupRow<V, ONE>& inv) {
  using F = typename Many<V>::F;
  constexpr bool P = sizeof(T) == 4;
  constexpr int N = Many<V>::N;
  auto put = [&](const Vec<T, V>& w) {
    F f[N], o[N];
    unpack_vec(w, f);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = act_value<KIND, P>(f_fma(f[i], a.f[i], b.f[i]));
    store_vec<T, V>(y, o);
    y += step;
    if constexpr (SAVE) {
      F c[N];
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] = code_bits(f_add(f[i], mid.at(i)), inv.at(i));
      store_codes<V>(codes, c);
      codes += step;
    }
  };
  if constexpr (V > 1 && Ring<V * sizeof(T), 0>::kAsync) {
    through_ring<V * sizeof(T), 0>(ring, (const char*)p, nullptr, step * sizeof(T), 0, count, [&](const uint32_t* wa, const uint32_t*) {
      Vec<T, V> w;
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) w.w[i] = wa[i];
      put(w);
    });
  } else {
#pragma unroll 4
    for (int k = 0; k < count; ++k) put(load_vec<T, V>(p + k * step));
  }
}

// stats[(n * G + group) * 4], unless NULL: kept for the backward pass.
template <typename T, int V, bool ONE, bool SAVE>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_forward_kernel(const T* __restrict__ x, const Part* __restrict__ parts, const float* __restrict__ gamma,
                  const float* __restrict__ beta, T* __restrict__ y, int8_t* __restrict__ codes, float* __restrict__ stats,
                  int kind, const GnShape g) {
  extern __shared__ float4 group_s[];                     // a group each, then the rings
  const BlockAt at = block_at(g);
  const int c0 = tile_first(g, at.tile), width = tile_end(g, at.tile) - c0;
  const int g0 = c0 / g.cpg, groups = g.parts == 1 ? width / g.cpg : 1;
  const int L = lanes_for(g.chunks * g.parts), per = blockDim.x / L, member = threadIdx.x & (L - 1);
  for (int j0 = 0; j0 < groups; j0 += per) {
    const int j = j0 + threadIdx.x / L;
    const bool in = j < groups && threadIdx.x < per * L;
    const float4 st = join_stats(parts + (at.n * g.G + g0 + (in ? j : 0)) * g.chunks * g.parts, in, g, member, L);
    if (in && member == 0) {
      group_s[j] = st;
      if (stats && at.chunk == 0 && (g.parts == 1 || at.tile % g.parts == 0))
        reinterpret_cast<float4*>(stats)[at.n * g.G + g0 + j] = st;
    }
  }
  __syncthreads();
  const int vecs = width / V, R = blockDim.x / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  const int64_t first = at.chunk * g.rows, end = min(g.S, first + g.rows);
  if (r >= R || first + r >= end) return;
  const int c = c0 + v * V;
  Row<V> a, b;
  GroupRow<V, ONE> mid, inv;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float4 st = group_s[(ONE ? c : c + i) / g.cpg - g0];
    mid.set(i, -st.z);
    inv.set(i, code_factor(st.w));
    const float w = st.y * (gamma ? __ldg(gamma + c + i) : 1.f);
    a.set(i, w);
    b.set(i, (beta ? __ldg(beta + c + i) : 0.f) - st.x * w);
  }
  const uint32_t ring = smem_addr(group_s + gn_table(g));
  const int64_t off = (at.n * g.S + first + r) * g.C + c, step = (int64_t)R * g.C;
  const int count = (int)((end - first - r + R - 1) / R);
  const T* p = x + off;
  T* q = y + off;
  int8_t* cd = SAVE ? codes + off : nullptr;
  switch (kind) {
    case kActNone: gn_apply<T, V, ONE, kActNone, SAVE>(ring, p, q, cd, count, step, a, b, mid, inv); break;
    case kActRelu: gn_apply<T, V, ONE, kActRelu, SAVE>(ring, p, q, cd, count, step, a, b, mid, inv); break;
    case kActSilu: gn_apply<T, V, ONE, kActSilu, SAVE>(ring, p, q, cd, count, step, a, b, mid, inv); break;
    case kActGelu: gn_apply<T, V, ONE, kActGelu, SAVE>(ring, p, q, cd, count, step, a, b, mid, inv); break;
    default: gn_apply<T, V, ONE, kActGeluTanh, SAVE>(ring, p, q, cd, count, step, a, b, mid, inv); break;
  }
}

// ------------------------------------------------------------------ backward
// What is kept of a position's V channels: codes, or the elements less the mean.  h = line.x * kept + line.y.
template <typename T, int V, bool CODES> struct Kept {
  static constexpr int kBytes = V * sizeof(T);
  using Words = Vec<T, V>;
  static ACTNN_DEV const char* from(const T* x, const int8_t*, int64_t at) { return (const char*)(x + at); }
  static ACTNN_DEV Words load(const char* p) { return load_vec<T, V>((const T*)p); }
  template <bool ONE>
  static ACTNN_DEV void get(const Words& w, typename Many<V>::F (&f)[Many<V>::N], const GroupRow<V, ONE>& mean) {
    unpack_vec(w, f);
#pragma unroll
    for (int i = 0; i < Many<V>::N; ++i) f[i] = f_add(f[i], mean.at(i));
  }
  static ACTNN_DEV float2 line(const float4& st) { return make_float2(st.y, 0.f); }
};
template <typename T, int V> struct Kept<T, V, true> {
  static constexpr int kBytes = V;
  using Words = Codes<V>;
  static ACTNN_DEV const char* from(const T*, const int8_t* codes, int64_t at) { return (const char*)(codes + at); }
  static ACTNN_DEV Words load(const char* p) { return load_codes<V>((const int8_t*)p); }
  template <bool ONE>
  static ACTNN_DEV void get(const Words& w, typename Many<V>::F (&f)[Many<V>::N], const GroupRow<V, ONE>&) { unpack_codes<V>(w, f); }
  static ACTNN_DEV float2 line(const float4& st) { return make_float2(code_step(st.w) * st.y, (st.z - st.x) * st.y); }
};
// The gradient and what is kept, position by position.
template <typename T, int V, bool CODES, typename Take>
ACTNN_DEV void gn_positions(uint32_t ring, const T* dy, const T* x, const int8_t* codes, int64_t at, int count, int64_t step, Take take) {
  using K = Kept<T, V, CODES>;
  constexpr int A = V * sizeof(T), B = K::kBytes;
  const char *a = (const char*)(dy + at), *b = K::from(x, codes, at);
  const int64_t step_a = step * (int64_t)sizeof(T), step_b = step * (B / V);
  if constexpr (V > 1 && Ring<A, B>::kAsync) {
    through_ring<A, B>(ring, a, b, step_a, step_b, count, [&](const uint32_t* wa, const uint32_t* wb) {
      Vec<T, V> w;
      typename K::Words k;
#pragma unroll
      for (int i = 0; i < A / 4; ++i) w.w[i] = wa[i];
#pragma unroll
      for (int i = 0; i < B / 4; ++i) k.w[i] = wb[i];
      take(w, k);
    });
  } else {
#pragma unroll 4
    for (int k = 0; k < count; ++k) {
      const typename K::Words w = K::load(b + k * step_b);
      take(load_vec<T, V>((const T*)(a + k * step_a)), w);
    }
  }
}

template <typename T, int V, bool ONE, int KIND, bool CODES>
ACTNN_DEV void gn_sums(uint32_t ring, const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes, int64_t at,
                       int count, int64_t step, const GroupRow<V, ONE>& mean, const Row<V>& za, const Row<V>& zb, Row<V>& s1, Row<V>& s2) {
  using F = typename Many<V>::F;
  using K = Kept<T, V, CODES>;
  constexpr bool P = sizeof(T) == 4;
  constexpr int N = Many<V>::N;
  gn_positions<T, V, CODES>(ring, dy, x, codes, at, count, step, [&](const Vec<T, V>& w, const typename K::Words& k) {
    F d[N], f[N];
    unpack_vec(w, d);
    K::get(k, f, mean);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const F dz = f_mul(d[i], act_slope<KIND, P>(f_fma(f[i], za.f[i], zb.f[i])));
      s1.f[i] = f_add(s1.f[i], dz);
      s2.f[i] = f_fma(dz, f[i], s2.f[i]);
    }
  });
}

// sums[(n * chunks + chunk) * C + c]: of dz and of dz * h over the chunk's positions.
template <typename T, int V, bool ONE, bool CODES>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_backward_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                        const float* __restrict__ stats, const float* __restrict__ gamma, const float* __restrict__ beta,
                        float2* __restrict__ sums, int kind, const GnShape g) {
  extern __shared__ float4 dynamic_s[];
  __shared__ float2 part_s[kGnThreads * V];
  const BlockAt at = block_at(g);
  const int c0 = tile_first(g, at.tile), width = tile_end(g, at.tile) - c0;
  const int vecs = width / V, R = blockDim.x / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  if (r < R) {
    const int c = c0 + v * V;
    Row<V> za, zb, s1, s2;
    GroupRow<V, ONE> mean;
    GroupRow<V, ONE> lx, ly;
    float2 l;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i == 0 || !ONE) {
        const float4 st = __ldg(reinterpret_cast<const float4*>(stats) + at.n * g.G + (c + i) / g.cpg);
        l = Kept<T, V, CODES>::line(st);
        mean.set(i, -st.x);
        lx.set(i, l.x);
        ly.set(i, l.y);
      }
      const float w = gamma ? __ldg(gamma + c + i) : 1.f;
      za.set(i, w * l.x);
      zb.set(i, fmaf(w, l.y, beta ? __ldg(beta + c + i) : 0.f));
      s1.set(i, 0.f);
      s2.set(i, 0.f);
    }
    const int64_t first = at.chunk * g.rows, end = min(g.S, first + g.rows), off = (at.n * g.S + first + r) * g.C + c;
    const int count = first + r < end ? (int)((end - first - r + R - 1) / R) : 0;
    const int64_t step = (int64_t)R * g.C;
    const uint32_t ring = smem_addr(dynamic_s);
    switch (kind) {
      case kActNone: gn_sums<T, V, ONE, kActNone, CODES>(ring, dy, x, codes, off, count, step, mean, za, zb, s1, s2); break;
      case kActRelu: gn_sums<T, V, ONE, kActRelu, CODES>(ring, dy, x, codes, off, count, step, mean, za, zb, s1, s2); break;
      case kActSilu: gn_sums<T, V, ONE, kActSilu, CODES>(ring, dy, x, codes, off, count, step, mean, za, zb, s1, s2); break;
      case kActGelu: gn_sums<T, V, ONE, kActGelu, CODES>(ring, dy, x, codes, off, count, step, mean, za, zb, s1, s2); break;
      default: gn_sums<T, V, ONE, kActGeluTanh, CODES>(ring, dy, x, codes, off, count, step, mean, za, zb, s1, s2); break;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
      part_s[r * width + v * V + i] = make_float2(s1.get(i), fmaf(lx.get(i), s2.get(i), ly.get(i) * s1.get(i)));
  }
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    float2 s = make_float2(0.f, 0.f);
    for (int k = 0; k < R; ++k) {
      s.x += part_s[k * width + c].x;
      s.y += part_s[k * width + c].y;
    }
    sums[(at.n * g.chunks + at.chunk) * g.C + c0 + c] = s;
  }
}

template <typename T, int V, bool ONE, int KIND, bool CODES>
ACTNN_DEV void gn_grad(uint32_t ring, const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                       T* __restrict__ dx, int64_t at, int count, int64_t step, const GroupRow<V, ONE>& mean, const Row<V>& za,
                       const Row<V>& zb, const Row<V>& k1, const GroupRow<V, ONE>& k2, const GroupRow<V, ONE>& k3) {
  using F = typename Many<V>::F;
  using K = Kept<T, V, CODES>;
  constexpr bool P = sizeof(T) == 4;
  constexpr int N = Many<V>::N;
  T* to = dx + at;
  gn_positions<T, V, CODES>(ring, dy, x, codes, at, count, step, [&](const Vec<T, V>& w, const typename K::Words& k) {
    F d[N], f[N];
    unpack_vec(w, d);
    K::get(k, f, mean);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const F dz = f_mul(d[i], act_slope<KIND, P>(f_fma(f[i], za.f[i], zb.f[i])));
      d[i] = f_fma(dz, k1.f[i], f_fma(f[i], k2.at(i), k3.at(i)));
    }
    store_vec<T, V>(to, d);
    to += step;
  });
}

template <typename T, int V, bool ONE, bool CODES>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_backward_kernel(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                   const float* __restrict__ stats, const float* __restrict__ gamma, const float* __restrict__ beta,
                   const float2* __restrict__ sums, T* __restrict__ dx, int kind, const GnShape g) {
  extern __shared__ float4 dynamic_s[];                   // a group each, then the rings
  float2* means_s = reinterpret_cast<float2*>(dynamic_s);
  const BlockAt at = block_at(g);
  const int c0 = tile_first(g, at.tile), width = tile_end(g, at.tile) - c0;
  const int g0 = c0 / g.cpg, groups = g.parts == 1 ? width / g.cpg : 1, entries = g.chunks * g.cpg;
  const int L = lanes_for(entries), per = blockDim.x / L, member = threadIdx.x & (L - 1);
  for (int j0 = 0; j0 < groups; j0 += per) {
    const int j = j0 + threadIdx.x / L;
    const bool in = j < groups && threadIdx.x < per * L;
    float a = 0.f, b = 0.f;
    for (int e = member; in && e < entries; e += L) {
      const int k = e / g.cpg, c = (g0 + j) * g.cpg + (e - k * g.cpg);
      const float2 s = sums[(at.n * g.chunks + k) * g.C + c];
      const float w = gamma ? __ldg(gamma + c) : 1.f;
      a = fmaf(w, s.x, a);
      b = fmaf(w, s.y, b);
    }
    const float m = (float)g.S * (float)g.cpg;
    a = lanes_sum(a, L) / m;
    b = lanes_sum(b, L) / m;
    if (in && member == 0) means_s[j] = make_float2(a, b);
  }
  __syncthreads();
  const int vecs = width / V, R = blockDim.x / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  const int64_t first = at.chunk * g.rows, end = min(g.S, first + g.rows);
  if (r >= R || first + r >= end) return;
  const int c = c0 + v * V;
  Row<V> za, zb, k1;
  GroupRow<V, ONE> mean, k2, k3;
  float4 st;
  float2 l;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i == 0 || !ONE) {
      st = __ldg(reinterpret_cast<const float4*>(stats) + at.n * g.G + (c + i) / g.cpg);
      l = Kept<T, V, CODES>::line(st);
      const float2 m = means_s[(c + i) / g.cpg - g0];
      mean.set(i, -st.x);
      k2.set(i, -st.y * m.y * l.x);
      k3.set(i, -st.y * fmaf(m.y, l.y, m.x));
    }
    const float w = gamma ? __ldg(gamma + c + i) : 1.f;
    za.set(i, w * l.x);
    zb.set(i, fmaf(w, l.y, beta ? __ldg(beta + c + i) : 0.f));
    k1.set(i, st.y * w);
  }
  const uint32_t ring = smem_addr(dynamic_s + gn_table(g));
  const int64_t off = (at.n * g.S + first + r) * g.C + c, step = (int64_t)R * g.C;
  const int count = (int)((end - first - r + R - 1) / R);
  switch (kind) {
    case kActNone: gn_grad<T, V, ONE, kActNone, CODES>(ring, dy, x, codes, dx, off, count, step, mean, za, zb, k1, k2, k3); break;
    case kActRelu: gn_grad<T, V, ONE, kActRelu, CODES>(ring, dy, x, codes, dx, off, count, step, mean, za, zb, k1, k2, k3); break;
    case kActSilu: gn_grad<T, V, ONE, kActSilu, CODES>(ring, dy, x, codes, dx, off, count, step, mean, za, zb, k1, k2, k3); break;
    case kActGelu: gn_grad<T, V, ONE, kActGelu, CODES>(ring, dy, x, codes, dx, off, count, step, mean, za, zb, k1, k2, k3); break;
    default: gn_grad<T, V, ONE, kActGeluTanh, CODES>(ring, dy, x, codes, dx, off, count, step, mean, za, zb, k1, k2, k3); break;
  }
}

// dgamma and dbeta: column sums of the [rows, C] partial sums.  A block takes 8 columns, its 128 threads of each runs of rows.
__global__ void __launch_bounds__(1024)
gn_column_sums_kernel(const float2* __restrict__ sums, float* __restrict__ dgamma, float* __restrict__ dbeta, int64_t rows, int C) {
  __shared__ float2 part_s[32][8];
  const int col = threadIdx.x & 7, run = threadIdx.x >> 3, c = blockIdx.x * 8 + col;
  float2 s = make_float2(0.f, 0.f);
  if (c < C) {
#pragma unroll 8
    for (int64_t k = run; k < rows; k += 128) s = f_add(s, __ldg(sums + k * C + c));
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) s = f_add(s, make_float2(__shfl_xor_sync(kFull, s.x, o), __shfl_xor_sync(kFull, s.y, o)));
  if ((threadIdx.x & 31) < 8) part_s[threadIdx.x >> 5][col] = s;
  __syncthreads();
  if (threadIdx.x < 8 && c < C) {
    s = make_float2(0.f, 0.f);
    for (int k = 0; k < 32; ++k) s = f_add(s, part_s[k][col]);
    if (dbeta) dbeta[c] = s.x;
    if (dgamma) dgamma[c] = s.y;
  }
}

// ------------------------------------------------------------------ launches
inline int gn_threads(const GnShape& g) {
  const int vecs = g.tile / g.V, R = kGnThreads / vecs;
  return (vecs * R + 31) / 32 * 32;
}
inline unsigned gn_grid(const GnCall& c, const GnShape& g) { return (unsigned)(c.N * g.chunks * g.tiles); }

// A launch with `bytes` of dynamic shared memory; the limit is raised once for a kernel and device (cached with its occupancy).
template <typename Kernel, typename... Args>
void gn_start(Kernel kernel, const GnCall& c, const GnShape& g, int table, int ring, Args... args) {
  constexpr int kMostTable = kGnThreads * 8 * 16;
  cached_blocks_per_sm((const void*)kernel, kGnThreads, kMostTable + ring);
  kernel<<<gn_grid(c, g), gn_threads(g), table * 16 + ring, c.stream>>>(args...);
}

template <typename T, int V, bool ONE> int gn_forward(const GnCall& c, const GnShape& g) {
  constexpr int kRing = Ring<V * sizeof(T), 0>::kBytes;
  Part* parts = (Part*)c.workspace;
  gn_start(gn_stats_kernel<T, V, ONE>, c, g, 0, kRing, (const T*)c.x, parts, g);
  gn_start(c.codes ? gn_forward_kernel<T, V, ONE, true> : gn_forward_kernel<T, V, ONE, false>, c, g, gn_table(g), kRing, (const T*)c.x,
           (const Part*)parts, c.gamma, c.beta, (T*)c.out, c.codes, c.stats, c.kind, g);
  return check_launch();
}
template <typename T, int V, bool ONE, bool CODES> int gn_backward(const GnCall& c, const GnShape& g) {
  constexpr int kRing = Ring<V * sizeof(T), Kept<T, V, CODES>::kBytes>::kBytes;
  float2* sums = (float2*)c.workspace;
  gn_start(gn_backward_sums_kernel<T, V, ONE, CODES>, c, g, 0, kRing, (const T*)c.dy, (const T*)c.x, (const int8_t*)c.codes,
           (const float*)c.stats, c.gamma, c.beta, sums, c.kind, g);
  gn_start(gn_backward_kernel<T, V, ONE, CODES>, c, g, gn_table(g), kRing, (const T*)c.dy, (const T*)c.x, (const int8_t*)c.codes,
           (const float*)c.stats, c.gamma, c.beta, (const float2*)sums, (T*)c.out, c.kind, g);
  if (c.dgamma || c.dbeta)
    gn_column_sums_kernel<<<(g.C + 7) / 8, 1024, 0, c.stream>>>(sums, c.dgamma, c.dbeta, c.N * g.chunks, g.C);
  return check_launch();
}
template <typename T, int V, bool ONE> int gn_one(const GnCall& c, const GnShape& g, bool forward) {
  return forward ? gn_forward<T, V, ONE>(c, g) : c.codes ? gn_backward<T, V, ONE, true>(c, g) : gn_backward<T, V, ONE, false>(c, g);
}
template <typename T> int gn_run(const GnCall& c, const GnShape& g, bool forward) {
  const bool one = g.cpg % g.V == 0;
  switch (g.V) {
    case 8: return one ? gn_one<T, 8, true>(c, g, forward) : gn_one<T, 8, false>(c, g, forward);
    case 4: return one ? gn_one<T, 4, true>(c, g, forward) : gn_one<T, 4, false>(c, g, forward);
    case 2: return one ? gn_one<T, 2, true>(c, g, forward) : gn_one<T, 2, false>(c, g, forward);
    default: return gn_one<T, 1, true>(c, g, forward);
  }
}

}  // namespace
}  // namespace actnn
