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
// writes.  A thread keeps V consecutive channels of one group and walks down the positions, so everything that belongs to a
// channel or group stays in registers, folded into as few constants as the formulas leave: z = za * code + zb and
// dx = k1 * dz + k2 * code + k3 take three a channel and two a group.  Rows are requested kGnAhead at a time.
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
  int V;                                // channels of a thread: 8, 4, 2 or 1, a divisor of cpg
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
int gn_forward_f32(const GnCall& c, const GnShape& g);
int gn_forward_f16(const GnCall& c, const GnShape& g);
int gn_forward_bf16(const GnCall& c, const GnShape& g);
int gn_backward_f32(const GnCall& c, const GnShape& g);
int gn_backward_f16(const GnCall& c, const GnShape& g);
int gn_backward_bf16(const GnCall& c, const GnShape& g);

namespace {

constexpr int kGnThreads = 256;
constexpr int kGnAheadStats = 4, kGnAhead = 2;

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

// Minimum and maximum of vectors.  Pairs of a 16-bit type are compared as they are.
template <typename T, int V> struct Extremes {
  float lo = kInf, hi = -kInf;
  ACTNN_DEV void take(const Vec<T, V>&, const typename Many<V>::F (&f)[Many<V>::N]) {
#pragma unroll
    for (int i = 0; i < Many<V>::N; ++i)
      f_each(f[i], [&](float v) {
        lo = min_nan(lo, v);
        hi = max_nan(hi, v);
        return v;
      });
  }
  ACTNN_DEV float lowest() const { return lo; }
  ACTNN_DEV float highest() const { return hi; }
};
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
template <typename T, int V> struct Extremes16 {
  uint32_t lo, hi;                                   // infinities: 0x7c00 in float16, 0x7f80 in bfloat16
  ACTNN_DEV Extremes16() {
    lo = pair_from_float(make_float2(kInf, kInf), T());
    hi = lo | 0x80008000u;
  }
  ACTNN_DEV void take(const Vec<T, V>& w, const float2 (&)[Many<V>::N]) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      lo = min2_nan(lo, w.w[i], T());
      hi = max2_nan(hi, w.w[i], T());
    }
  }
  ACTNN_DEV float lowest() const {
    const float2 p = pair_to_float(lo, T());
    return min_nan(p.x, p.y);
  }
  ACTNN_DEV float highest() const {
    const float2 p = pair_to_float(hi, T());
    return max_nan(p.x, p.y);
  }
};

template <int V> struct Extremes<__half, V> : Extremes16<__half, V> {};
template <int V> struct Extremes<__nv_bfloat16, V> : Extremes16<__nv_bfloat16, V> {};
template <> struct Extremes<__half, 1> : Extremes<float, 1> {
  ACTNN_DEV void take(const Vec<__half, 1>&, const float (&f)[1]) { Extremes<float, 1>::take(Vec<float, 1>(), f); }
};
template <> struct Extremes<__nv_bfloat16, 1> : Extremes<float, 1> {
  ACTNN_DEV void take(const Vec<__nv_bfloat16, 1>&, const float (&f)[1]) { Extremes<float, 1>::take(Vec<float, 1>(), f); }
};

// ------------------------------------------------------------------ statistics
// A block per sample, run of positions and run of channels.  out[((n * G + group) * chunks + chunk) * parts + part].
template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads)
gn_stats_kernel(const T* __restrict__ x, Part* __restrict__ out, const GnShape g) {
  using F = typename Many<V>::F;
  __shared__ float4 part_s[kGnThreads];
  const BlockAt at = block_at(g);
  const int c0 = tile_first(g, at.tile), width = tile_end(g, at.tile) - c0;
  const int vecs = width / V, R = blockDim.x / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  const int64_t first = at.chunk * g.rows, end = min(g.S, first + g.rows);
  const int64_t step = (int64_t)R * g.C;
  if (r < R) {
    float4 mine = make_float4(0.f, 0.f, kInf, -kInf);
    if (first + r < end) {
      int64_t count = (end - first - r + R - 1) / R;
      const float items = (float)(count * V);
      const T* p = x + (at.n * g.S + first + r) * g.C + c0 + v * V;
      const float shift = to_float(p[0]);
      F s2 = f_both<F>(0.f), q2 = f_both<F>(0.f);
      const F off = f_both<F>(-shift);
      Extremes<T, V> ex;
      auto take = [&](const Vec<T, V>& w) {
        F f[Many<V>::N];
        unpack_vec(w, f);
#pragma unroll
        for (int i = 0; i < Many<V>::N; ++i) {
          const F d = f_add(f[i], off);
          s2 = f_add(s2, d);
          q2 = f_fma(d, d, q2);
        }
        ex.take(w, f);
      };
      for (; count >= kGnAheadStats; count -= kGnAheadStats) {
        Vec<T, V> w[kGnAheadStats];
#pragma unroll
        for (int i = 0; i < kGnAheadStats; ++i, p += step) w[i] = load_vec<T, V>(p);
#pragma unroll
        for (int i = 0; i < kGnAheadStats; ++i) take(w[i]);
      }
      for (; count > 0; --count, p += step) take(load_vec<T, V>(p));
      const float s = f_sum(s2), q = f_sum(q2);
      mine = make_float4(fmaf(items, shift, s), q - s * (s / items), ex.lowest(), ex.highest());
    }
    part_s[threadIdx.x] = mine;
  }
  __syncthreads();
  // Lanes that share a group of the tile: its sum, then the squares about its mean.
  const int groups = g.parts == 1 ? width / g.cpg : 1, vpg = vecs / groups, entries = R * vpg, L = lanes_for(entries);
  const int member = threadIdx.x & (L - 1), per = blockDim.x / L;
  for (int j0 = 0; j0 < groups; j0 += per) {
    const int j = j0 + threadIdx.x / L;
    float sum = 0.f, lo = kInf, hi = -kInf, m2 = 0.f;
    const bool in = j < groups && threadIdx.x < per * L;
    for (int e = member; in && e < entries; e += L) {
      const int er = e / vpg;
      const float4 q = part_s[er * vecs + j * vpg + (e - er * vpg)];
      sum += q.x;
      lo = min_nan(lo, q.z);
      hi = max_nan(hi, q.w);
    }
    sum = lanes_sum(sum, L);
    const float mean = sum / ((float)(end - first) * (float)(vpg * V));
    for (int e = member; in && e < entries; e += L) {
      const int er = e / vpg;
      const float4 q = part_s[er * vecs + j * vpg + (e - er * vpg)];
      if (first + er < end) {
        const float items = (float)((end - first - er + R - 1) / R * V), d = q.x / items - mean;
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

// ------------------------------------------------------------------ output and codes
template <typename T, int V, int KIND, bool SAVE>
ACTNN_DEV void gn_apply(const T* __restrict__ p, T* __restrict__ y, int8_t* __restrict__ codes, int64_t count, int64_t step,
                        const Row<V>& a, const Row<V>& b, float mid, float inv) {
  using F = typename Many<V>::F;
  constexpr bool P = sizeof(T) == 4;
  constexpr int N = Many<V>::N;
  const F off = f_both<F>(-mid), factor = f_both<F>(inv);
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
      for (int i = 0; i < N; ++i) c[i] = code_bits(f_add(f[i], off), factor);
      store_codes<V>(codes, c);
      codes += step;
    }
  };
  for (; count >= kGnAhead; count -= kGnAhead) {
    Vec<T, V> w[kGnAhead];
#pragma unroll
    for (int i = 0; i < kGnAhead; ++i, p += step) w[i] = load_vec<T, V>(p);
#pragma unroll
    for (int i = 0; i < kGnAhead; ++i) put(w[i]);
  }
  for (; count > 0; --count, p += step) put(load_vec<T, V>(p));
}

// stats[(n * G + group) * 4], unless NULL: kept for the backward pass.
template <typename T, int V, bool SAVE>
__global__ void __launch_bounds__(kGnThreads)
gn_forward_kernel(const T* __restrict__ x, const Part* __restrict__ parts, const float* __restrict__ gamma,
                  const float* __restrict__ beta, T* __restrict__ y, int8_t* __restrict__ codes, float* __restrict__ stats,
                  int kind, const GnShape g) {
  extern __shared__ float4 group_s[];                     // a group each
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
  const float4 st = group_s[c / g.cpg - g0];
  Row<V> a, b;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float w = st.y * (gamma ? __ldg(gamma + c + i) : 1.f);
    a.set(i, w);
    b.set(i, (beta ? __ldg(beta + c + i) : 0.f) - st.x * w);
  }
  const float mid = st.z, inv = code_factor(st.w);
  const int64_t off = (at.n * g.S + first + r) * g.C + c, count = (end - first - r + R - 1) / R, step = (int64_t)R * g.C;
  const T* p = x + off;
  T* q = y + off;
  int8_t* cd = SAVE ? codes + off : nullptr;
  switch (kind) {
    case kActNone: gn_apply<T, V, kActNone, SAVE>(p, q, cd, count, step, a, b, mid, inv); break;
    case kActRelu: gn_apply<T, V, kActRelu, SAVE>(p, q, cd, count, step, a, b, mid, inv); break;
    case kActSilu: gn_apply<T, V, kActSilu, SAVE>(p, q, cd, count, step, a, b, mid, inv); break;
    case kActGelu: gn_apply<T, V, kActGelu, SAVE>(p, q, cd, count, step, a, b, mid, inv); break;
    default: gn_apply<T, V, kActGeluTanh, SAVE>(p, q, cd, count, step, a, b, mid, inv); break;
  }
}

// ------------------------------------------------------------------ backward
// What is kept of a position's V channels: codes, or the elements less the mean.  h = line.x * kept + line.y.
template <typename T, int V, bool CODES> struct Kept {
  Vec<T, V> w;
  ACTNN_DEV void load(const T* x, const int8_t*, int64_t at) { w = load_vec<T, V>(x + at); }
  ACTNN_DEV void get(typename Many<V>::F (&f)[Many<V>::N], float mean) const {
    unpack_vec(w, f);
#pragma unroll
    for (int i = 0; i < Many<V>::N; ++i) f[i] = f_add(f[i], f_both<typename Many<V>::F>(-mean));
  }
  static ACTNN_DEV float2 line(const float4& st) { return make_float2(st.y, 0.f); }
};
template <typename T, int V> struct Kept<T, V, true> {
  Codes<V> w;
  ACTNN_DEV void load(const T*, const int8_t* codes, int64_t at) { w = load_codes<V>(codes + at); }
  ACTNN_DEV void get(typename Many<V>::F (&f)[Many<V>::N], float) const { unpack_codes<V>(w, f); }
  static ACTNN_DEV float2 line(const float4& st) { return make_float2(code_step(st.w) * st.y, (st.z - st.x) * st.y); }
};

template <typename T, int V, int KIND, bool CODES>
ACTNN_DEV void gn_sums(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes, int64_t at, int64_t count,
                       int64_t step, float mean, const Row<V>& za, const Row<V>& zb, Row<V>& s1, Row<V>& s2) {
  using F = typename Many<V>::F;
  using K = Kept<T, V, CODES>;
  constexpr bool P = sizeof(T) == 4;
  constexpr int N = Many<V>::N;
  auto take = [&](const Vec<T, V>& w, const K& k) {
    F d[N], f[N];
    unpack_vec(w, d);
    k.get(f, mean);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const F dz = f_mul(d[i], act_slope<KIND, P>(f_fma(f[i], za.f[i], zb.f[i])));
      s1.f[i] = f_add(s1.f[i], dz);
      s2.f[i] = f_fma(dz, f[i], s2.f[i]);
    }
  };
  for (; count >= kGnAhead; count -= kGnAhead) {
    Vec<T, V> w[kGnAhead];
    K k[kGnAhead];
#pragma unroll
    for (int i = 0; i < kGnAhead; ++i, at += step) {
      w[i] = load_vec<T, V>(dy + at);
      k[i].load(x, codes, at);
    }
#pragma unroll
    for (int i = 0; i < kGnAhead; ++i) take(w[i], k[i]);
  }
  for (; count > 0; --count, at += step) {
    K k;
    k.load(x, codes, at);
    take(load_vec<T, V>(dy + at), k);
  }
}

// sums[(n * chunks + chunk) * C + c]: of dz and of dz * h over the chunk's positions.
template <typename T, int V, bool CODES>
__global__ void __launch_bounds__(kGnThreads)
gn_backward_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                        const float* __restrict__ stats, const float* __restrict__ gamma, const float* __restrict__ beta,
                        float2* __restrict__ sums, int kind, const GnShape g) {
  __shared__ float2 part_s[kGnThreads * V];
  const BlockAt at = block_at(g);
  const int c0 = tile_first(g, at.tile), width = tile_end(g, at.tile) - c0;
  const int vecs = width / V, R = blockDim.x / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  if (r < R) {
    const int c = c0 + v * V;
    const float4 st = __ldg(reinterpret_cast<const float4*>(stats) + at.n * g.G + c / g.cpg);
    const float2 l = Kept<T, V, CODES>::line(st);
    Row<V> za, zb, s1, s2;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float w = gamma ? __ldg(gamma + c + i) : 1.f;
      za.set(i, w * l.x);
      zb.set(i, fmaf(w, l.y, beta ? __ldg(beta + c + i) : 0.f));
      s1.set(i, 0.f);
      s2.set(i, 0.f);
    }
    const int64_t first = at.chunk * g.rows, end = min(g.S, first + g.rows), off = (at.n * g.S + first + r) * g.C + c;
    const int64_t count = first + r < end ? (end - first - r + R - 1) / R : 0, step = (int64_t)R * g.C;
    switch (kind) {
      case kActNone: gn_sums<T, V, kActNone, CODES>(dy, x, codes, off, count, step, st.x, za, zb, s1, s2); break;
      case kActRelu: gn_sums<T, V, kActRelu, CODES>(dy, x, codes, off, count, step, st.x, za, zb, s1, s2); break;
      case kActSilu: gn_sums<T, V, kActSilu, CODES>(dy, x, codes, off, count, step, st.x, za, zb, s1, s2); break;
      case kActGelu: gn_sums<T, V, kActGelu, CODES>(dy, x, codes, off, count, step, st.x, za, zb, s1, s2); break;
      default: gn_sums<T, V, kActGeluTanh, CODES>(dy, x, codes, off, count, step, st.x, za, zb, s1, s2); break;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) part_s[r * width + v * V + i] = make_float2(s1.get(i), fmaf(l.x, s2.get(i), l.y * s1.get(i)));
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

template <typename T, int V, int KIND, bool CODES>
ACTNN_DEV void gn_grad(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes, T* __restrict__ dx,
                       int64_t at, int64_t count, int64_t step, float mean, const Row<V>& za, const Row<V>& zb, const Row<V>& k1,
                       float k2, float k3) {
  using F = typename Many<V>::F;
  using K = Kept<T, V, CODES>;
  constexpr bool P = sizeof(T) == 4;
  constexpr int N = Many<V>::N;
  const F slope = f_both<F>(k2), level = f_both<F>(k3);
  int64_t to = at;
  auto put = [&](const Vec<T, V>& w, const K& k) {
    F d[N], f[N];
    unpack_vec(w, d);
    k.get(f, mean);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const F dz = f_mul(d[i], act_slope<KIND, P>(f_fma(f[i], za.f[i], zb.f[i])));
      d[i] = f_fma(dz, k1.f[i], f_fma(f[i], slope, level));
    }
    store_vec<T, V>(dx + to, d);
    to += step;
  };
  for (; count >= kGnAhead; count -= kGnAhead) {
    Vec<T, V> w[kGnAhead];
    K k[kGnAhead];
#pragma unroll
    for (int i = 0; i < kGnAhead; ++i, at += step) {
      w[i] = load_vec<T, V>(dy + at);
      k[i].load(x, codes, at);
    }
#pragma unroll
    for (int i = 0; i < kGnAhead; ++i) put(w[i], k[i]);
  }
  for (; count > 0; --count, at += step) {
    K k;
    k.load(x, codes, at);
    put(load_vec<T, V>(dy + at), k);
  }
}

template <typename T, int V, bool CODES>
__global__ void __launch_bounds__(kGnThreads)
gn_backward_kernel(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                   const float* __restrict__ stats, const float* __restrict__ gamma, const float* __restrict__ beta,
                   const float2* __restrict__ sums, T* __restrict__ dx, int kind, const GnShape g) {
  extern __shared__ float2 means_s[];                     // a group each
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
  const float4 st = __ldg(reinterpret_cast<const float4*>(stats) + at.n * g.G + c / g.cpg);
  const float2 l = Kept<T, V, CODES>::line(st), m = means_s[c / g.cpg - g0];
  Row<V> za, zb, k1;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float w = gamma ? __ldg(gamma + c + i) : 1.f;
    za.set(i, w * l.x);
    zb.set(i, fmaf(w, l.y, beta ? __ldg(beta + c + i) : 0.f));
    k1.set(i, st.y * w);
  }
  const float k2 = -st.y * m.y * l.x, k3 = -st.y * fmaf(m.y, l.y, m.x);
  const int64_t off = (at.n * g.S + first + r) * g.C + c, count = (end - first - r + R - 1) / R, step = (int64_t)R * g.C;
  switch (kind) {
    case kActNone: gn_grad<T, V, kActNone, CODES>(dy, x, codes, dx, off, count, step, st.x, za, zb, k1, k2, k3); break;
    case kActRelu: gn_grad<T, V, kActRelu, CODES>(dy, x, codes, dx, off, count, step, st.x, za, zb, k1, k2, k3); break;
    case kActSilu: gn_grad<T, V, kActSilu, CODES>(dy, x, codes, dx, off, count, step, st.x, za, zb, k1, k2, k3); break;
    case kActGelu: gn_grad<T, V, kActGelu, CODES>(dy, x, codes, dx, off, count, step, st.x, za, zb, k1, k2, k3); break;
    default: gn_grad<T, V, kActGeluTanh, CODES>(dy, x, codes, dx, off, count, step, st.x, za, zb, k1, k2, k3); break;
  }
}

// dgamma and dbeta: column sums of the [rows, C] partial sums.  A block takes 32 columns, its warps runs of rows.
__global__ void __launch_bounds__(1024)
gn_column_sums_kernel(const float2* __restrict__ sums, float* __restrict__ dgamma, float* __restrict__ dbeta, int64_t rows, int C) {
  __shared__ float2 part_s[32][32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float2 s = make_float2(0.f, 0.f);
  if (c < C) {
#pragma unroll 8
    for (int64_t k = wid; k < rows; k += 32) {
      const float2 v = sums[k * C + c];
      s.x += v.x;
      s.y += v.y;
    }
  }
  part_s[wid][lane] = s;
  __syncthreads();
  if (wid == 0 && c < C) {
    s = make_float2(0.f, 0.f);
    for (int k = 0; k < 32; ++k) {
      s.x += part_s[k][lane].x;
      s.y += part_s[k][lane].y;
    }
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

template <typename T, int V> int gn_forward(const GnCall& c, const GnShape& g) {
  Part* parts = (Part*)c.workspace;
  gn_stats_kernel<T, V><<<gn_grid(c, g), gn_threads(g), 0, c.stream>>>((const T*)c.x, parts, g);
  auto* second = c.codes ? gn_forward_kernel<T, V, true> : gn_forward_kernel<T, V, false>;
  const size_t smem = sizeof(float4) * (g.parts == 1 ? g.tile / g.cpg : 1);
  second<<<gn_grid(c, g), gn_threads(g), smem, c.stream>>>((const T*)c.x, parts, c.gamma, c.beta, (T*)c.out, c.codes, c.stats, c.kind, g);
  return check_launch();
}
template <typename T, int V> int gn_backward(const GnCall& c, const GnShape& g) {
  float2* sums = (float2*)c.workspace;
  auto* first = c.codes ? gn_backward_sums_kernel<T, V, true> : gn_backward_sums_kernel<T, V, false>;
  auto* second = c.codes ? gn_backward_kernel<T, V, true> : gn_backward_kernel<T, V, false>;
  first<<<gn_grid(c, g), gn_threads(g), 0, c.stream>>>((const T*)c.dy, (const T*)c.x, c.codes, c.stats, c.gamma, c.beta, sums, c.kind, g);
  const size_t smem = sizeof(float2) * (g.parts == 1 ? g.tile / g.cpg : 1);
  second<<<gn_grid(c, g), gn_threads(g), smem, c.stream>>>((const T*)c.dy, (const T*)c.x, c.codes, c.stats, c.gamma, c.beta, sums,
                                                          (T*)c.out, c.kind, g);
  if (c.dgamma || c.dbeta)
    gn_column_sums_kernel<<<(g.C + 31) / 32, 1024, 0, c.stream>>>(sums, c.dgamma, c.dbeta, c.N * g.chunks, g.C);
  return check_launch();
}
template <typename T> int gn_forward_of(const GnCall& c, const GnShape& g) {
  return g.V == 8 ? gn_forward<T, 8>(c, g) : g.V == 4 ? gn_forward<T, 4>(c, g) : g.V == 2 ? gn_forward<T, 2>(c, g) : gn_forward<T, 1>(c, g);
}
template <typename T> int gn_backward_of(const GnCall& c, const GnShape& g) {
  return g.V == 8 ? gn_backward<T, 8>(c, g) : g.V == 4 ? gn_backward<T, 4>(c, g) : g.V == 2 ? gn_backward<T, 2>(c, g) : gn_backward<T, 1>(c, g);
}

}  // namespace
}  // namespace actnn
