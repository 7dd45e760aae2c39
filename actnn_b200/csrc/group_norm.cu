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
// writes.  A thread keeps V consecutive channels and walks down the positions, so everything that belongs to a channel stays in
// registers.  Bound by HBM: forward 2 + 2 (read twice) + 2 + 1 bytes an element of a 16-bit type, backward 3 + 3 + 2, less what the
// second pass still finds in the L2.
//
// The range, and with it the codes, follow from exact minima and maxima by single fp32 operations: reproducible to the bit.
// The variance is joined from sums about a value of each thread's own (its first one), which loses nothing to cancellation
// however far the mean is from zero: the sum of squares about one of n values exceeds the one about their mean n-fold at most.
#include "activation.cuh"

namespace actnn {
namespace {

constexpr int kGnThreads = 256;

// How the channels are cut: `tiles` runs of `tile` channels, at most 256 vectors each.  A run holds whole groups, or is a part of
// one (`parts` of them a group).
struct GnShape {
  int64_t S;
  int C, G, cpg;                        // channels, groups, channels of a group
  int tile, tiles, parts;
  int chunks;                           // runs of positions, `rows` each but the last
  int64_t rows;
  float eps;
};
ACTNN_DEV int tile_first(const GnShape& g, int t) {
  return g.parts == 1 ? t * g.tile : t / g.parts * g.cpg + t % g.parts * g.tile;
}
ACTNN_DEV int tile_end(const GnShape& g, int t) {
  return g.parts == 1 ? min(g.C, (t + 1) * g.tile) : min((t / g.parts + 1) * g.cpg, tile_first(g, t) + g.tile);
}

// The block's place: sample, run of positions, run of channels.
struct BlockAt { int64_t n; int chunk, tile; };
ACTNN_DEV BlockAt block_at(int tiles, int chunks) {
  const uint32_t k = blockIdx.x / (uint32_t)tiles, n = k / (uint32_t)chunks;
  return BlockAt{(int64_t)n, (int)(k - n * (uint32_t)chunks), (int)(blockIdx.x - k * (uint32_t)tiles)};
}

// One partial result of the statistics: of `rows` x channels elements.
struct Part { float mean, m2, lo, hi; };

ACTNN_DEV float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
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
ACTNN_DEV float warp_min_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = min_nan(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
ACTNN_DEV float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// ------------------------------------------------------------------ statistics
// A block per sample, run of positions and run of channels.  parts_out[((n * G + group) * chunks + chunk) * parts + part].
template <typename T, int V>
__global__ void __launch_bounds__(kGnThreads)
gn_stats_kernel(const T* __restrict__ x, Part* __restrict__ parts_out, const GnShape g) {
  __shared__ float sum_s[kGnThreads * V], m2_s[kGnThreads * V], lo_s[kGnThreads * V], hi_s[kGnThreads * V];
  const BlockAt at_ = block_at(g.tiles, g.chunks);
  const int t = at_.tile, chunk = at_.chunk;
  const int64_t n = at_.n;
  const int c0 = tile_first(g, t), width = tile_end(g, t) - c0;
  const int vecs = width / V, R = kGnThreads / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  const int64_t first = chunk * g.rows, end = min(g.S, first + g.rows);
  const T* p = x + (n * g.S) * g.C + c0 + v * V;
  float shift[V], s[V], q[V], lo[V], hi[V];
  int64_t count = 0;
  if (r < R && first + r < end) {
    unpack_vec(load_vec<T, V>(p + (first + r) * g.C), shift);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = q[i] = 0.f, lo[i] = hi[i] = shift[i];
    count = (end - first - r + R - 1) / R;
#pragma unroll 4
    for (int64_t k = 1; k < count; ++k) {
      float f[V];
      unpack_vec(load_vec<T, V>(p + (first + r + k * R) * g.C), f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = f[i] - shift[i];
        s[i] += d;
        q[i] = fmaf(d, d, q[i]);
        lo[i] = min_nan(lo[i], f[i]);
        hi[i] = max_nan(hi[i], f[i]);
      }
    }
  }
  if (r < R) {
    const float cnt = (float)count;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = r * width + v * V + i;
      const bool any = count > 0;
      sum_s[e] = any ? fmaf(cnt, shift[i], s[i]) : 0.f;
      m2_s[e] = any ? q[i] - s[i] * (s[i] / cnt) : 0.f;
      lo_s[e] = any ? lo[i] : __int_as_float(0x7f800000);
      hi_s[e] = any ? hi[i] : __int_as_float(0xff800000);
    }
  }
  __syncthreads();
  // A warp per group of the tile: its sum, then the squares about its mean.
  const int lane = threadIdx.x & 31, groups = g.parts == 1 ? width / g.cpg : 1, gw = g.parts == 1 ? g.cpg : width;
  for (int j = threadIdx.x >> 5; j < groups; j += kGnThreads / 32) {
    float sum = 0.f, mn = __int_as_float(0x7f800000), mx = __int_as_float(0xff800000);
    for (int e = lane; e < R * gw; e += 32) {
      const int er = e / gw, at = er * width + j * gw + (e - er * gw);
      sum += sum_s[at];
      mn = min_nan(mn, lo_s[at]);
      mx = max_nan(mx, hi_s[at]);
    }
    sum = warp_sum(sum);
    const float mean = sum / ((float)(end - first) * (float)gw);
    float m2 = 0.f;
    for (int e = lane; e < R * gw; e += 32) {
      const int er = e / gw, at = er * width + j * gw + (e - er * gw);
      const int64_t c = (end - first - er + R - 1) / R;
      if (first + er < end) {
        const float d = sum_s[at] / (float)c - mean;
        m2 += fmaf((float)c * d, d, m2_s[at]);
      }
    }
    m2 = warp_sum(m2);
    mn = warp_min_nan(mn);
    mx = warp_max_nan(mx);
    if (lane == 0) {
      const int group = c0 / g.cpg + j, part = g.parts == 1 ? 0 : t % g.parts;
      parts_out[((n * g.G + group) * g.chunks + chunk) * g.parts + part] = Part{mean, m2, mn, mx};
    }
  }
}

// Joins the partial results of one (sample, group); every lane gets mean, rstd, mid and half of the range.
ACTNN_DEV float4 join_stats(const Part* __restrict__ parts, int64_t n, int group, const GnShape& g, int lane) {
  const Part* p = parts + (n * g.G + group) * g.chunks * g.parts;
  const int count = g.chunks * g.parts;
  float sum = 0.f, mn = __int_as_float(0x7f800000), mx = __int_as_float(0xff800000);
  for (int i = lane; i < count; i += 32) {
    const int chunk = i / g.parts, part = i - chunk * g.parts;
    const float c = (float)(min(g.S, (chunk + 1) * g.rows) - chunk * g.rows) *
                    (float)(g.parts == 1 ? g.cpg : min(g.cpg, (part + 1) * g.tile) - part * g.tile);
    const Part q = p[i];
    sum = fmaf(c, q.mean, sum);
    mn = min_nan(mn, q.lo);
    mx = max_nan(mx, q.hi);
  }
  const float m = (float)g.S * (float)g.cpg;
  const float mean = warp_sum(sum) / m;
  float m2 = 0.f;
  for (int i = lane; i < count; i += 32) {
    const int chunk = i / g.parts, part = i - chunk * g.parts;
    const float c = (float)(min(g.S, (chunk + 1) * g.rows) - chunk * g.rows) *
                    (float)(g.parts == 1 ? g.cpg : min(g.cpg, (part + 1) * g.tile) - part * g.tile);
    const Part q = p[i];
    const float d = q.mean - mean;
    m2 += fmaf(c * d, d, q.m2);
  }
  const float var = warp_sum(m2) / m;
  mn = warp_min_nan(mn);
  mx = warp_max_nan(mx);
  const float mid = __fadd_rn(__fmul_rn(0.5f, mx), __fmul_rn(0.5f, mn));
  float half = __fsub_rn(__fmul_rn(0.5f, mx), __fmul_rn(0.5f, mn));
  half = half < kTiny ? kTiny : half;                                      // a NaN stays one
  return make_float4(mean, 1.f / sqrtf(var + g.eps), mid, half);
}

// ------------------------------------------------------------------ output and codes
template <typename T, int V, int KIND, bool SAVE>
ACTNN_DEV void gn_apply(const T* __restrict__ p, T* __restrict__ y, int8_t* __restrict__ codes, int64_t C, int64_t first, int64_t end,
                        int64_t step, const float (&a)[V], const float (&b)[V], const float (&mid)[V], const float (&inv)[V]) {
  constexpr bool P = sizeof(T) == 4;
#pragma unroll 2
  for (int64_t k = first; k < end; k += step) {
    float f[V], o[V];
    unpack_vec(load_vec<T, V>(p + k * C), f);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = act_value<KIND, P>(fmaf(f[i], a[i], b[i]));
    store_vec<T, V>(y + k * C, o);
    if constexpr (SAVE) {
      uint32_t c[V];
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = code_bits(__fsub_rn(f[i], mid[i]), inv[i]);
      store_codes<V>(codes + k * C, c);
    }
  }
}

// A block per sample, run of positions and run of channels, the chunks of this pass.  stats[(n * G + group) * 4]: kept for the backward pass.
template <typename T, int V, bool SAVE>
__global__ void __launch_bounds__(kGnThreads)
gn_forward_kernel(const T* __restrict__ x, const Part* __restrict__ parts, const float* __restrict__ gamma,
                  const float* __restrict__ beta, T* __restrict__ y, int8_t* __restrict__ codes, float* __restrict__ stats,
                  int kind, const GnShape g, int chunks, int64_t rows) {
  extern __shared__ float4 group_s[];                     // a group each
  const BlockAt at_ = block_at(g.tiles, chunks);
  const int t = at_.tile, chunk = at_.chunk;
  const int64_t n = at_.n;
  const int c0 = tile_first(g, t), width = tile_end(g, t) - c0, lane = threadIdx.x & 31;
  const int g0 = c0 / g.cpg, groups = g.parts == 1 ? width / g.cpg : 1;
  for (int j = threadIdx.x >> 5; j < groups; j += kGnThreads / 32) {
    const float4 st = join_stats(parts, n, g0 + j, g, lane);
    if (lane == 0) {
      group_s[j] = st;
      if (stats && chunk == 0 && (g.parts == 1 || t % g.parts == 0))
        reinterpret_cast<float4*>(stats)[n * g.G + g0 + j] = st;
    }
  }
  __syncthreads();
  const int vecs = width / V, R = kGnThreads / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  if (r >= R) return;
  float a[V], b[V], mid[V], inv[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = c0 + v * V + i;
    const float4 st = group_s[c / g.cpg - g0];
    const float w = gamma ? __ldg(gamma + c) : 1.f;
    a[i] = st.y * w;
    b[i] = (beta ? __ldg(beta + c) : 0.f) - st.x * a[i];
    mid[i] = st.z;
    inv[i] = code_factor(st.w);
  }
  const int64_t at = (n * g.S) * g.C + c0 + v * V, first = chunk * rows + r, end = min(g.S, (chunk + 1) * rows);
  const T* p = x + at;
  T* q = y + at;
  int8_t* cd = SAVE ? codes + at : nullptr;
  switch (kind) {
    case kActNone: gn_apply<T, V, kActNone, SAVE>(p, q, cd, g.C, first, end, R, a, b, mid, inv); break;
    case kActRelu: gn_apply<T, V, kActRelu, SAVE>(p, q, cd, g.C, first, end, R, a, b, mid, inv); break;
    case kActSilu: gn_apply<T, V, kActSilu, SAVE>(p, q, cd, g.C, first, end, R, a, b, mid, inv); break;
    case kActGelu: gn_apply<T, V, kActGelu, SAVE>(p, q, cd, g.C, first, end, R, a, b, mid, inv); break;
    default: gn_apply<T, V, kActGeluTanh, SAVE>(p, q, cd, g.C, first, end, R, a, b, mid, inv); break;
  }
}

// ------------------------------------------------------------------ backward
// h = ha * saved + hb, saved a code or (without codes) an element
template <typename T, int V, bool CODES>
ACTNN_DEV void saved_values(const T* __restrict__ x, const int8_t* __restrict__ codes, int64_t at, float (&f)[V]) {
  if constexpr (CODES) unpack_codes<V>(load_codes<V>(codes + at), f);
  else unpack_vec(load_vec<T, V>(x + at), f);
}
template <bool CODES> ACTNN_DEV float2 normal_line(const float4& st) {
  if constexpr (CODES) return make_float2(code_step(st.w) * st.y, (st.z - st.x) * st.y);
  else return make_float2(st.y, -st.x * st.y);
}

template <typename T, int V, int KIND, bool CODES>
ACTNN_DEV void gn_sums(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes, int64_t at0, int64_t C,
                       int64_t first, int64_t end, int64_t step, const float (&ha)[V], const float (&hb)[V], const float (&w)[V],
                       const float (&b)[V], float (&s1)[V], float (&s2)[V]) {
  constexpr bool P = sizeof(T) == 4;
#pragma unroll 2
  for (int64_t k = first; k < end; k += step) {
    const int64_t at = at0 + k * C;
    float d[V], f[V];
    unpack_vec(load_vec<T, V>(dy + at), d);
    saved_values<T, V, CODES>(x, codes, at, f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float h = fmaf(f[i], ha[i], hb[i]);
      const float dz = d[i] * act_both<KIND, P>(fmaf(h, w[i], b[i])).y;
      s1[i] += dz;
      s2[i] = fmaf(dz, h, s2[i]);
    }
  }
}

// A block per sample, run of positions and run of channels.  sums[((n * chunks + chunk) * C + c) * 2]: of dz and of dz * h over the chunk's positions.
template <typename T, int V, bool CODES>
__global__ void __launch_bounds__(kGnThreads)
gn_backward_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                        const float* __restrict__ stats, const float* __restrict__ gamma, const float* __restrict__ beta,
                        float2* __restrict__ sums, int kind, const GnShape g) {
  __shared__ float2 part_s[kGnThreads * V];
  const BlockAt at_ = block_at(g.tiles, g.chunks);
  const int t = at_.tile, chunk = at_.chunk;
  const int64_t n = at_.n;
  const int c0 = tile_first(g, t), width = tile_end(g, t) - c0;
  const int vecs = width / V, R = kGnThreads / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  if (r < R) {
    float ha[V], hb[V], w[V], b[V], s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = c0 + v * V + i;
      const float2 l = normal_line<CODES>(__ldg(reinterpret_cast<const float4*>(stats) + n * g.G + c / g.cpg));
      ha[i] = l.x;
      hb[i] = l.y;
      w[i] = gamma ? __ldg(gamma + c) : 1.f;
      b[i] = beta ? __ldg(beta + c) : 0.f;
      s1[i] = s2[i] = 0.f;
    }
    const int64_t at = (n * g.S) * g.C + c0 + v * V, first = chunk * g.rows + r, end = min(g.S, (chunk + 1) * g.rows);
    switch (kind) {
      case kActNone: gn_sums<T, V, kActNone, CODES>(dy, x, codes, at, g.C, first, end, R, ha, hb, w, b, s1, s2); break;
      case kActRelu: gn_sums<T, V, kActRelu, CODES>(dy, x, codes, at, g.C, first, end, R, ha, hb, w, b, s1, s2); break;
      case kActSilu: gn_sums<T, V, kActSilu, CODES>(dy, x, codes, at, g.C, first, end, R, ha, hb, w, b, s1, s2); break;
      case kActGelu: gn_sums<T, V, kActGelu, CODES>(dy, x, codes, at, g.C, first, end, R, ha, hb, w, b, s1, s2); break;
      default: gn_sums<T, V, kActGeluTanh, CODES>(dy, x, codes, at, g.C, first, end, R, ha, hb, w, b, s1, s2); break;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) part_s[r * width + v * V + i] = make_float2(s1[i], s2[i]);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += kGnThreads) {
    float2 s = make_float2(0.f, 0.f);
    for (int k = 0; k < R; ++k) {
      s.x += part_s[k * width + c].x;
      s.y += part_s[k * width + c].y;
    }
    sums[(n * g.chunks + chunk) * g.C + c0 + c] = s;
  }
}

template <typename T, int V, int KIND, bool CODES>
ACTNN_DEV void gn_grad(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes, T* __restrict__ dx,
                       int64_t at0, int64_t C, int64_t first, int64_t end, int64_t step, const float (&ha)[V], const float (&hb)[V],
                       const float (&w)[V], const float (&b)[V], const float (&rs)[V], const float (&ga)[V], const float (&gb)[V]) {
  constexpr bool P = sizeof(T) == 4;
#pragma unroll 2
  for (int64_t k = first; k < end; k += step) {
    const int64_t at = at0 + k * C;
    float d[V], f[V];
    unpack_vec(load_vec<T, V>(dy + at), d);
    saved_values<T, V, CODES>(x, codes, at, f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float h = fmaf(f[i], ha[i], hb[i]);
      const float dz = d[i] * act_both<KIND, P>(fmaf(h, w[i], b[i])).y;
      d[i] = rs[i] * (fmaf(dz, w[i], -ga[i]) - h * gb[i]);
    }
    store_vec<T, V>(dx + at, d);
  }
}

// A block per sample, run of positions and run of channels, the chunks of this pass.
template <typename T, int V, bool CODES>
__global__ void __launch_bounds__(kGnThreads)
gn_backward_kernel(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                   const float* __restrict__ stats, const float* __restrict__ gamma, const float* __restrict__ beta,
                   const float2* __restrict__ sums, T* __restrict__ dx, int kind, const GnShape g, int chunks, int64_t rows) {
  extern __shared__ float2 means_s[];                     // a group each
  const BlockAt at_ = block_at(g.tiles, chunks);
  const int t = at_.tile, chunk = at_.chunk;
  const int64_t n = at_.n;
  const int c0 = tile_first(g, t), width = tile_end(g, t) - c0, lane = threadIdx.x & 31;
  const int g0 = c0 / g.cpg, groups = g.parts == 1 ? width / g.cpg : 1;
  for (int j = threadIdx.x >> 5; j < groups; j += kGnThreads / 32) {
    float a = 0.f, b = 0.f;
    for (int e = lane; e < g.chunks * g.cpg; e += 32) {
      const int k = e / g.cpg, c = (g0 + j) * g.cpg + (e - k * g.cpg);
      const float2 s = sums[(n * g.chunks + k) * g.C + c];
      const float w = gamma ? __ldg(gamma + c) : 1.f;
      a = fmaf(w, s.x, a);
      b = fmaf(w, s.y, b);
    }
    const float m = (float)g.S * (float)g.cpg;
    a = warp_sum(a) / m;
    b = warp_sum(b) / m;
    if (lane == 0) means_s[j] = make_float2(a, b);
  }
  __syncthreads();
  const int vecs = width / V, R = kGnThreads / vecs;
  const int r = threadIdx.x / vecs, v = threadIdx.x - r * vecs;
  if (r >= R) return;
  float ha[V], hb[V], w[V], b[V], rs[V], ga[V], gb[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = c0 + v * V + i;
    const float4 st = __ldg(reinterpret_cast<const float4*>(stats) + n * g.G + c / g.cpg);
    const float2 l = normal_line<CODES>(st), m = means_s[c / g.cpg - g0];
    ha[i] = l.x;
    hb[i] = l.y;
    w[i] = gamma ? __ldg(gamma + c) : 1.f;
    b[i] = beta ? __ldg(beta + c) : 0.f;
    rs[i] = st.y;
    ga[i] = m.x;
    gb[i] = m.y;
  }
  const int64_t at = (n * g.S) * g.C + c0 + v * V, first = chunk * rows + r, end = min(g.S, (chunk + 1) * rows);
  switch (kind) {
    case kActNone: gn_grad<T, V, kActNone, CODES>(dy, x, codes, dx, at, g.C, first, end, R, ha, hb, w, b, rs, ga, gb); break;
    case kActRelu: gn_grad<T, V, kActRelu, CODES>(dy, x, codes, dx, at, g.C, first, end, R, ha, hb, w, b, rs, ga, gb); break;
    case kActSilu: gn_grad<T, V, kActSilu, CODES>(dy, x, codes, dx, at, g.C, first, end, R, ha, hb, w, b, rs, ga, gb); break;
    case kActGelu: gn_grad<T, V, kActGelu, CODES>(dy, x, codes, dx, at, g.C, first, end, R, ha, hb, w, b, rs, ga, gb); break;
    default: gn_grad<T, V, kActGeluTanh, CODES>(dy, x, codes, dx, at, g.C, first, end, R, ha, hb, w, b, rs, ga, gb); break;
  }
}

// dgamma and dbeta: column sums of the [rows, C] partial sums.  A block takes 32 columns, its warps runs of rows.
__global__ void __launch_bounds__(1024)
gn_column_sums_kernel(const float2* __restrict__ sums, float* __restrict__ dgamma, float* __restrict__ dbeta, int64_t rows, int C) {
  __shared__ float2 part_s[32][32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float2 s = make_float2(0.f, 0.f);
  if (c < C) {
#pragma unroll 4
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

// ------------------------------------------------------------------ host
int gcd(int a, int b) {
  while (b) {
    const int c = a % b;
    a = b;
    b = c;
  }
  return a;
}
// Cuts the channels for vectors of V; false where V does not fit.
bool cut_channels(GnShape& g, int V) {
  if (g.C % V != 0) return false;
  const int most = kGnThreads * V, whole = g.cpg / gcd(g.cpg, V) * V;      // whole vectors of whole groups
  g.parts = 1;
  if (g.C <= most) {
    g.tile = g.C;
  } else if (whole <= most) {
    g.tile = most / whole * whole;
  } else if (g.cpg % V == 0) {
    g.tile = most;
    g.parts = (g.cpg + most - 1) / most;
    g.tiles = g.G * g.parts;
    return true;
  } else {
    return false;
  }
  g.tiles = (g.C + g.tile - 1) / g.tile;
  return true;
}
// Runs of positions for a pass: enough blocks to fill the GPU `waves` times, but `least` positions a thread at least.
void cut_positions(const GnShape& g, int64_t N, int V, int least, int waves, int* chunks, int64_t* rows) {
  const int vecs = (g.tile < g.C ? g.tile : g.C) / V, R = kGnThreads / (vecs > 0 ? vecs : 1);
  const int64_t want = (int64_t)device_info().sm_count * waves;
  int64_t k = (want + N * g.tiles - 1) / (N * g.tiles);
  const int64_t most = (g.S + (int64_t)R * least - 1) / ((int64_t)R * least);
  if (k > most) k = most;
  if (k < 1) k = 1;
  *rows = ((g.S + k - 1) / k + R - 1) / R * R;
  *chunks = (int)((g.S + *rows - 1) / *rows);
}
constexpr int kGnLeast = 4, kGnWaves = 8;

int gn_shape(GnShape& g, int64_t N, int64_t S, int64_t C, int64_t G) {
  if (N < 0 || S < 0 || C < 1 || G < 1 || C % G != 0 || C > (1 << 24)) return ACTNN_ERR_SHAPE;
  if (S > ((int64_t)1 << 40) / C || (N > 0 && S * C > ((int64_t)1 << 42) / N)) return ACTNN_ERR_SHAPE;
  g.S = S;
  g.C = (int)C;
  g.G = (int)G;
  g.cpg = (int)(C / G);
  return ACTNN_OK;
}
// The widest vectors that the channels and (n_io of them) pointers take: 8, 4 or 1 elements.
int gn_vector(GnShape& g, int dtype, const void* const* io, int n_io) {
  for (int V : {8, 4}) {
    const int bytes = V * dtype_size(dtype) < 16 ? V * dtype_size(dtype) : 16;
    bool ok = true;
    for (int i = 0; i < n_io; ++i) ok = ok && aligned(io[i], bytes);
    if (ok && cut_channels(g, V)) return V;
  }
  cut_channels(g, 1);
  return 1;
}
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
// Most bytes that any vector width needs.
int64_t gn_bytes(GnShape g, int64_t N) {
  int64_t most = 0;
  for (int V : {8, 4, 1}) {
    if (!cut_channels(g, V)) continue;
    int chunks;
    int64_t rows;
    cut_positions(g, N, V, kGnLeast, kGnWaves, &chunks, &rows);
    const int64_t fwd = N * g.G * chunks * g.parts * (int64_t)sizeof(Part), bwd = N * chunks * g.C * (int64_t)sizeof(float2);
    most = fwd > most ? fwd : most;
    most = bwd > most ? bwd : most;
  }
  return align256(most);
}

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

template <typename T, int V> int gn_forward(const GnCall& c, GnShape g) {
  cut_positions(g, c.N, V, kGnLeast, kGnWaves, &g.chunks, &g.rows);
  const int64_t blocks = c.N * g.chunks * g.tiles;
  if (blocks > 0x7fffffff) return ACTNN_ERR_SHAPE;
  const unsigned grid = (unsigned)blocks;
  const size_t smem = sizeof(float4) * (g.parts == 1 ? g.tile / g.cpg : 1);
  Part* parts = (Part*)c.workspace;
  gn_stats_kernel<T, V><<<grid, kGnThreads, 0, c.stream>>>((const T*)c.x, parts, g);
  auto* second = c.codes ? gn_forward_kernel<T, V, true> : gn_forward_kernel<T, V, false>;
  second<<<grid, kGnThreads, smem, c.stream>>>((const T*)c.x, parts, c.gamma, c.beta, (T*)c.out, c.codes, c.stats, c.kind, g,
                                               g.chunks, g.rows);
  return check_launch();
}
template <typename T, int V, bool CODES> int gn_backward(const GnCall& c, GnShape g) {
  cut_positions(g, c.N, V, kGnLeast, kGnWaves, &g.chunks, &g.rows);
  const int64_t blocks = c.N * g.chunks * g.tiles;
  if (blocks > 0x7fffffff) return ACTNN_ERR_SHAPE;
  const unsigned grid = (unsigned)blocks;
  const size_t smem = sizeof(float2) * (g.parts == 1 ? g.tile / g.cpg : 1);
  float2* sums = (float2*)c.workspace;
  gn_backward_sums_kernel<T, V, CODES><<<grid, kGnThreads, 0, c.stream>>>((const T*)c.dy, (const T*)c.x, c.codes, c.stats, c.gamma,
                                                                         c.beta, sums, c.kind, g);
  gn_backward_kernel<T, V, CODES><<<grid, kGnThreads, smem, c.stream>>>((const T*)c.dy, (const T*)c.x, c.codes, c.stats, c.gamma,
                                                                       c.beta, sums, (T*)c.out, c.kind, g, g.chunks, g.rows);
  if (c.dgamma || c.dbeta)
    gn_column_sums_kernel<<<(g.C + 31) / 32, 1024, 0, c.stream>>>(sums, c.dgamma, c.dbeta, c.N * g.chunks, g.C);
  return check_launch();
}

template <typename T> int gn_launch(const GnCall& c, const GnShape& g, int V, bool forward) {
#define GN_PICK(W) \
  (forward ? gn_forward<T, W>(c, g) : c.codes ? gn_backward<T, W, true>(c, g) : gn_backward<T, W, false>(c, g))
  return V == 8 ? GN_PICK(8) : V == 4 ? GN_PICK(4) : GN_PICK(1);
#undef GN_PICK
}
int gn_dispatch(const GnCall& c, const GnShape& g, int V, int dtype, bool forward) {
  switch (dtype) {
    case ACTNN_F32: return gn_launch<float>(c, g, V, forward);
    case ACTNN_F16: return gn_launch<__half>(c, g, V, forward);
    default: return gn_launch<__nv_bfloat16>(c, g, V, forward);
  }
}

}  // namespace
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_group_norm_workspace(int64_t N, int64_t S, int64_t C, int64_t G, int64_t* bytes) {
  if (!bytes) return ACTNN_ERR_NULL;
  GnShape g{};
  if (int st = gn_shape(g, N, S, C, G)) return st;
  *bytes = N == 0 || S == 0 ? 256 : gn_bytes(g, N);
  return ACTNN_OK;
}

extern "C" int actnn_group_norm_forward(const void* x, const float* gamma, const float* beta, void* y, int8_t* codes, float* stats,
                                        int64_t N, int64_t S, int64_t C, int64_t G, double eps, int kind, int dtype,
                                        void* workspace, int64_t workspace_bytes, actnn_stream_t stream) {
  GnShape g{};
  if (int st = gn_shape(g, N, S, C, G)) return st;
  if (kind < 0 || kind >= kActKinds || !(eps >= 0.0)) return ACTNN_ERR_ARG;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (N == 0 || S == 0) return ACTNN_OK;
  if (!x || !y || !workspace || (codes && !stats)) return ACTNN_ERR_NULL;
  const int size = dtype_size(dtype);
  if (!aligned(x, size) || !aligned(y, size) || !aligned(workspace, 16) || !aligned(stats, 16)) return ACTNN_ERR_ALIGN;
  if (workspace_bytes < gn_bytes(g, N)) return ACTNN_ERR_CAPACITY;
  g.eps = (float)eps;
  const void* io[2] = {x, y};
  GnCall c{};
  c.x = x; c.gamma = gamma; c.beta = beta; c.out = y; c.codes = codes; c.stats = stats; c.workspace = workspace; c.N = N;
  c.kind = kind; c.stream = (cudaStream_t)stream;
  int V = gn_vector(g, dtype, io, 2);
  if (codes && V > 1 && !aligned(codes, V)) { V = 1; cut_channels(g, 1); }
  return gn_dispatch(c, g, V, dtype, true);
}

extern "C" int actnn_group_norm_backward(const void* grad_y, const void* x, const int8_t* codes, const float* stats,
                                         const float* gamma, const float* beta, void* grad_x, float* grad_gamma, float* grad_beta,
                                         int64_t N, int64_t S, int64_t C, int64_t G, int kind, int dtype, void* workspace,
                                         int64_t workspace_bytes, actnn_stream_t stream) {
  GnShape g{};
  if (int st = gn_shape(g, N, S, C, G)) return st;
  if (kind < 0 || kind >= kActKinds) return ACTNN_ERR_ARG;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (N == 0 || S == 0) {                                  // the gradients of the parameters are sums of nothing
    for (float* p : {grad_gamma, grad_beta})
      if (p && cudaMemsetAsync(p, 0, C * sizeof(float), (cudaStream_t)stream) != cudaSuccess) return ACTNN_ERR_LAUNCH;
    return ACTNN_OK;
  }
  if (!grad_y || !grad_x || !stats || !workspace || (!x && !codes)) return ACTNN_ERR_NULL;
  const int size = dtype_size(dtype);
  if (!aligned(grad_y, size) || !aligned(grad_x, size) || !aligned(workspace, 16) || !aligned(stats, 16)) return ACTNN_ERR_ALIGN;
  if (!codes && !aligned(x, size)) return ACTNN_ERR_ALIGN;
  if (workspace_bytes < gn_bytes(g, N)) return ACTNN_ERR_CAPACITY;
  const void* io[3] = {grad_y, grad_x, codes ? grad_y : x};
  GnCall c{};
  c.x = x; c.dy = grad_y; c.gamma = gamma; c.beta = beta; c.out = grad_x; c.codes = (int8_t*)codes; c.stats = (float*)stats;
  c.dgamma = grad_gamma; c.dbeta = grad_beta; c.workspace = workspace; c.N = N; c.kind = kind; c.stream = (cudaStream_t)stream;
  int V = gn_vector(g, dtype, io, 3);
  if (codes && V > 1 && !aligned(codes, V)) { V = 1; cut_channels(g, 1); }
  return gn_dispatch(c, g, V, dtype, false);
}
