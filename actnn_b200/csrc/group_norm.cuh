// Group norm with an activation on channels-last activations [N, S, C], S positions of C channels, G groups of C / G channels.
//
//   forward   mean, var over the S * C / G elements of a (sample, group);  z = (x - mean) * rstd * gamma + beta;  y = f(z)
//             codes: (x - mid) in 127 steps either way of half the group's range, mid the middle of the range
//   backward  x^ = mid + code * step,  h = (x^ - mean) * rstd,  dz = dy * f'(h * gamma + beta)
//             dgamma = sum dz * h,  dbeta = sum dz   (over samples and positions)
//             dx = rstd * (dz * gamma - A - h * B),  A, B = means over the group of dz * gamma and dz * gamma * h
//
// Every output needs a sum over its group.  Where the positions of a sample's groups fit the shared memory of a cluster, one
// launch does each way: a block requests its share of the positions at once, all of it (cp.async), sums while they arrive, joins its
// sums with those of the cluster's other blocks through distributed shared memory, and computes the outputs from what it
// holds.  HBM sees every byte once.  Where they do not fit, two launches: the first leaves partial sums of `chunks` runs of
// positions, the second joins those it needs before it starts and reads the data again.  Either way sums are taken in a fixed
// order, so results are reproducible.
//
// A thread keeps V consecutive channels and walks down the positions: everything that belongs to a channel or group stays in
// registers, folded into as few constants as the formulas leave.  z = za * code + zb and dx = k1 * dz + k2 * code + k3 take
// three a channel and two a group (one set of these for the thread where V divides a group's channels).  What a thread will
// read it copies to places of its own in shared memory, so that neither registers nor barriers limit how many bytes are under
// way.
//
// Measured on a B200, float16, 512 x 256 x 28 x 28 (103 M elements), two launches each way: statistics 45 us, output and codes 79, sums 73,
// gradient 80; their bytes take 31, 79, 47 and 79 at the copy rate.  The sums wait for nothing but instructions: 14 an element, the
// unit of exponentials and reciprocals 60 - 70 % busy.  Batches of samples small enough for the L2 between the two launches were
// slower (fills and drains of the GPU), so was one launch in several waves; one reciprocal for a pair of elements changed nothing.
//
// The range, and with it the codes, follow from exact minima and maxima by single fp32 operations: reproducible to the bit.
// The variance is joined from sums about a value of each thread's own (its first one), which loses nothing to cancellation
// however far the mean is from zero: the sum of squares about one of n values exceeds the one about their mean n-fold at most.
#pragma once

#include <atomic>

#include "activation.cuh"
#include "cluster.cuh"

namespace actnn {

// How the work is cut.  Channels: `tiles` runs of `tile` channels, at most kGnThreads vectors each, of whole groups or a part of one
// group (`parts` of them a group).  Positions: `chunks` runs of `rows`, the last one shorter; with one launch they are the blocks
// of a cluster.
struct GnShape {
  int64_t S;
  int C, G, cpg;                        // channels, groups, channels of a group
  int V;                                // channels of a thread: 8, 4, 2 or 1, a divisor of C
  int tile, tiles, parts;
  int chunks;
  int64_t rows;
  int first_chunks, first_parts;        // the cut of the first of two launches, whose partial results the second one joins
  int64_t first_rows;
  int held;                             // positions a thread holds at most; 0: two launches
  bool wide;                            // gamma and beta on 16 bytes
  FastDiv by_tiles, by_chunks, by_vecs, by_cpg, by_cells;       // by_vecs: of a whole tile; by_cells: sums of a group in a row of threads
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

// group_norm.cu, group_norm_f16.cu, group_norm_bf16.cu: the launches of a type; and, in the first,
// the cut of the positions for a launch of which `resident` blocks fit the GPU at a time, and a block spends as long as `extra`
// positions of a thread take before and after them.
void gn_cut_positions(GnShape& g, int64_t N, int64_t resident, int extra);
int gn_run_f32(const GnCall& c, const GnShape& g, bool forward);
int gn_run_f16(const GnCall& c, const GnShape& g, bool forward);
int gn_run_bf16(const GnCall& c, const GnShape& g, bool forward);

constexpr int kGnThreads = 256;
constexpr int kGnMostSmem = 224 * 1024;         // of an SM's 227 KB
// Shared memory of a block besides the positions it holds: the scratch of its sums (a value of 16 bytes each thread and kind,
// or of 8 each channel) and two tables of the groups.
ACTNN_HD int gn_groups(const GnShape& g) { return g.parts == 1 ? g.tile / g.cpg : 1; }
ACTNN_HD int gn_scratch(const GnShape& g, bool forward) {
  return forward ? kGnThreads * (g.cpg % g.V == 0 ? 1 : g.V) * 16 : kGnThreads * g.V * 8;
}
ACTNN_HD int gn_tables(const GnShape& g) { return 2 * gn_groups(g) * 16; }

namespace {

template <typename T> constexpr int kGnResident = sizeof(T) == 2 ? 3 : 2;      // blocks of an SM that the registers have to allow

ACTNN_DEV int tile_first(const GnShape& g, int t) {
  return g.parts == 1 ? t * g.tile : t / g.parts * g.cpg + t % g.parts * g.tile;
}
ACTNN_DEV int tile_end(const GnShape& g, int t) {
  return g.parts == 1 ? min(g.C, (t + 1) * g.tile) : min((t / g.parts + 1) * g.cpg, tile_first(g, t) + g.tile);
}
// The place of a block and thread: sample, run of positions, run of channels; the thread's row of positions r, R of them, and
// its channels c to c + V.
struct Place {
  int64_t n, first;                     // sample, first position of the block
  int rows;                             // positions of the block; less than one in the last blocks of a short cluster
  int chunk, tile, c0, width, vecs, R, r, c, count, g0;         // g0: the tile's first group
  int full, more;                       // every row of threads has `full` positions, the first `more` of them one more
  int64_t at, step;                     // the thread's first element, and from one of its positions to the next
};
ACTNN_DEV int row_count(const Place& p, int r) { return p.full + (r < p.more ? 1 : 0); }
// BACK: from the last sample to the first, for a launch that reads what the one before it read: the end is still in the L2.
template <int V, bool BACK = false> ACTNN_DEV Place place_of(const GnShape& g) {
  Place p;
  const uint32_t block = BACK ? gridDim.x - 1 - blockIdx.x : blockIdx.x, a = fast_div(block, g.by_chunks), n = fast_div(a, g.by_tiles);
  p.n = n;
  p.chunk = (int)(block - a * (uint32_t)g.chunks);
  p.tile = (int)(a - n * (uint32_t)g.tiles);
  p.c0 = tile_first(g, p.tile);
  p.width = tile_end(g, p.tile) - p.c0;
  p.g0 = (int)fast_div(p.c0, g.by_cpg);
  p.vecs = p.width / V;
  if (p.width == g.tile) {
    p.R = (int)fast_div(blockDim.x, g.by_vecs);
    p.r = (int)fast_div(threadIdx.x, g.by_vecs);
  } else {
    p.R = blockDim.x / p.vecs;
    p.r = threadIdx.x / p.vecs;
  }
  p.c = p.c0 + (threadIdx.x - p.r * p.vecs) * V;
  p.first = p.chunk * g.rows;
  p.rows = (int)min(g.S - p.first, g.rows);
  p.full = p.rows > 0 ? (int)((uint32_t)p.rows / (uint32_t)p.R) : 0;
  p.more = p.rows > 0 ? p.rows - p.full * p.R : 0;
  p.count = p.r < p.R ? row_count(p, p.r) : 0;
  p.at = (p.n * g.S + p.first + p.r) * g.C + p.c;
  p.step = (int64_t)p.R * g.C;
  return p;
}
// The group of channel p.c + i, counted from the tile's first.
ACTNN_DEV int group_at(const Place& p, const GnShape& g, int i) { return (int)fast_div(p.c + i, g.by_cpg) - p.g0; }
// Parameters of the thread's channels; `absent` where there are none.
template <int V> ACTNN_DEV void parameters(const float* p, int c, bool wide, float absent, float (&v)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = absent;
  } else if (V >= 4 && wide) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(p + c) + i);
      v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __ldg(p + c + i);
  }
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
// How many lanes share a group of `entries`: so many that none idles, and that the block has lanes for all `groups` at a time.
ACTNN_DEV int lanes_for(int entries, int groups) {
  const int wanted = entries >= 32 ? 32 : entries <= 1 ? 1 : 1 << (32 - __clz(entries - 1));
  const int there = groups >= (int)blockDim.x ? 1 : 1 << (31 - __clz((int)blockDim.x / groups));
  return min(wanted, min(there, 32));
}

constexpr float kInf = __builtin_huge_valf();

// ------------------------------------------------------------------ what a thread reads
// A position is a vector of V elements of T and, in the backward pass, one of what is kept of the input: codes, or elements.
struct Nothing {};
template <typename T, int V, bool CODES> struct Kept {
  static constexpr int kBytes = V * sizeof(T);
  using Words = Vec<T, V>;
  static ACTNN_DEV Words load(const char* p) { return load_vec<T, V>((const T*)p); }
};
template <typename T, int V> struct Kept<T, V, true> {
  static constexpr int kBytes = V;
  using Words = Codes<V>;
  static ACTNN_DEV Words load(const char* p) { return load_codes<V>((const int8_t*)p); }
};
template <typename T, int V> struct Alone {
  static constexpr int kBytes = 0;
  using Words = Nothing;
  static ACTNN_DEV Words load(const char*) { return Words(); }
};

template <int BYTES> ACTNN_DEV void copy_async(uint32_t dst, const char* src) {
  if constexpr (BYTES == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(dst), "l"(src) : "memory");
  else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" :: "r"(dst), "l"(src) : "memory");
  else
#pragma unroll
    for (int i = 0; i < BYTES; i += 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst + i), "l"(src + i) : "memory");
}
ACTNN_DEV void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> ACTNN_DEV void copy_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(LEFT) : "memory"); }
template <int BYTES> ACTNN_DEV void from_shared(uint32_t src, uint32_t* w) {
  if constexpr (BYTES == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(src) : "memory");
  else if constexpr (BYTES == 8) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(src) : "memory");
  else
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                   : "r"(src + 16 * i) : "memory");
}

// The positions of a thread, in places of its own: `places` of them for every thread of the block from `shared` on.
// SUMS: for a pass that writes nothing of a position's size.
template <typename T, int V, typename K, bool SUMS> struct Positions {
  static constexpr int A = V * sizeof(T), B = K::kBytes;
  static constexpr bool kAsync = V > 1 && A >= (SUMS ? 8 : 4) && (B == 0 || B >= 4);        // the asynchronous copy knows 4, 8 and 16 bytes
  static constexpr int kAhead = SUMS ? 8 : 4;
  static constexpr int kDepth = B == 0 ? 8 : 6;                                // positions of a ring
  static constexpr int kPlace = kAsync ? kGnThreads * (A + B) : 0;             // bytes of a position of all threads
  using Words = typename K::Words;
  const char *a, *b;
  int64_t step_a, step_b;
  int count;
  uint32_t to_a, to_b;

  ACTNN_DEV Positions(const T* x, const void* kept, const Place& p, uint32_t shared, int places) {
    a = (const char*)(x + p.at);
    step_a = p.step * (int64_t)sizeof(T);
    b = (const char*)kept + p.at * (B / V);
    step_b = p.step * (B / V);
    count = p.count;
    to_a = shared + threadIdx.x * A;
    to_b = shared + places * (kGnThreads * A) + threadIdx.x * B;
  }
  ACTNN_DEV void ask(int place) {                        // the next position
    copy_async<A>(to_a + place * (kGnThreads * A), a);
    a += step_a;
    if constexpr (B > 0) {
      copy_async<B>(to_b + place * (kGnThreads * B), b);
      b += step_b;
    }
  }
  template <typename Take> ACTNN_DEV void give(int place, Take& take) {
    Vec<T, V> w;
    Words k;
    if constexpr (kAsync) {
      from_shared<A>(to_a + place * (kGnThreads * A), w.w);
      if constexpr (B > 0) from_shared<B>(to_b + place * (kGnThreads * B), k.w);
    }
    take(w, k);
  }
  // Two launches: once through, kDepth - 1 positions ahead.
  ACTNN_DEV void start() {
    if constexpr (kAsync) {
#pragma unroll
      for (int i = 0; i < kDepth - 1; ++i) {
        if (i < count) ask(i);
        copy_commit();
      }
    }
  }
  template <typename Take> ACTNN_DEV void through(Take take) {
    if constexpr (kAsync) {
      for (int base = 0; base < count; base += kDepth) {
#pragma unroll
        for (int s = 0; s < kDepth; ++s) {
          if (base + s < count) {
            copy_wait<kDepth - 2>();
            Vec<T, V> w;
            Words k;
            from_shared<A>(to_a + s * (kGnThreads * A), w.w);
            if constexpr (B > 0) from_shared<B>(to_b + s * (kGnThreads * B), k.w);
            if (base + s + kDepth - 1 < count) ask((s + kDepth - 1) % kDepth);      // the place that the position before has left
            copy_commit();
            take(w, k);
          }
        }
      }
    } else {
      int i = 0;
      for (; i + kAhead <= count; i += kAhead) {          // kAhead requests before the first is used
        Vec<T, V> w[kAhead];
        Words k[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j, a += step_a, b += step_b) {
          w[j] = load_vec<T, V>((const T*)a);
          k[j] = K::load(b);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) take(w[j], k[j]);
      }
      for (; i < count; ++i, a += step_a, b += step_b) {
        const Words k = K::load(b);
        take(load_vec<T, V>((const T*)a), k);
      }
    }
  }
  // One launch: all of them, in four portions, and then again from where they are.
  ACTNN_DEV void start_all() {
    if constexpr (kAsync) {
      const int per = (count + 3) >> 2;
      int i = 0;
#pragma unroll
      for (int q = 1; q <= 4; ++q) {
        for (const int end = min(count, q * per); i < end; ++i) ask(i);
        copy_commit();
      }
    }
  }
  template <typename Take> ACTNN_DEV void as_they_come(Take take) {
    const int per = (count + 3) >> 2;
    int i = 0;
    auto portion = [&](int q) {
#pragma unroll 2
      for (const int end = min(count, q * per); i < end; ++i) give(i, take);
    };
    copy_wait<3>();
    portion(1);
    copy_wait<2>();
    portion(2);
    copy_wait<1>();
    portion(3);
    copy_wait<0>();
    portion(4);
  }
  template <typename Take> ACTNN_DEV void again(Take take) {
#pragma unroll 2
    for (int i = 0; i < count; ++i) give(i, take);
  }
};

// ------------------------------------------------------------------ constants and running values of a thread
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
// Of a thread: ONE value of each kind where V divides cpg, else one a channel.
template <typename T, int V, bool ONE> struct ThreadStats {
  using F = typename Many<V>::F;
  static constexpr int N = Many<V>::N, M = ONE ? 1 : V, kSums = ONE ? 1 : N;
  F shift[kSums], s2[kSums], q2[kSums];                        // less the shift; sums of differences and of their squares
  Extremes<T, V, M> ex;

  ACTNN_DEV void start(const T* p) {                           // the thread's first position
    if constexpr (ONE || V == 1) {
      shift[0] = f_both<F>(-to_float(p[0]));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) shift[i] = make_float2(-to_float(p[2 * i]), -to_float(p[2 * i + 1]));
    }
#pragma unroll
    for (int i = 0; i < kSums; ++i) s2[i] = q2[i] = f_both<F>(0.f);
  }
  ACTNN_DEV void operator()(const Vec<T, V>& w, const Nothing&) {
    F f[N];
    unpack_vec(w, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int to = ONE ? 0 : i;
      const F d = f_add(f[i], shift[to]);
      s2[to] = f_add(s2[to], d);
      q2[to] = f_fma(d, d, q2[to]);
    }
    ex.take(w, f);
  }
  static ACTNN_DEV float part_of(const F (&v)[kSums], int i) {
    if constexpr (V == 1) return v[0];
    else return i & 1 ? v[i / 2].y : v[i / 2].x;
  }
  // To cells[0 .. M): sum, squares about the mean, minimum, maximum, of `count` positions.
  ACTNN_DEV void finish(float4* cells, int count) const {
    const float items = (float)(count * (V / M));
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const float s = ONE ? f_sum(s2[0]) : part_of(s2, i), q = ONE ? f_sum(q2[0]) : part_of(q2, i);
      const float2 e = ex.get(i);
      cells[i] = make_float4(fmaf(items, -part_of(shift, i), s), q - s * (s / items), e.x, e.y);
    }
  }
  static ACTNN_DEV void none(float4* cells) {
#pragma unroll
    for (int i = 0; i < M; ++i) cells[i] = make_float4(0.f, 0.f, kInf, -kInf);
  }
};

// Joins the cells of a block's threads: give(group of the tile, Part), once for each, `M` cells a thread.  Lanes that share a group
// take its sum, then the squares about its mean.
template <int V, int M, typename Give> ACTNN_DEV void join_block(const float4* cell_s, const Place& p, const GnShape& g, Give give) {
  const int cells = p.vecs * M, groups = g.parts == 1 ? (int)fast_div(p.width, g.by_cpg) : 1;
  const int cpg = g.parts == 1 ? (int)g.by_cells.d : cells, entries = p.R * cpg;       // cells of a group in a row of threads
  const float items_full = (float)(p.full * (V / M)), items_more = (float)((p.full + 1) * (V / M));
  const float per_full = 1.f / items_full, per_more = 1.f / items_more;
  auto row_of = [&](int e) { return g.parts == 1 ? (int)fast_div(e, g.by_cells) : e / cpg; };
  const int L = lanes_for(entries, groups), member = threadIdx.x & (L - 1), per = blockDim.x / L;
  for (int j0 = 0; j0 < groups; j0 += per) {
    const int j = j0 + threadIdx.x / L;
    const bool in = j < groups;
    float sum = 0.f, lo = kInf, hi = -kInf, m2 = 0.f;
    for (int e = member; in && e < entries; e += L) {
      const int er = row_of(e);
      const float4 q = cell_s[er * cells + j * cpg + (e - er * cpg)];
      sum += q.x;
      lo = min_nan(lo, q.z);
      hi = max_nan(hi, q.w);
    }
    sum = lanes_sum(sum, L);
    const float mean = sum / ((float)p.rows * (float)(cpg * (V / M)));
    for (int e = member; in && e < entries; e += L) {
      const int er = row_of(e);
      const float4 q = cell_s[er * cells + j * cpg + (e - er * cpg)];
      const bool one_more = er < p.more;
      const float items = one_more ? items_more : items_full;
      if (items > 0.f) {
        const float d = q.x * (one_more ? per_more : per_full) - mean;
        m2 += fmaf(items * d, d, q.y);
      }
    }
    m2 = lanes_sum(m2, L);
    lo = lanes_min(lo, L);
    hi = lanes_max(hi, L);
    if (in && member == 0) give(j, Part{mean, m2, lo, hi});
  }
}

ACTNN_DEV float run_rows(int64_t S, int64_t rows, int run) { return (float)max((int64_t)0, min(S, (run + 1) * rows) - run * rows); }
// Elements of partial result i of a group.
ACTNN_DEV float part_items(const GnShape& g, int i) {
  if (g.first_parts == 1) return run_rows(g.S, g.first_rows, i) * (float)g.cpg;
  const int chunk = i / g.first_parts, part = i - chunk * g.first_parts;
  return run_rows(g.S, g.first_rows, chunk) * (float)(min(g.cpg, (part + 1) * g.tile) - part * g.tile);
}
// Joins `count` partial results, load(i) of items(i) elements each, over L lanes.
template <typename Load, typename Items>
ACTNN_DEV Part join_parts(int count, const GnShape& g, int member, int L, Load load, Items items) {
  float sum = 0.f, lo = kInf, hi = -kInf, m2 = 0.f;
  for (int i = member; i < count; i += L) {
    const Part q = load(i);
    const float c = items(i);
    if (c > 0.f) sum = fmaf(c, q.mean, sum);
    lo = min_nan(lo, q.lo);
    hi = max_nan(hi, q.hi);
  }
  const float m = (float)g.S * (float)g.cpg;
  const float mean = lanes_sum(sum, L) / m;
  for (int i = member; i < count; i += L) {
    const Part q = load(i);
    const float c = items(i), d = q.mean - mean;
    if (c > 0.f) m2 += fmaf(c * d, d, q.m2);
  }
  return Part{mean, lanes_sum(m2, L), lanes_min(lo, L), lanes_max(hi, L)};
}
// Mean, rstd, mid and half of the range.
ACTNN_DEV float4 stats_of(const Part& q, const GnShape& g) {
  const float var = q.m2 / ((float)g.S * (float)g.cpg);
  const float mid = __fadd_rn(__fmul_rn(0.5f, q.hi), __fmul_rn(0.5f, q.lo));
  float half = __fsub_rn(__fmul_rn(0.5f, q.hi), __fmul_rn(0.5f, q.lo));
  half = half < kTiny ? kTiny : half;                                      // a NaN stays one
  return make_float4(q.mean, 1.f / sqrtf(var + g.eps), mid, half);
}

// ------------------------------------------------------------------ output and codes
template <typename T, int V, bool ONE, int KIND, bool SAVE> struct Apply {
  using F = typename Many<V>::F;
  static constexpr int N = Many<V>::N;
  const Row<V>&a, &b;
  const GroupRow<V, ONE>&mid, &inv;                     // less the middle; codes a unit
  T* y;
  int8_t* codes;
  int64_t step;
  ACTNN_DEV void operator()(const Vec<T, V>& w, const Nothing&) {
    F f[N], o[N];
    unpack_vec(w, f);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = act_value<KIND, sizeof(T) == 4>(f_fma(f[i], a.f[i], b.f[i]));
    store_vec<T, V>(y, o);
    y += step;
    if constexpr (SAVE) {
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = code_bits(f_add(f[i], mid.at(i)), inv.at(i));
      store_codes<V>(codes, o);
      codes += step;
    }
  }
};
// The second half of the forward pass: group_s holds mean, rstd, mid and half range of the tile's groups; HELD: the positions
// are in shared memory.
template <typename T, int V, bool ONE, bool SAVE, bool HELD, bool SUMS>
ACTNN_DEV void apply_all(Positions<T, V, Alone<T, V>, SUMS>& pos, const float4* group_s, const Place& p, const GnShape& g, const float* gamma,
                         const float* beta, T* y, int8_t* codes, int kind) {
  Row<V> a, b;
  GroupRow<V, ONE> mid, inv;
  float w[V], shift[V];
  parameters<V>(gamma, p.c, g.wide, 1.f, w);
  parameters<V>(beta, p.c, g.wide, 0.f, shift);
  float4 st;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i == 0 || !ONE) {
      st = group_s[group_at(p, g, i)];
      mid.set(i, -st.z);
      inv.set(i, code_factor(st.w));
    }
    a.set(i, st.y * w[i]);
    b.set(i, shift[i] - st.x * (st.y * w[i]));
  }
  y += p.at;
  codes = SAVE ? codes + p.at : nullptr;
  auto with = [&](auto put) {
    if constexpr (HELD) pos.again(put);
    else pos.through(put);
  };
  switch (kind) {
    case kActNone: with(Apply<T, V, ONE, kActNone, SAVE>{a, b, mid, inv, y, codes, p.step}); break;
    case kActRelu: with(Apply<T, V, ONE, kActRelu, SAVE>{a, b, mid, inv, y, codes, p.step}); break;
    case kActSilu: with(Apply<T, V, ONE, kActSilu, SAVE>{a, b, mid, inv, y, codes, p.step}); break;
    case kActGelu: with(Apply<T, V, ONE, kActGelu, SAVE>{a, b, mid, inv, y, codes, p.step}); break;
    default: with(Apply<T, V, ONE, kActGeluTanh, SAVE>{a, b, mid, inv, y, codes, p.step}); break;
  }
}
ACTNN_DEV void keep_stats(float* stats, const Place& p, const GnShape& g, int group, const float4& st) {
  if (stats && p.chunk == 0 && (g.parts == 1 || p.tile % g.parts == 0)) reinterpret_cast<float4*>(stats)[p.n * g.G + group] = st;
}

// Two launches, the first.  out[((n * G + group) * chunks + chunk) * parts + part].
template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_stats_kernel(const T* __restrict__ x, Part* __restrict__ out, const GnShape g) {
  using Stats = ThreadStats<T, V, ONE>;
  extern __shared__ float4 dynamic_s[];                   // scratch, ring
  const Place p = place_of<V>(g);
  Positions<T, V, Alone<T, V>, true> pos(x, nullptr, p, smem_addr(dynamic_s) + gn_scratch(g, true), Positions<T, V, Alone<T, V>, true>::kDepth);
  pos.start();
  float4* cells = dynamic_s + threadIdx.x * Stats::M;
  if (p.count > 0) {
    Stats s;
    s.start(x + p.at);
    pos.through([&](const Vec<T, V>& w, const Nothing& k) { s(w, k); });
    s.finish(cells, p.count);
  } else {
    Stats::none(cells);
  }
  __syncthreads();
  join_block<V, Stats::M>(dynamic_s, p, g, [&](int j, const Part& q) {
    const int group = p.g0 + j, part = g.parts == 1 ? 0 : p.tile % g.parts;
    out[((p.n * g.G + group) * g.chunks + p.chunk) * g.parts + part] = q;
  });
}
// The second.  stats[(n * G + group) * 4], unless NULL: kept for the backward pass.
template <typename T, int V, bool ONE, bool SAVE>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_forward_kernel(const T* __restrict__ x, const Part* __restrict__ parts, const float* __restrict__ gamma,
                  const float* __restrict__ beta, T* __restrict__ y, int8_t* __restrict__ codes, float* __restrict__ stats,
                  int kind, const GnShape g) {
  extern __shared__ float4 dynamic_s[];                   // tables, ring
  const Place p = place_of<V, true>(g);
  Positions<T, V, Alone<T, V>, false> pos(x, nullptr, p, smem_addr(dynamic_s) + gn_tables(g), Positions<T, V, Alone<T, V>, false>::kDepth);
  pos.start();
  const int g0 = p.g0, groups = g.parts == 1 ? (int)fast_div(p.width, g.by_cpg) : 1, count = g.first_chunks * g.first_parts;
  const int L = lanes_for(count, groups), per = blockDim.x / L, member = threadIdx.x & (L - 1);
  for (int j0 = 0; j0 < groups; j0 += per) {
    const int j = j0 + threadIdx.x / L;
    const Part* q = parts + (p.n * g.G + g0 + (j < groups ? j : 0)) * count;
    const Part one = join_parts(j < groups ? count : 0, g, member, L, [&](int i) { return q[i]; }, [&](int i) { return part_items(g, i); });
    const float4 st = stats_of(one, g);
    if (j < groups && member == 0) {
      dynamic_s[j] = st;
      keep_stats(stats, p, g, g0 + j, st);
    }
  }
  __syncthreads();
  if (p.count > 0) apply_all<T, V, ONE, SAVE, false, false>(pos, dynamic_s, p, g, gamma, beta, y, codes, kind);
}
// One launch, a cluster of `chunks` blocks for each sample and run of channels (whole groups).
template <typename T, int V, bool ONE, bool SAVE>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_forward_held_kernel(const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta, T* __restrict__ y,
                       int8_t* __restrict__ codes, float* __restrict__ stats, int kind, const GnShape g) {
  using Stats = ThreadStats<T, V, ONE>;
  extern __shared__ float4 dynamic_s[];                   // tables (own partial results, joined ones), scratch, positions
  const int table = gn_groups(g);
  float4 *own_s = dynamic_s, *group_s = dynamic_s + table, *cell_s = group_s + table;
  const Place p = place_of<V>(g);
  Positions<T, V, Alone<T, V>, false> pos(x, nullptr, p, smem_addr(cell_s) + gn_scratch(g, true), g.held);
  pos.start_all();
  float4* cells = cell_s + threadIdx.x * Stats::M;
  if (p.count > 0) {
    Stats s;
    s.start(x + p.at);
    pos.as_they_come([&](const Vec<T, V>& w, const Nothing& k) { s(w, k); });
    s.finish(cells, p.count);
  } else {
    Stats::none(cells);
  }
  __syncthreads();
  join_block<V, Stats::M>(cell_s, p, g, [&](int j, const Part& q) { own_s[j] = make_float4(q.mean, q.m2, q.lo, q.hi); });
  if (g.chunks > 1) cluster_sync();
  else __syncthreads();
  const int g0 = p.g0, groups = (int)fast_div(p.width, g.by_cpg), L = lanes_for(g.chunks, groups), per = blockDim.x / L, member = threadIdx.x & (L - 1);
  for (int j0 = 0; j0 < groups; j0 += per) {
    const int j = j0 + threadIdx.x / L;
    const uint32_t own = smem_addr(own_s + (j < groups ? j : 0));
    const float4 st = stats_of(join_parts(j < groups ? g.chunks : 0, g, member, L, [&](int i) {
      const float4 q = peer_load4(own, i);
      return Part{q.x, q.y, q.z, q.w};
    }, [&](int i) { return run_rows(g.S, g.rows, i) * (float)g.cpg; }), g);
    if (j < groups && member == 0) {
      group_s[j] = st;
      keep_stats(stats, p, g, g0 + j, st);
    }
  }
  if (g.chunks > 1) cluster_arrive();                     // what was read of the others' tables is read
  __syncthreads();
  if (p.count > 0) apply_all<T, V, ONE, SAVE, true, false>(pos, group_s, p, g, gamma, beta, y, codes, kind);
  if (g.chunks > 1) cluster_wait();
}

// ------------------------------------------------------------------ backward
// h = line.x * kept + line.y, kept a code or the element less the mean
template <bool CODES> ACTNN_DEV float2 normal_line(const float4& st) {
  return CODES ? make_float2(code_step(st.w) * st.y, (st.z - st.x) * st.y) : make_float2(st.y, 0.f);
}
// z = za * kept + zb, and what is needed with it
template <typename T, int V, bool ONE, bool CODES> struct Line {
  using F = typename Many<V>::F;
  Row<V> za, zb;
  GroupRow<V, ONE> mean;                                  // less it
  ACTNN_DEV void start(const Place& p, const GnShape& g, const float* stats, const float* gamma, const float* beta) {
    float w[V], shift[V];
    parameters<V>(gamma, p.c, g.wide, 1.f, w);
    parameters<V>(beta, p.c, g.wide, 0.f, shift);
    float2 line;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i == 0 || !ONE) {
        const float4 st = stats_at(p, g, stats, i);
        line = normal_line<CODES>(st);
        mean.set(i, -st.x);
      }
      za.set(i, w[i] * line.x);
      zb.set(i, fmaf(w[i], line.y, shift[i]));
    }
  }
  static ACTNN_DEV float4 stats_at(const Place& p, const GnShape& g, const float* stats, int i) {
    return __ldg(reinterpret_cast<const float4*>(stats) + p.n * g.G + p.g0 + group_at(p, g, i));
  }
  ACTNN_DEV void kept(const typename Kept<T, V, CODES>::Words& k, F (&f)[Many<V>::N]) const {
    if constexpr (CODES) {
      unpack_codes<V>(k, f);
    } else {
      unpack_vec(k, f);
#pragma unroll
      for (int i = 0; i < Many<V>::N; ++i) f[i] = f_add(f[i], mean.at(i));
    }
  }
};
template <typename T, int V, bool ONE, int KIND, bool CODES> struct Sums {
  using F = typename Many<V>::F;
  static constexpr int N = Many<V>::N;
  const Line<T, V, ONE, CODES>& l;
  Row<V>&s1, &s2;                                         // of dz and of dz * kept
  ACTNN_DEV void operator()(const Vec<T, V>& w, const typename Kept<T, V, CODES>::Words& k) {
    F d[N], f[N];
    unpack_vec(w, d);
    l.kept(k, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const F dz = f_mul(d[i], act_slope<KIND, sizeof(T) == 4>(f_fma(f[i], l.za.f[i], l.zb.f[i])));
      s1.f[i] = f_add(s1.f[i], dz);
      s2.f[i] = f_fma(dz, f[i], s2.f[i]);
    }
  }
};
template <typename T, int V, bool ONE, int KIND, bool CODES> struct Grad {
  using F = typename Many<V>::F;
  static constexpr int N = Many<V>::N;
  const Line<T, V, ONE, CODES>& l;
  const Row<V>& k1;
  const GroupRow<V, ONE>&k2, &k3;
  T* dx;
  int64_t step;
  ACTNN_DEV void operator()(const Vec<T, V>& w, const typename Kept<T, V, CODES>::Words& k) {
    F d[N], f[N];
    unpack_vec(w, d);
    l.kept(k, f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const F dz = f_mul(d[i], act_slope<KIND, sizeof(T) == 4>(f_fma(f[i], l.za.f[i], l.zb.f[i])));
      d[i] = f_fma(dz, k1.f[i], f_fma(f[i], k2.at(i), k3.at(i)));
    }
    store_vec<T, V>(dx, d);
    dx += step;
  }
};

// The first half: the sums of the block's positions for each channel, over its threads in order: give(channel of the tile, sums of
// dz and of dz * h).  sum_s: a place for each thread and channel.
template <typename T, int V, bool ONE, bool CODES, bool HELD, bool SUMS, typename Give>
ACTNN_DEV void sums_all(Positions<T, V, Kept<T, V, CODES>, SUMS>& pos, const Line<T, V, ONE, CODES>& l, float2* sum_s, const Place& p,
                        const GnShape& g, const float* stats, int kind, Give give) {
  if (p.r < p.R) {
    Row<V> s1, s2;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s1.set(i, 0.f);
      s2.set(i, 0.f);
    }
    auto with = [&](auto take) {
      if constexpr (HELD) pos.as_they_come(take);
      else pos.through(take);
    };
    switch (kind) {
      case kActNone: with(Sums<T, V, ONE, kActNone, CODES>{l, s1, s2}); break;
      case kActRelu: with(Sums<T, V, ONE, kActRelu, CODES>{l, s1, s2}); break;
      case kActSilu: with(Sums<T, V, ONE, kActSilu, CODES>{l, s1, s2}); break;
      case kActGelu: with(Sums<T, V, ONE, kActGelu, CODES>{l, s1, s2}); break;
      default: with(Sums<T, V, ONE, kActGeluTanh, CODES>{l, s1, s2}); break;
    }
    float2 line;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i == 0 || !ONE) line = normal_line<CODES>(Line<T, V, ONE, CODES>::stats_at(p, g, stats, i));
      sum_s[p.r * p.width + (p.c - p.c0) + i] = make_float2(s1.get(i), fmaf(line.x, s2.get(i), line.y * s1.get(i)));
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
    float2 s = sum_s[c];
    for (int k = 1; k < p.R; ++k) s = f_add(s, sum_s[k * p.width + c]);
    give(c, s);
  }
}
// The second half: mean_s holds the means over the tile's groups of dz * gamma and of dz * gamma * h.
template <typename T, int V, bool ONE, bool CODES, bool HELD, bool SUMS>
ACTNN_DEV void grad_all(Positions<T, V, Kept<T, V, CODES>, SUMS>& pos, const Line<T, V, ONE, CODES>& l, const float4* mean_s, const Place& p,
                        const GnShape& g, const float* stats, const float* gamma, T* dx, int kind) {
  Row<V> k1;
  GroupRow<V, ONE> k2, k3;
  float w[V];
  parameters<V>(gamma, p.c, g.wide, 1.f, w);
  float4 st;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (i == 0 || !ONE) {
      st = Line<T, V, ONE, CODES>::stats_at(p, g, stats, i);
      const float2 line = normal_line<CODES>(st);
      const float4 m = mean_s[group_at(p, g, i)];
      k2.set(i, -st.y * m.y * line.x);
      k3.set(i, -st.y * fmaf(m.y, line.y, m.x));
    }
    k1.set(i, st.y * w[i]);
  }
  dx += p.at;
  auto with = [&](auto put) {
    if constexpr (HELD) pos.again(put);
    else pos.through(put);
  };
  switch (kind) {
    case kActNone: with(Grad<T, V, ONE, kActNone, CODES>{l, k1, k2, k3, dx, p.step}); break;
    case kActRelu: with(Grad<T, V, ONE, kActRelu, CODES>{l, k1, k2, k3, dx, p.step}); break;
    case kActSilu: with(Grad<T, V, ONE, kActSilu, CODES>{l, k1, k2, k3, dx, p.step}); break;
    case kActGelu: with(Grad<T, V, ONE, kActGelu, CODES>{l, k1, k2, k3, dx, p.step}); break;
    default: with(Grad<T, V, ONE, kActGeluTanh, CODES>{l, k1, k2, k3, dx, p.step}); break;
  }
}
// Means over a group from `runs` sets of its channels' sums, load(run, channel of the tile): mean_s[group of the tile].
template <typename Load>
ACTNN_DEV void group_means(float4* mean_s, const Place& p, const GnShape& g, const float* gamma, int runs, Load load) {
  const int groups = g.parts == 1 ? (int)fast_div(p.width, g.by_cpg) : 1, entries = runs * g.cpg;
  const int L = lanes_for(entries, groups), per = blockDim.x / L, member = threadIdx.x & (L - 1), gc0 = p.g0 * g.cpg;
  for (int j0 = 0; j0 < groups; j0 += per) {
    const int j = j0 + threadIdx.x / L;
    float a = 0.f, b = 0.f;
    for (int e = member; j < groups && e < entries; e += L) {
      const int k = (int)fast_div(e, g.by_cpg), c = gc0 + j * g.cpg + (e - k * g.cpg);
      const float2 s = load(k, c);
      const float w = gamma ? __ldg(gamma + c) : 1.f;
      a = fmaf(w, s.x, a);
      b = fmaf(w, s.y, b);
    }
    const float m = (float)g.S * (float)g.cpg;
    a = lanes_sum(a, L) / m;
    b = lanes_sum(b, L) / m;
    if (j < groups && member == 0) mean_s[j] = make_float4(a, b, 0.f, 0.f);
  }
}

// Two launches, the first.  sums[(n * chunks + chunk) * C + c].
template <typename T, int V, bool ONE, bool CODES>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_backward_sums_kernel(const T* __restrict__ dy, const void* __restrict__ kept, const float* __restrict__ stats,
                        const float* __restrict__ gamma, const float* __restrict__ beta, float2* __restrict__ sums, int kind,
                        const GnShape g) {
  extern __shared__ float4 dynamic_s[];                   // scratch, ring
  const Place p = place_of<V>(g);
  Positions<T, V, Kept<T, V, CODES>, true> pos(dy, kept, p, smem_addr(dynamic_s) + gn_scratch(g, false), Positions<T, V, Kept<T, V, CODES>, true>::kDepth);
  pos.start();
  float2* out = sums + (p.n * g.chunks + p.chunk) * g.C + p.c0;
  Line<T, V, ONE, CODES> l;
  if (p.r < p.R) l.start(p, g, stats, gamma, beta);
  sums_all<T, V, ONE, CODES, false, true>(pos, l, reinterpret_cast<float2*>(dynamic_s), p, g, stats, kind,
                                    [&](int c, float2 s) { out[c] = s; });
}
// The second.
template <typename T, int V, bool ONE, bool CODES>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_backward_kernel(const T* __restrict__ dy, const void* __restrict__ kept, const float* __restrict__ stats,
                   const float* __restrict__ gamma, const float* __restrict__ beta, const float2* __restrict__ sums,
                   T* __restrict__ dx, int kind, const GnShape g) {
  extern __shared__ float4 dynamic_s[];                   // tables, ring
  const Place p = place_of<V, true>(g);
  Positions<T, V, Kept<T, V, CODES>, false> pos(dy, kept, p, smem_addr(dynamic_s) + gn_tables(g), Positions<T, V, Kept<T, V, CODES>, false>::kDepth);
  pos.start();
  group_means(dynamic_s, p, g, gamma, g.first_chunks, [&](int k, int c) { return sums[(p.n * g.first_chunks + k) * g.C + c]; });
  __syncthreads();
  if (p.count == 0) return;
  Line<T, V, ONE, CODES> l;
  l.start(p, g, stats, gamma, beta);
  grad_all<T, V, ONE, CODES, false, false>(pos, l, dynamic_s, p, g, stats, gamma, dx, kind);
}
// One launch, a cluster of `chunks` blocks for each sample and run of channels (whole groups); the sums of each block are written
// for the gradients of the parameters.
template <typename T, int V, bool ONE, bool CODES>
__global__ void __launch_bounds__(kGnThreads, kGnResident<T>)
gn_backward_held_kernel(const T* __restrict__ dy, const void* __restrict__ kept, const float* __restrict__ stats,
                        const float* __restrict__ gamma, const float* __restrict__ beta, float2* __restrict__ sums,
                        T* __restrict__ dx, int kind, const GnShape g) {
  extern __shared__ float4 dynamic_s[];                   // tables (own sums, joined means), scratch, positions
  const int table = gn_groups(g);
  float4 *own_s = dynamic_s, *mean_s = dynamic_s + table;
  float2* sum_s = reinterpret_cast<float2*>(mean_s + table);
  const Place p = place_of<V>(g);
  Positions<T, V, Kept<T, V, CODES>, false> pos(dy, kept, p, smem_addr(sum_s) + gn_scratch(g, false), g.held);
  pos.start_all();
  float2* out = sums + (p.n * g.chunks + p.chunk) * g.C + p.c0;
  Line<T, V, ONE, CODES> l;
  if (p.r < p.R) l.start(p, g, stats, gamma, beta);
  sums_all<T, V, ONE, CODES, true, false>(pos, l, sum_s, p, g, stats, kind, [&](int c, float2 s) {
    out[c] = s;
    sum_s[c] = s;                                         // its own column alone was read for it
  });
  __syncthreads();
  group_means(own_s, p, g, gamma, 1, [&](int, int c) { return sum_s[c - p.c0]; });
  if (g.chunks > 1) cluster_sync();
  else __syncthreads();
  const int groups = (int)fast_div(p.width, g.by_cpg);
  for (int j = threadIdx.x; j < groups; j += blockDim.x) {
    float4 m = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < g.chunks; ++k) {
      const float4 q = peer_load4(smem_addr(own_s + j), k);
      m.x += q.x;
      m.y += q.y;
    }
    mean_s[j] = m;
  }
  if (g.chunks > 1) cluster_arrive();
  __syncthreads();
  if (p.count > 0) grad_all<T, V, ONE, CODES, true, false>(pos, l, mean_s, p, g, stats, gamma, dx, kind);
  if (g.chunks > 1) cluster_wait();
}

// Many runs: partial results joined once, in a launch between the two, instead of by every block of the second.  A warp per group.
__global__ void __launch_bounds__(kGnThreads)
gn_fold_parts_kernel(const Part* __restrict__ parts, Part* __restrict__ out, int64_t groups, const GnShape g) {
  const int64_t group = (int64_t)blockIdx.x * (kGnThreads / 32) + (threadIdx.x >> 5);
  if (group >= groups) return;
  const int count = g.first_chunks * g.first_parts, lane = threadIdx.x & 31;
  const Part* q = parts + group * count;
  const Part one = join_parts(count, g, lane, 32, [&](int i) { return q[i]; }, [&](int i) { return part_items(g, i); });
  if (lane == 0) out[group] = one;
}
// The sums of a sample's runs, a block for 8 channels.
__global__ void __launch_bounds__(kGnThreads)
gn_fold_sums_kernel(const float2* __restrict__ sums, float2* __restrict__ out, int runs, int C, int blocks) {
  __shared__ float2 part_s[kGnThreads / 32][8];
  const int64_t n = blockIdx.x / blocks;
  const int col = threadIdx.x & 7, c = (int)(blockIdx.x - n * blocks) * 8 + col;
  float2 s = make_float2(0.f, 0.f);
  if (c < C) {
#pragma unroll 4
    for (int k = threadIdx.x >> 3; k < runs; k += kGnThreads / 8) s = f_add(s, __ldg(sums + (n * runs + k) * C + c));
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) s = f_add(s, make_float2(__shfl_xor_sync(kFull, s.x, o), __shfl_xor_sync(kFull, s.y, o)));
  if ((threadIdx.x & 31) < 8) part_s[threadIdx.x >> 5][col] = s;
  __syncthreads();
  if (threadIdx.x < 8 && c < C) {
    s = part_s[0][col];
    for (int k = 1; k < kGnThreads / 32; ++k) s = f_add(s, part_s[k][col]);
    out[n * C + c] = s;
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
// What a block of each kernel does besides its positions, in positions of a thread.
constexpr int kExtraStats = 14, kExtraSums = 8, kExtraSecond = 6;
// Partial results of a group that every block of the second launch joins for itself; more of them are folded before it.
constexpr int kFold = 8;

inline int gn_threads(const GnShape& g) {
  const int vecs = g.tile / g.V, R = kGnThreads / vecs;
  return (vecs * R + 31) / 32 * 32;
}
// KERNEL's limit of dynamic shared memory, raised to what any call may ask for, once on a device.
template <auto KERNEL> bool gn_raise() {
  static std::atomic<uint64_t> raised{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (raised.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, kGnMostSmem) != cudaSuccess) return false;
  raised.fetch_or(bit, std::memory_order_release);
  return true;
}
template <auto KERNEL, typename... Args> bool gn_start(const GnCall& c, const GnShape& g, int smem, Args... args) {
  if (!gn_raise<KERNEL>()) return false;
  if (c.N * g.chunks * g.tiles > 0x7fffffff) return false;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(c.N * g.chunks * g.tiles));
  cfg.blockDim = dim3((unsigned)gn_threads(g));
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = c.stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = g.held ? (unsigned)g.chunks : 1u;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, KERNEL, args...) == cudaSuccess;
}
// The cut of one of two launches of KERNEL, by the blocks of 256 threads that an SM holds of it with `smem` bytes each.  The last
// answer is kept with its question (bytes in the upper half, blocks in the lower one); one that failed is not.
template <auto KERNEL> void gn_cut_for(GnShape& g, int64_t N, int smem, int extra) {
  static std::atomic<uint64_t> answer{0};
  const uint64_t kept = answer.load(std::memory_order_acquire);
  int n = (int)(uint32_t)kept;
  if (n == 0 || (int)(kept >> 32) != smem) {
    if (gn_raise<KERNEL>() && cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, kGnThreads, smem) == cudaSuccess && n > 0) {
      answer.store((uint64_t)smem << 32 | (uint32_t)n, std::memory_order_release);
    } else {
      cudaGetLastError();
      n = 1;
    }
  }
  gn_cut_positions(g, N, (int64_t)device_info().sm_count * n, extra);
}

template <typename T, int V, bool ONE, bool SAVE> bool gn_forward(const GnCall& c, const GnShape& g) {
  using Pos = Positions<T, V, Alone<T, V>, false>;
  using Pos1 = Positions<T, V, Alone<T, V>, true>;
  const T* x = (const T*)c.x;
  Part* parts = (Part*)c.workspace;
  if constexpr (Pos::kAsync) {
    if (g.held)
      return gn_start<gn_forward_held_kernel<T, V, ONE, SAVE>>(c, g, gn_tables(g) + gn_scratch(g, true) + g.held * Pos::kPlace, x, c.gamma, c.beta,
                                                               (T*)c.out, c.codes, c.stats, c.kind, g);
  }
  GnShape first = g, second = g;
  const int smem1 = gn_scratch(g, true) + Pos1::kDepth * Pos1::kPlace, smem2 = gn_tables(g) + Pos::kDepth * Pos::kPlace;
  gn_cut_for<gn_stats_kernel<T, V, ONE>>(first, c.N, smem1, kExtraStats);
  gn_cut_for<gn_forward_kernel<T, V, ONE, SAVE>>(second, c.N, smem2, kExtraSecond);
  second.first_chunks = first.first_chunks = first.chunks;
  second.first_parts = first.first_parts = g.parts;
  second.first_rows = first.first_rows = first.rows;
  if (!gn_start<gn_stats_kernel<T, V, ONE>>(c, first, smem1, x, parts, first)) return false;
  if (first.chunks * g.parts > kFold) {
    const int64_t groups = c.N * g.G, blocks = (groups + kGnThreads / 32 - 1) / (kGnThreads / 32);
    Part* joined = parts + groups * first.chunks * g.parts;
    if (blocks > 0x7fffffff) return false;
    gn_fold_parts_kernel<<<(unsigned)blocks, kGnThreads, 0, c.stream>>>(parts, joined, groups, first);
    parts = joined;
    second.first_chunks = second.first_parts = 1;
    second.first_rows = g.S;
  }
  return gn_start<gn_forward_kernel<T, V, ONE, SAVE>>(c, second, smem2, x, (const Part*)parts, c.gamma, c.beta, (T*)c.out, c.codes, c.stats,
                                                      c.kind, second);
}
template <typename T, int V, bool ONE, bool CODES> bool gn_backward(const GnCall& c, const GnShape& g) {
  using Pos = Positions<T, V, Kept<T, V, CODES>, false>;
  using Pos1 = Positions<T, V, Kept<T, V, CODES>, true>;
  const T* dy = (const T*)c.dy;
  const void* kept = CODES ? (const void*)c.codes : c.x;
  const float* stats = c.stats;
  float2* sums = (float2*)c.workspace;
  bool ok;
  GnShape first = g, second = g;
  if (g.held) {
    if constexpr (Pos::kAsync)
      ok = gn_start<gn_backward_held_kernel<T, V, ONE, CODES>>(c, g, gn_tables(g) + gn_scratch(g, false) + g.held * Pos::kPlace, dy, kept, stats,
                                                              c.gamma, c.beta, sums, (T*)c.out, c.kind, g);
    else
      ok = false;
  } else {
    const int smem1 = gn_scratch(g, false) + Pos1::kDepth * Pos1::kPlace, smem2 = gn_tables(g) + Pos::kDepth * Pos::kPlace;
    gn_cut_for<gn_backward_sums_kernel<T, V, ONE, CODES>>(first, c.N, smem1, kExtraSums);
    gn_cut_for<gn_backward_kernel<T, V, ONE, CODES>>(second, c.N, smem2, kExtraSecond);
    second.first_chunks = first.chunks;
    ok = gn_start<gn_backward_sums_kernel<T, V, ONE, CODES>>(c, first, smem1, dy, kept, stats, c.gamma, c.beta, sums, c.kind, first);
    if (ok && first.chunks > kFold) {
      const int per = (g.C + 7) / 8;
      float2* joined = sums + c.N * first.chunks * g.C;
      if (c.N * per > 0x7fffffff) return false;
      gn_fold_sums_kernel<<<(unsigned)(c.N * per), kGnThreads, 0, c.stream>>>(sums, joined, first.chunks, g.C, per);
      sums = joined;
      second.first_chunks = first.chunks = 1;
    }
    ok = ok && gn_start<gn_backward_kernel<T, V, ONE, CODES>>(c, second, smem2, dy, kept, stats, c.gamma, c.beta, (const float2*)sums, (T*)c.out,
                                                       c.kind, second);
  }
  if (ok && (c.dgamma || c.dbeta))
    gn_column_sums_kernel<<<(g.C + 7) / 8, 1024, 0, c.stream>>>(sums, c.dgamma, c.dbeta, c.N * first.chunks, g.C);
  return ok;
}
template <typename T, int V, bool ONE> bool gn_one(const GnCall& c, const GnShape& g, bool forward) {
  if (forward) return c.codes ? gn_forward<T, V, ONE, true>(c, g) : gn_forward<T, V, ONE, false>(c, g);
  return c.codes ? gn_backward<T, V, ONE, true>(c, g) : gn_backward<T, V, ONE, false>(c, g);
}
template <typename T> int gn_run(const GnCall& c, const GnShape& g, bool forward) {
  const bool one = g.cpg % g.V == 0;
  bool ok;
  if (g.V == 8) {
    if constexpr (sizeof(T) == 2) ok = one ? gn_one<T, 8, true>(c, g, forward) : gn_one<T, 8, false>(c, g, forward);
    else ok = false;                                      // 16 bytes of a float32 row are four channels
  } else if (g.V == 4) {
    ok = one ? gn_one<T, 4, true>(c, g, forward) : gn_one<T, 4, false>(c, g, forward);
  } else if (g.V == 2) {
    ok = one ? gn_one<T, 2, true>(c, g, forward) : gn_one<T, 2, false>(c, g, forward);
  } else {
    ok = gn_one<T, 1, true>(c, g, forward);
  }
  if (!ok) {
    cudaGetLastError();
    return ACTNN_ERR_LAUNCH;
  }
  return check_launch();
}

}  // namespace
}  // namespace actnn
