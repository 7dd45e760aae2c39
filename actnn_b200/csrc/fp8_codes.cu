// Codes of matrices for the product in 8-bit floating point (fp8.cuh): of rows alone, of rows and columns at once, of squares.
//
// A layer's three products reduce over input channels, output channels and tokens, and each wants its operands coded in blocks along
// its own reduction.  What is read once is coded both ways: tokens along their channels for the product they enter, and along the
// tokens, transposed, for the gradient of the weight.  A weight is coded in squares, whose codes are the same either way.
// Bound by HBM, 2 + 1 bytes an element one way, 2 + 2 both ways, and by instructions: 16384 x 4096 bf16 by rows 37 us (31 at the copy
// rate); 8192 x 6144 both ways, as two matrices, 45 (31); 4096 x 2048 in squares, both ways, 8.5 (5).
#include "cluster.cuh"
#include "fp8.cuh"

namespace actnn {
namespace {

constexpr int kCodeThreads = 256;

// A warp has 512 elements of a row, two vectors a lane, TASKS times; half a warp and a vector are a block.
template <typename T, bool VEC, int TASKS>
__global__ void __launch_bounds__(kCodeThreads)
fp8_row_codes_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t rows, int64_t cols,
                     int64_t ldx, int64_t ldc, int groups) {
  const int lane = threadIdx.x & 31;
  const int64_t first = ((int64_t)blockIdx.x * (kCodeThreads / 32) + (threadIdx.x >> 5)) * TASKS;
  grid_release();                                      // of the product that may follow: it waits for the end of this launch itself
  int64_t row[TASKS];
  int g[TASKS];
  Vec<T, 8> v[TASKS][2];
#pragma unroll
  for (int i = 0; i < TASKS; ++i) {
    row[i] = (first + i) / groups;
    g[i] = (int)(first + i - row[i] * groups);
#pragma unroll
    for (int k = 0; k < 2; ++k) v[i][k] = fp8_load<T, VEC>(x + row[i] * ldx, g[i] * 512 + k * 256 + lane * 8, row[i] < rows ? cols : 0);
  }
#pragma unroll
  for (int i = 0; i < TASKS; ++i) {
    if (row[i] >= rows) return;
    uint32_t byte[2];
    fp8_block_bits(v[i][0], v[i][1], byte);
    uint8_t* to = codes + row[i] * ldc + g[i] * 512 + lane * 8;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      byte[k] = fp8_scale_byte(byte[k]);
      if (g[i] * 512 + k * 256 + lane * 8 < ldc) *reinterpret_cast<uint2*>(to + k * 256) = fp8_codes8(v[i][k], fp8_factor(byte[k]));
    }
    const uint32_t mine = byte[0] | byte[1] << 16, other = __shfl_xor_sync(kFull, mine, 16);
    if (lane == 0) *reinterpret_cast<uint32_t*>(scales + fp8_scale_at(row[i], g[i] * 4, (rows + 127) / 128)) = mine | other << 8;
  }
}

// Elements of a word of columns, and the bits of float32 of one of its magnitudes.
template <typename T> constexpr int word_columns() { return 4 / (int)sizeof(T); }
template <typename T> ACTNN_DEV uint32_t word_bits(uint32_t w, int which) {
  const float2 f = pair_to_float(w, T());
  return __float_as_uint(which ? f.y : f.x);
}
template <> ACTNN_DEV uint32_t word_bits<float>(uint32_t w, int) { return w; }
// Columns 2 j and 2 j + 1 of a vector.
template <typename T> ACTNN_DEV float2 column_pair(const Vec<T, 8>& v, int j) { return pair_to_float(v.w[j], T()); }
template <> ACTNN_DEV float2 column_pair<float>(const Vec<float, 8>& v, int j) {
  return make_float2(__uint_as_float(v.w[2 * j]), __uint_as_float(v.w[2 * j + 1]));
}

// A tile of 128 x 128: a thread has eight neighbouring columns of eight neighbouring rows.  SQUARE: one scale for the tile.
// codes, codes_t and parts may be NULL; parts [tiles of rows][cols] are the sums of the tile's columns.  Registers are what bounds the
// loads under way: three blocks an SM hold 96 KB of a 16-bit type.  What is not finite is looked for once in a warp's part and set aside, so that
// nothing below asks again (a test for every row and word: 208 instructions a vector, 59 us where 45 are taken now).
template <typename T, bool VEC, bool SQUARE>
__global__ void __launch_bounds__(kCodeThreads, sizeof(T) == 4 ? 2 : 3)
fp8_tile_codes_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, uint8_t* __restrict__ codes_t,
                      uint8_t* __restrict__ scales_t, float* __restrict__ parts, int64_t rows, int64_t cols, int64_t ldx, int64_t ldc,
                      int64_t ldt, int column_tiles) {
  constexpr int kWords = 8 / word_columns<T>();
  const int64_t row_tiles = (rows + 127) / 128;
  __shared__ uint4 turned_s[128 * 8];                  // [column][128 rows], chunks of eight rows in the order rotated by column / 8
  __shared__ __align__(16) uint32_t most_s[16][128];                 // [team][word of columns]; later float sums of columns
  __shared__ __align__(16) float factor_s[128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c8 = lane & 15, team = warp * 2 + (lane >> 4);
  const int64_t tr = blockIdx.x / column_tiles, tc = blockIdx.x - tr * column_tiles, r0 = tr * 128 + team * 8, c = tc * 128 + c8 * 8;
  Vec<T, 8> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fp8_load<T, VEC>(x + (r0 + i) * ldx, c, r0 + i < rows ? cols : 0);

  // ---- sums of columns
  float2 sum[4] = {};
  if (parts) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = f_add(sum[j], column_pair(v[i], j));
  }

  // ---- the largest magnitudes of the thread's rows and columns, as words; what is not finite does not count, and is made NaN
  uint32_t of_row[8], most[kWords] = {}, any = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    of_row[i] = fp8_words_most(v[i]);
    any = fp8_word_max<T>(any, of_row[i]);
#pragma unroll
    for (int j = 0; j < kWords; ++j) most[j] = fp8_word_max<T>(most[j], fp8_word_abs<T>(v[i].w[j]));
  }
  if (__any_sync(kFull, fp8_word_bad<T>(any))) {
    any = 0;
#pragma unroll
    for (int j = 0; j < kWords; ++j) most[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      of_row[i] = 0;
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        const uint32_t w = fp8_word_abs<T>(fp8_word_finite<T>(v[i].w[j]));
        of_row[i] = fp8_word_max<T>(of_row[i], w);
        most[j] = fp8_word_max<T>(most[j], w);
        v[i].w[j] = fp8_word_nan<T>(v[i].w[j]);
      }
      any = fp8_word_max<T>(any, of_row[i]);
    }
  }
  uint32_t square = 0;
  if (SQUARE) {
    square = __reduce_max_sync(kFull, max(word_bits<T>(any, 0), word_bits<T>(any, 1)));
    if (lane == 0) most_s[0][warp] = square;
    __syncthreads();
    square = most_s[0][0];
#pragma unroll
    for (int w = 1; w < kCodeThreads / 32; ++w) square = max(square, most_s[0][w]);
    square = fp8_scale_byte(square);
  }

  // ---- rows, two at a time
  if (codes) {
    const int left = (int)min((int64_t)8, rows - r0);   // rows that there are
    uint8_t *to = codes + r0 * ldc + c, *to_s = scales + fp8_scale_at(r0, tc, row_tiles);          // eight rows lie 16 bytes apart
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      uint32_t byte[2] = {square, square};
      if (!SQUARE) {
        fp8_half_warp<T>(of_row[i], of_row[i + 1], byte);
        byte[0] = fp8_scale_byte(byte[0]), byte[1] = fp8_scale_byte(byte[1]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint2 q = fp8_codes8(v[i + k], fp8_factor(byte[k]));
        if (i + k < left && c < ldc) *reinterpret_cast<uint2*>(to + (i + k) * ldc) = q;
        if (i + k < left && c8 == 0) to_s[16 * (i + k)] = (uint8_t)byte[k];
      }
    }
  }

  // ---- columns
  if (codes_t) {
    if (!SQUARE) {
#pragma unroll
      for (int j = 0; j < kWords; ++j) most_s[team][c8 * kWords + j] = most[j];
      __syncthreads();
      if (threadIdx.x < 128) {
        const int word = threadIdx.x / word_columns<T>();
        uint32_t all = most_s[0][word];
#pragma unroll
        for (int k = 1; k < 16; ++k) all = fp8_word_max<T>(all, most_s[k][word]);
        const uint32_t byte = fp8_scale_byte(word_bits<T>(all, threadIdx.x % word_columns<T>()));
        factor_s[threadIdx.x] = fp8_factor(byte);
        if (tc * 128 + threadIdx.x < cols) scales_t[fp8_scale_at(tc * 128 + threadIdx.x, tr, column_tiles)] = (uint8_t)byte;
      }
      __syncthreads();
    } else if (threadIdx.x < 128 && tc * 128 + threadIdx.x < cols) {
      scales_t[fp8_scale_at(tc * 128 + threadIdx.x, tr, column_tiles)] = (uint8_t)square;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 by = SQUARE ? make_float2(fp8_factor(square), fp8_factor(square)) : *reinterpret_cast<const float2*>(&factor_s[c8 * 8 + 2 * j]);
      uint32_t px[4], py[4];                           // two rows each
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float2 a = f_mul(column_pair(v[i], j), by), b = f_mul(column_pair(v[i + 1], j), by);
        px[i / 2] = fp8_pair(a.x, b.x);
        py[i / 2] = fp8_pair(a.y, b.y);
      }
      uint2* at = reinterpret_cast<uint2*>(turned_s) + (c8 * 8 + 2 * j) * 16 + (team ^ c8);
      at[0] = make_uint2(px[0] | px[1] << 16, px[2] | px[3] << 16);
      at[16] = make_uint2(py[0] | py[1] << 16, py[2] | py[3] << 16);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int column = k * 32 + (threadIdx.x >> 3), s = column >> 3 & 15, q = threadIdx.x & 7;     // rows 16 q on
      uint4 w = turned_s[column * 8 + (q ^ (s >> 1))];
      if (s & 1) w = make_uint4(w.z, w.w, w.x, w.y);
      const int64_t row = tr * 128 + q * 16;
      if (tc * 128 + column < cols && row < ldt) *reinterpret_cast<uint4*>(codes_t + (tc * 128 + column) * ldt + row) = w;
    }
  }

  if (parts) {
    __syncthreads();
    float* sum_s = reinterpret_cast<float*>(most_s);
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(&sum_s[team * 128 + c8 * 8 + 2 * j]) = sum[j];
    __syncthreads();
    if (threadIdx.x < 128 && tc * 128 + threadIdx.x < cols) {
      float s = sum_s[threadIdx.x];
#pragma unroll
      for (int k = 1; k < 16; ++k) s += sum_s[k * 128 + threadIdx.x];
      parts[tr * cols + tc * 128 + threadIdx.x] = s;
    }
  }
}

// The sums over the rows of parts [runs, cols], in a fixed order: a block has 32 columns, eight threads a column.
template <typename T>
__global__ void __launch_bounds__(kCodeThreads) fp8_join_kernel(const float* __restrict__ parts, T* __restrict__ out, int64_t runs, int64_t cols) {
  __shared__ float part_s[kCodeThreads / 32][32];
  const int way = threadIdx.x >> 5;
  const int64_t column = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  float s = 0.f;
  if (column < cols) {
#pragma unroll 4
    for (int64_t k = way; k < runs; k += kCodeThreads / 32) s += __ldg(parts + k * cols + column);
  }
  part_s[way][threadIdx.x & 31] = s;
  __syncthreads();
  if (way == 0 && column < cols) {
#pragma unroll
    for (int w = 1; w < kCodeThreads / 32; ++w) s += part_s[w][threadIdx.x];
    out[column] = from_float<T>(s);
  }
}

// code * 2^e, eight elements a thread.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kCodeThreads)
fp8_decode_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, int64_t rows, int64_t cols,
                  int64_t ldc, int64_t octs) {
  const int64_t i = (int64_t)blockIdx.x * kCodeThreads + threadIdx.x, row = i / octs, e = (i - row * octs) * 8;
  if (row >= rows) return;
  const float s = fp8_scale(__ldg(scales + fp8_scale_at(row, e / kFpBlock, (rows + 127) / 128)));
  const uint8_t* p = codes + row * ldc + e;
  float2 f[4];
  if constexpr (VEC) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    f[0] = fp8_unpack(w.x & 0xffff), f[1] = fp8_unpack(w.x >> 16), f[2] = fp8_unpack(w.y & 0xffff), f[3] = fp8_unpack(w.y >> 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = f_mul(f[j], make_float2(s, s));
    store_vec<T, 8>(out + row * cols + e, f);
  } else {
    for (int j = 0; j < 8 && e + j < cols; ++j) out[row * cols + e + j] = from_float<T>(fp8_unpack(load_one(p + j)).x * s);
  }
}

template <typename T>
int row_codes(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, int64_t ldx, int64_t ldc, cudaStream_t s) {
  const int64_t groups = (cols + 511) / 512, tasks = rows * groups;
  const int each = tasks >= (int64_t)device_info().sm_count * 256 ? 2 : 1;
  const int64_t grid = (tasks + kCodeThreads / 32 * each - 1) / (kCodeThreads / 32 * each);
  if (grid > 0x7fffffff) return ACTNN_ERR_SHAPE;
  const bool vec = cols % 8 == 0 && (ldx % 8 == 0 || rows == 1) && aligned(x, 16);
  auto* kernel = vec ? (each == 2 ? fp8_row_codes_kernel<T, true, 2> : fp8_row_codes_kernel<T, true, 1>)
                     : (each == 2 ? fp8_row_codes_kernel<T, false, 2> : fp8_row_codes_kernel<T, false, 1>);
  kernel<<<(unsigned)grid, kCodeThreads, 0, s>>>((const T*)x, codes, scales, rows, cols, ldx, ldc, (int)groups);
  return check_launch();
}
template <typename T>
int tile_codes(const void* x, uint8_t* codes, uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, float* parts, int64_t rows, int64_t cols,
               int64_t ldx, int64_t ldc, int64_t ldt, bool square, cudaStream_t s) {
  const int64_t column_tiles = (cols + 127) / 128, grid = (rows + 127) / 128 * column_tiles;
  if (grid > 0x7fffffff) return ACTNN_ERR_SHAPE;
  const bool vec = cols % 8 == 0 && (ldx % 8 == 0 || rows == 1) && aligned(x, 16);
  auto* kernel = vec ? (square ? fp8_tile_codes_kernel<T, true, true> : fp8_tile_codes_kernel<T, true, false>)
                     : (square ? fp8_tile_codes_kernel<T, false, true> : fp8_tile_codes_kernel<T, false, false>);
  kernel<<<(unsigned)grid, kCodeThreads, 0, s>>>((const T*)x, codes, scales, codes_t, scales_t, parts, rows, cols, ldx, ldc, ldt, (int)column_tiles);
  return check_launch();
}
template <typename T>
int decode(const uint8_t* codes, const uint8_t* scales, void* out, int64_t rows, int64_t cols, int64_t ldc, cudaStream_t s) {
  const int64_t octs = (cols + 7) / 8, grid = (rows * octs + kCodeThreads - 1) / kCodeThreads;
  if (grid > 0x7fffffff) return ACTNN_ERR_SHAPE;
  auto* kernel = cols % 8 == 0 && ldc % 8 == 0 && aligned(codes, 8) && aligned(out, 16) ? fp8_decode_kernel<T, true> : fp8_decode_kernel<T, false>;
  kernel<<<(unsigned)grid, kCodeThreads, 0, s>>>(codes, scales, (T*)out, rows, cols, ldc, octs);
  return check_launch();
}
bool bad_shape(int64_t rows, int64_t cols) { return rows < 0 || cols < 0 || cols > ((int64_t)1 << 31) || rows > ((int64_t)1 << 31); }
bool bad_row(int64_t ldc, int64_t cols) { return ldc < cols || ldc % 16 != 0 || ldc - cols >= 16; }

}  // namespace
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_fp8_row_codes(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, int64_t ldx, int64_t ldc,
                                   int dtype, actnn_stream_t stream) {
  if (bad_shape(rows, cols) || (rows > 1 && ldx < cols) || bad_row(ldc, cols)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (rows == 0 || cols == 0) return ACTNN_OK;
  if (!x || !codes || !scales) return ACTNN_ERR_NULL;
  if (!aligned(x, dtype_size(dtype)) || !aligned(codes, 16) || !aligned(scales, 16)) return ACTNN_ERR_ALIGN;
  switch (dtype) {
    case ACTNN_F32: return row_codes<float>(x, codes, scales, rows, cols, ldx, ldc, (cudaStream_t)stream);
    case ACTNN_F16: return row_codes<__half>(x, codes, scales, rows, cols, ldx, ldc, (cudaStream_t)stream);
    default: return row_codes<__nv_bfloat16>(x, codes, scales, rows, cols, ldx, ldc, (cudaStream_t)stream);
  }
}

extern "C" int actnn_fp8_tile_codes(const void* x, uint8_t* codes, uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, float* parts,
                                    int64_t rows, int64_t cols, int64_t ldx, int64_t ldc, int64_t ldt, int square, int dtype,
                                    actnn_stream_t stream) {
  if (bad_shape(rows, cols) || (rows > 1 && ldx < cols) || (codes && bad_row(ldc, cols)) || (codes_t && bad_row(ldt, rows))) return ACTNN_ERR_SHAPE;
  if (square < 0 || square > 1) return ACTNN_ERR_ARG;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (rows == 0 || cols == 0) return ACTNN_OK;
  if (!x || (!codes && !codes_t && !parts) || (codes && !scales) || (codes_t && !scales_t)) return ACTNN_ERR_NULL;
  if (!aligned(x, dtype_size(dtype)) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(codes_t, 16) || !aligned(scales_t, 16) ||
      !aligned(parts, 4)) return ACTNN_ERR_ALIGN;
  const cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case ACTNN_F32: return tile_codes<float>(x, codes, scales, codes_t, scales_t, parts, rows, cols, ldx, ldc, ldt, square, s);
    case ACTNN_F16: return tile_codes<__half>(x, codes, scales, codes_t, scales_t, parts, rows, cols, ldx, ldc, ldt, square, s);
    default: return tile_codes<__nv_bfloat16>(x, codes, scales, codes_t, scales_t, parts, rows, cols, ldx, ldc, ldt, square, s);
  }
}

extern "C" int actnn_fp8_join_sums(const float* parts, void* out, int64_t runs, int64_t cols, int dtype, actnn_stream_t stream) {
  if (bad_shape(runs, cols)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (cols == 0) return ACTNN_OK;
  if (!out || (runs > 0 && !parts)) return ACTNN_ERR_NULL;
  if (!aligned(out, dtype_size(dtype)) || !aligned(parts, 4)) return ACTNN_ERR_ALIGN;
  const unsigned grid = (unsigned)((cols + 31) / 32);
  const cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case ACTNN_F32: fp8_join_kernel<float><<<grid, kCodeThreads, 0, s>>>(parts, (float*)out, runs, cols); break;
    case ACTNN_F16: fp8_join_kernel<__half><<<grid, kCodeThreads, 0, s>>>(parts, (__half*)out, runs, cols); break;
    default: fp8_join_kernel<__nv_bfloat16><<<grid, kCodeThreads, 0, s>>>(parts, (__nv_bfloat16*)out, runs, cols); break;
  }
  return check_launch();
}

extern "C" int actnn_fp8_decode(const uint8_t* codes, const uint8_t* scales, void* out, int64_t rows, int64_t cols, int64_t ldc, int dtype,
                                actnn_stream_t stream) {
  if (bad_shape(rows, cols) || (rows > 1 && ldc < cols)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (rows == 0 || cols == 0) return ACTNN_OK;
  if (!codes || !scales || !out) return ACTNN_ERR_NULL;
  if (!aligned(out, dtype_size(dtype))) return ACTNN_ERR_ALIGN;
  switch (dtype) {
    case ACTNN_F32: return decode<float>(codes, scales, out, rows, cols, ldc, (cudaStream_t)stream);
    case ACTNN_F16: return decode<__half>(codes, scales, out, rows, cols, ldc, (cudaStream_t)stream);
    default: return decode<__nv_bfloat16>(codes, scales, out, rows, cols, ldc, (cudaStream_t)stream);
  }
}
