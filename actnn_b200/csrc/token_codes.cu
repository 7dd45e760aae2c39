// 8-bit codes of rows (tokens, or output channels of a weight): one scale a row.
//
//   a = max |x|,  scale = a * (1 / 127),  code = rint(x * (127 * (1 / a)))
//
// And the column sums that a bias's gradient is.
//
// A row is read once where the threads that share it can hold it in registers (up to 32 elements each), else twice, the
// second time from the L2.  Bound by HBM: 2 + 1 bytes an element of a 16-bit type; 16384 x 4096 bfloat16 take 30.7 us, the copy
// rate (one block a row, a quarter of its registers idle: 48), 8192 x 2048 8.6, rows that no vector fits 12.9.
#include "activation.cuh"
#include "cluster.cuh"

namespace actnn {
namespace {

constexpr int kRowThreads = 256;
constexpr int kHeld = 4;                               // vectors of eight that a thread holds

// The largest of `most` over the LANES threads of a row; every thread of the block takes part.
template <int LANES> ACTNN_DEV uint32_t row_max(uint32_t most) {
  most = __reduce_max_sync(kFull, most);
  if constexpr (LANES > 32) {
    __shared__ uint32_t warp_most[kRowThreads / 32];
    if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = most;
    __syncthreads();
    const int first = threadIdx.x / LANES * (LANES / 32);
    most = warp_most[first];
#pragma unroll
    for (int i = 1; i < LANES / 32; ++i) most = max(most, warp_most[first + i]);
  }
  return most;
}

// VEC: rows of x are whole aligned vectors of eight.  codes: rows `ldc` bytes apart (a multiple of 8), zero from cols to ldc.
template <typename T, int LANES, bool VEC>
__global__ void __launch_bounds__(kRowThreads)
row_codes_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, float* __restrict__ scale, int64_t rows, int64_t cols,
                 int64_t ldx, int64_t ldc) {
  const int lane = threadIdx.x % LANES;
  const int64_t mine = (int64_t)blockIdx.x * (kRowThreads / LANES) + threadIdx.x / LANES;
  const bool in = mine < rows;
  const int64_t row = in ? mine : rows - 1;            // threads without a row do the last one again, and write nothing
  grid_release();                                      // of the product that may follow: it waits for the end of this launch itself
  const T* p = x + row * ldx;
  int8_t* q = codes + row * ldc;
  Vec<T, 8> held[kHeld];
  auto load = [&](int64_t e) {
    if (VEC && e < cols) return load_vec<T, 8>(p + e);
    Vec<T, 8> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(v.w)[i] = !VEC && e + i < cols ? __ldg(p + e + i) : from_float<T>(0.f);
    return v;
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k) held[k] = load((int64_t)(k * LANES + lane) * 8);
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) most = max(most, most_of(held[k]));
  for (int64_t e = (int64_t)(kHeld * LANES + lane) * 8; e < cols; e += LANES * 8) most = max(most, most_of(load(e)));
  const float a = largest(row_max<LANES>(most));
  const float inv = code_factor(a);
  if (!in) return;
  if (lane == 0) scale[row] = code_step(a);
  auto store = [&](int64_t e, const Vec<T, 8>& v) {
    float2 f[4];
    unpack_vec(v, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = code_bits(f[i], make_float2(inv, inv));
    store_codes<8>(q + e, f);
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const int64_t e = (int64_t)(k * LANES + lane) * 8;
    if (e < ldc) store(e, held[k]);
  }
  for (int64_t e = (int64_t)(kHeld * LANES + lane) * 8; e < ldc; e += LANES * 8) store(e, load(e));
}

// code * scale, eight elements a thread.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads)
row_decode_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scale, T* __restrict__ out, int64_t rows, int64_t cols,
                  int64_t ldc, int64_t octs) {
  const int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  const int64_t row = i / octs, e = (i - row * octs) * 8;
  if (row >= rows) return;
  const float s = __ldg(scale + row);
  if constexpr (VEC) {
    float2 f[4];
    unpack_codes(load_codes<8>(codes + row * ldc + e), f);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = f_mul(f[j], make_float2(s, s));
    store_vec<T, 8>(out + row * cols + e, f);
  } else {
    for (int j = 0; j < 8 && e + j < cols; ++j) out[row * cols + e + j] = from_float<T>((float)codes[row * ldc + e + j] * s);
  }
}

// Column sums of x [rows, cols]: a block takes 64 columns of a run of rows (8 threads of 8 columns, 32 rows at a time), the
// second launch adds the runs in order.  VEC: rows are whole aligned vectors.
constexpr int kSumColumns = 64;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads)
column_sums_kernel(const T* __restrict__ x, float* __restrict__ parts, int64_t rows, int64_t cols, int64_t run) {
  __shared__ float2 part_s[kRowThreads / 32][8][4];
  const int64_t blocks = (cols + kSumColumns - 1) / kSumColumns, k = blockIdx.x / blocks;
  const int v = threadIdx.x & 7;
  const int64_t c = (blockIdx.x - k * blocks) * kSumColumns + v * 8, end = min(rows, (k + 1) * run);
  float2 s[4] = {};
  if (c < cols) {
#pragma unroll 4
    for (int64_t r = k * run + (threadIdx.x >> 3); r < end; r += kRowThreads / 8) {
      const T* p = x + r * cols + c;
      Vec<T, 8> w;
      if constexpr (VEC) {
        w = load_vec<T, 8>(p);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(w.w)[i] = c + i < cols ? __ldg(p + i) : from_float<T>(0.f);
      }
      float2 f[4];
      unpack_vec(w, f);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = f_add(s[i], f[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) s[i] = f_add(s[i], make_float2(__shfl_xor_sync(kFull, s[i].x, o), __shfl_xor_sync(kFull, s[i].y, o)));
    if ((threadIdx.x & 31) < 8) part_s[threadIdx.x >> 5][v][i] = s[i];
  }
  __syncthreads();
  if (threadIdx.x < 32) {                               // thread: pair i of vector q
    const int q = threadIdx.x >> 2, i = threadIdx.x & 3;
    float2 sum = part_s[0][q][i];
    for (int w = 1; w < kRowThreads / 32; ++w) sum = f_add(sum, part_s[w][q][i]);
    const int64_t to = (blockIdx.x - k * blocks) * kSumColumns + q * 8 + 2 * i;
    if (to < cols) parts[k * cols + to] = sum.x;
    if (to + 1 < cols) parts[k * cols + to + 1] = sum.y;
  }
}
template <typename T>
__global__ void __launch_bounds__(kRowThreads) column_join_kernel(const float* __restrict__ parts, T* __restrict__ out, int64_t cols, int runs) {
  const int64_t c = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < runs; ++k) s += __ldg(parts + k * cols + c);
  out[c] = from_float<T>(s);
}
// Runs of rows: four blocks for every SM, 64 rows at least.
int64_t sum_runs(int64_t rows, int64_t cols) {
  const int64_t blocks = (cols + kSumColumns - 1) / kSumColumns;
  int64_t k = ((int64_t)device_info().sm_count * 4 + blocks - 1) / blocks;
  if (k > (rows + 63) / 64) k = (rows + 63) / 64;
  return k < 1 ? 1 : k;
}
template <typename T> int column_sums(const void* x, void* out, float* parts, int64_t rows, int64_t cols, cudaStream_t s) {
  const int64_t blocks = (cols + kSumColumns - 1) / kSumColumns, runs = sum_runs(rows, cols), run = (rows + runs - 1) / runs;
  if (blocks * runs > 0x7fffffff) return ACTNN_ERR_SHAPE;
  auto* kernel = cols % 8 == 0 && aligned(x, 16) ? column_sums_kernel<T, true> : column_sums_kernel<T, false>;
  kernel<<<(unsigned)(blocks * runs), kRowThreads, 0, s>>>((const T*)x, parts, rows, cols, run);
  column_join_kernel<T><<<(unsigned)((cols + kRowThreads - 1) / kRowThreads), kRowThreads, 0, s>>>(parts, (T*)out, cols, (int)runs);
  return check_launch();
}

template <typename T>
int encode(const void* x, int8_t* codes, float* scale, int64_t rows, int64_t cols, int64_t ldx, int64_t ldc, cudaStream_t s) {
  const bool vec = cols % 8 == 0 && ldx % 8 == 0 && aligned(x, 16);
  // as few threads a row as hold it: 32 elements each
  const int lanes = cols <= 1024 ? 32 : cols <= 2048 ? 64 : cols <= 4096 ? 128 : 256;
  const int64_t per = kRowThreads / lanes, grid = (rows + per - 1) / per;
  if (grid > 0x7fffffff) return ACTNN_ERR_SHAPE;
  auto* kernel = lanes == 32 ? (vec ? row_codes_kernel<T, 32, true> : row_codes_kernel<T, 32, false>)
                 : lanes == 64 ? (vec ? row_codes_kernel<T, 64, true> : row_codes_kernel<T, 64, false>)
                 : lanes == 128 ? (vec ? row_codes_kernel<T, 128, true> : row_codes_kernel<T, 128, false>)
                                : (vec ? row_codes_kernel<T, 256, true> : row_codes_kernel<T, 256, false>);
  kernel<<<(unsigned)grid, kRowThreads, 0, s>>>((const T*)x, codes, scale, rows, cols, ldx, ldc);
  return check_launch();
}
template <typename T>
int decode(const int8_t* codes, const float* scale, void* out, int64_t rows, int64_t cols, int64_t ldc, cudaStream_t s) {
  const bool vec = cols % 8 == 0 && ldc % 8 == 0 && aligned(codes, 8) && aligned(out, 16);
  const int64_t octs = (cols + 7) / 8, grid = (rows * octs + kRowThreads - 1) / kRowThreads;
  if (grid > 0x7fffffff) return ACTNN_ERR_SHAPE;
  auto* kernel = vec ? row_decode_kernel<T, true> : row_decode_kernel<T, false>;
  kernel<<<(unsigned)grid, kRowThreads, 0, s>>>(codes, scale, (T*)out, rows, cols, ldc, octs);
  return check_launch();
}

}  // namespace
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_row_codes(const void* x, int8_t* codes, float* scale, int64_t rows, int64_t cols, int64_t ldx, int64_t ldc,
                               int dtype, actnn_stream_t stream) {
  if (rows < 0 || cols < 0 || cols > ((int64_t)1 << 31) || rows > ((int64_t)1 << 40) || (rows > 1 && ldx < cols) || ldc < cols ||
      ldc % 16 != 0 || ldc - cols >= 16) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (rows == 0 || cols == 0) return ACTNN_OK;
  if (!x || !codes || !scale) return ACTNN_ERR_NULL;
  if (!aligned(x, dtype_size(dtype)) || !aligned(codes, 16) || !aligned(scale, 4)) return ACTNN_ERR_ALIGN;
  switch (dtype) {
    case ACTNN_F32: return encode<float>(x, codes, scale, rows, cols, ldx, ldc, (cudaStream_t)stream);
    case ACTNN_F16: return encode<__half>(x, codes, scale, rows, cols, ldx, ldc, (cudaStream_t)stream);
    default: return encode<__nv_bfloat16>(x, codes, scale, rows, cols, ldx, ldc, (cudaStream_t)stream);
  }
}

extern "C" int actnn_row_decode(const int8_t* codes, const float* scale, void* out, int64_t rows, int64_t cols, int64_t ldc,
                                int dtype, actnn_stream_t stream) {
  if (rows < 0 || cols < 0 || cols > ((int64_t)1 << 31) || rows > ((int64_t)1 << 40) || (rows > 1 && ldc < cols)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (rows == 0 || cols == 0) return ACTNN_OK;
  if (!codes || !scale || !out) return ACTNN_ERR_NULL;
  if (!aligned(out, dtype_size(dtype)) || !aligned(scale, 4)) return ACTNN_ERR_ALIGN;
  switch (dtype) {
    case ACTNN_F32: return decode<float>(codes, scale, out, rows, cols, ldc, (cudaStream_t)stream);
    case ACTNN_F16: return decode<__half>(codes, scale, out, rows, cols, ldc, (cudaStream_t)stream);
    default: return decode<__nv_bfloat16>(codes, scale, out, rows, cols, ldc, (cudaStream_t)stream);
  }
}

extern "C" int actnn_column_sums_workspace(int64_t rows, int64_t cols, int64_t* bytes) {
  if (!bytes) return ACTNN_ERR_NULL;
  if (rows < 0 || cols < 0 || cols > ((int64_t)1 << 31) || rows > ((int64_t)1 << 40)) return ACTNN_ERR_SHAPE;
  *bytes = sum_runs(rows, cols < 1 ? 1 : cols) * cols * (int64_t)sizeof(float);
  return ACTNN_OK;
}

extern "C" int actnn_column_sums(const void* x, void* out, int64_t rows, int64_t cols, int dtype, void* workspace,
                                 int64_t workspace_bytes, actnn_stream_t stream) {
  if (rows < 0 || cols < 0 || cols > ((int64_t)1 << 31) || rows > ((int64_t)1 << 40)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (cols == 0) return ACTNN_OK;
  const int size = dtype_size(dtype);
  if (!out || (rows > 0 && (!x || !workspace))) return ACTNN_ERR_NULL;
  if (!aligned(out, size) || !aligned(x, size) || !aligned(workspace, 4)) return ACTNN_ERR_ALIGN;
  if (rows == 0) return cudaMemsetAsync(out, 0, cols * size, (cudaStream_t)stream) == cudaSuccess ? ACTNN_OK : ACTNN_ERR_LAUNCH;
  if (workspace_bytes < sum_runs(rows, cols) * cols * (int64_t)sizeof(float)) return ACTNN_ERR_CAPACITY;
  switch (dtype) {
    case ACTNN_F32: return column_sums<float>(x, out, (float*)workspace, rows, cols, (cudaStream_t)stream);
    case ACTNN_F16: return column_sums<__half>(x, out, (float*)workspace, rows, cols, (cudaStream_t)stream);
    default: return column_sums<__nv_bfloat16>(x, out, (float*)workspace, rows, cols, (cudaStream_t)stream);
  }
}
