// Activation functions whose backward pass reads an 8-bit copy of the input.
//
//   forward   y = f(x)                codes, scale <- x               (gated: y = f(gate) * up, codes of both)
//   backward  dx = dy * f'(x^)        x^ = code * scale               (gated: dgate = dy * up^ * f'(gate^), dup = dy * f(gate^))
//
// A scale belongs to 256 consecutive elements of the output (of each half, in the gated form), whatever the rows are: a warp
// holds them, eight a lane, so the range is one redux instruction and the input is read once.  Bound by HBM: 2 + 2 + 1 bytes an
// element each way for 16-bit types, 4 + 2 + 2 gated.  With `codes` NULL the input itself is what the backward pass reads.
//
// Measured on a B200: GELU (tanh) of 8192 x 4096 float16 31 us forward and 29 back (26 each at the copy rate of 6.5 TB/s), SiLU-gated
// 16384 x 4096 bfloat16 93 and 80 (82 each); rows of 4097 columns, which no vector fits, take 1.8 times their bytes' time.
#include "activation.cuh"

namespace actnn {
namespace {

constexpr int kActThreads = 256;
constexpr int kActWarps = kActThreads / 32;

// Where the inputs of eight consecutive outputs lie.  The gated input is [rows, 2 * cols]: gate, then up.
struct GluShape {
  FastDiv oct_cols;      // cols / 8, vector form
  int64_t cols;
};
template <bool GATED> ACTNN_DEV int64_t input_of_oct(int64_t oct, const GluShape& g) {
  if constexpr (!GATED) return oct * 8;
  return (oct + (int64_t)fast_div((uint32_t)oct, g.oct_cols) * g.oct_cols.d) * 8;
}

ACTNN_DEV void codes_of(const float2 (&f)[4], uint32_t most, int8_t* codes, float* scale, int lane) {
  const float a = largest(__reduce_max_sync(kFull, most));
  const float inv = code_factor(a);
  float2 c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = code_bits(f[i], make_float2(inv, inv));
  store_codes<8>(codes, c);
  if (lane == 0) *scale = code_step(a);
}

// Eight elements, or the first `count` of them and zeros.
template <typename T> ACTNN_DEV Vec<T, 8> load_some(const T* p, int count) {
  if (count >= 8) return load_vec<T, 8>(p);
  Vec<T, 8> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(r.w)[i] = i < count ? p[i] : from_float<T>(0.f);
  return r;
}
template <typename T, bool STREAM> ACTNN_DEV void store_some(T* p, int count, const float2 (&f)[4]) {
  if (count >= 8) {
    store_vec<T, 8, STREAM>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < count) p[i] = from_float<T>(i & 1 ? f[i / 2].y : f[i / 2].x);
  }
}

// One warp per block of 256 outputs.  Every lane of a warp takes part in the reductions; codes are written for whole blocks
// (the buffer is a multiple of 256), zeros behind the end.
template <typename T, int KIND, bool GATED, bool SAVE>
__global__ void __launch_bounds__(kActThreads)
act_forward_kernel(const T* __restrict__ x, T* __restrict__ y, int8_t* __restrict__ codes, float* __restrict__ scale,
                   int64_t numel, int64_t blocks, const GluShape g) {
  constexpr bool P = sizeof(T) == 4;
  const int lane = threadIdx.x & 31;
  const int64_t b = (int64_t)blockIdx.x * kActWarps + (threadIdx.x >> 5);
  if (b >= blocks) return;
  const int64_t oct = b * 32 + lane;
  const int64_t left = numel - oct * 8;
  const int count = left >= 8 ? 8 : left > 0 ? (int)left : 0;
  float2 f[4], u[4], out[4];
  const int64_t at = count > 0 ? input_of_oct<GATED>(oct, g) : 0;
  const Vec<T, 8> fv = load_some(x + at, count), uv = GATED ? load_some(x + at + g.cols, count) : fv;
  unpack_vec(fv, f);
  if constexpr (GATED) unpack_vec(uv, u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i] = act_value<KIND, P>(f[i]);
    if constexpr (GATED) out[i] = f_mul(out[i], u[i]);
  }
  if (count > 0) store_some<T, false>(y + oct * 8, count, out);
  if constexpr (SAVE) {
    codes_of(f, most_of(fv), codes + oct * 8, scale + b, lane);
    if constexpr (GATED) codes_of(u, most_of(uv), codes + (blocks * 32 + oct) * 8, scale + blocks + b, lane);
  }
}

template <typename T, int KIND, bool GATED, bool CODES>
__global__ void __launch_bounds__(kActThreads)
act_backward_kernel(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                    const float* __restrict__ scale, T* __restrict__ dx, int64_t numel, int64_t blocks, const GluShape g) {
  constexpr bool P = sizeof(T) == 4;
  const int lane = threadIdx.x & 31;
  const int64_t b = (int64_t)blockIdx.x * kActWarps + (threadIdx.x >> 5);
  if (b >= blocks) return;
  const int64_t oct = b * 32 + lane;
  const int64_t left = numel - oct * 8;
  if (left <= 0) return;
  const int count = left >= 8 ? 8 : (int)left;
  const int64_t at = input_of_oct<GATED>(oct, g);
  float2 f[4], u[4], d[4], df[4], du[4];
  const Vec<T, 8> dv = load_some(dy + oct * 8, count);
  if constexpr (CODES) {
    const Codes<8> cf = load_codes<8>(codes + oct * 8), cu = GATED ? load_codes<8>(codes + (blocks * 32 + oct) * 8) : cf;
    const float sf = __ldg(scale + b), su = GATED ? __ldg(scale + blocks + b) : sf;
    unpack_codes(cf, f);
    if constexpr (GATED) unpack_codes(cu, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = f_mul(f[i], make_float2(sf, sf));
      if constexpr (GATED) u[i] = f_mul(u[i], make_float2(su, su));
    }
  } else {
    const Vec<T, 8> fv = load_some(x + at, count), uv = GATED ? load_some(x + at + g.cols, count) : fv;
    unpack_vec(fv, f);
    if constexpr (GATED) unpack_vec(uv, u);
  }
  unpack_vec(dv, d);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 value;
    df[i] = f_mul(d[i], act_slope<KIND, P>(f[i], GATED ? &value : nullptr));
    if constexpr (GATED) {
      df[i] = f_mul(df[i], u[i]);
      du[i] = f_mul(d[i], value);
    }
  }
  // evict-first stores: 16384 x 4096 gated bfloat16 81.3 -> 77.9 us; the output of the forward pass gains nothing by them
  store_some<T, true>(dx + at, count, df);
  if constexpr (GATED) store_some<T, true>(dx + at + g.cols, count, du);
}

// The gated form where a row is not a whole number of aligned vectors: element j * 32 + lane of a block is the lane's j-th, so
// that a warp's loads of one element each are consecutive.
template <typename T, int KIND, bool SAVE>
__global__ void __launch_bounds__(kActThreads)
glu_forward_any_kernel(const T* __restrict__ x, T* __restrict__ y, int8_t* __restrict__ codes, float* __restrict__ scale,
                       int64_t numel, int64_t blocks, int64_t cols) {
  constexpr bool P = sizeof(T) == 4;
  const int lane = threadIdx.x & 31;
  const int64_t b = (int64_t)blockIdx.x * kActWarps + (threadIdx.x >> 5);
  if (b >= blocks) return;
  const int64_t first = b * 256 + lane;
  int64_t row = first / cols, col = first - row * cols;
  float f[8], u[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = first + 32 * j < numel;
    const T* p = x + row * 2 * cols + col;
    f[j] = in ? to_float(p[0]) : 0.f;
    u[j] = in ? to_float(p[cols]) : 0.f;
    if (in) y[first + 32 * j] = from_float<T>(act_value<KIND, P>(f[j]) * u[j]);
    for (col += 32; col >= cols; col -= cols) ++row;
  }
  if constexpr (SAVE) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, abs_bits(half ? u[j] : f[j]));
      const float a = largest(__reduce_max_sync(kFull, most)), inv = code_factor(a);
      int8_t* c = codes + (half * blocks + b) * 256 + lane;
#pragma unroll
      for (int j = 0; j < 8; ++j) c[32 * j] = (int8_t)__float_as_uint(code_bits(half ? u[j] : f[j], inv));
      if (lane == 0) scale[half * blocks + b] = code_step(a);
    }
  }
}

template <typename T, int KIND, bool CODES>
__global__ void __launch_bounds__(kActThreads)
glu_backward_any_kernel(const T* __restrict__ dy, const T* __restrict__ x, const int8_t* __restrict__ codes,
                        const float* __restrict__ scale, T* __restrict__ dx, int64_t numel, int64_t blocks, int64_t cols) {
  constexpr bool P = sizeof(T) == 4;
  const int lane = threadIdx.x & 31;
  const int64_t b = (int64_t)blockIdx.x * kActWarps + (threadIdx.x >> 5);
  if (b >= blocks) return;
  const int64_t first = b * 256 + lane;
  int64_t row = first / cols, col = first - row * cols;
  const float sf = CODES ? __ldg(scale + b) : 1.f, su = CODES ? __ldg(scale + blocks + b) : 1.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (first + 32 * j < numel) {
      const int64_t at = row * 2 * cols + col;
      float f, u;
      if constexpr (CODES) {
        f = (float)codes[b * 256 + lane + 32 * j] * sf;
        u = (float)codes[(blocks + b) * 256 + lane + 32 * j] * su;
      } else {
        f = to_float(x[at]);
        u = to_float(x[at + cols]);
      }
      const float d = to_float(dy[first + 32 * j]);
      float value;
      dx[at] = from_float<T>(d * act_slope<KIND, P>(f, &value) * u);
      dx[at + cols] = from_float<T>(d * value);
    }
    for (col += 32; col >= cols; col -= cols) ++row;
  }
}

struct ActCall {
  const void *x, *dy;
  void* out;
  int8_t* codes;
  float* scale;
  int64_t rows, cols, numel, blocks;
  bool gated, forward, vectors;
  cudaStream_t stream;
};

template <typename T, int KIND> int launch(const ActCall& c) {
  const unsigned grid = (unsigned)((c.blocks + kActWarps - 1) / kActWarps);
  const GluShape g{make_fast_div(c.gated && c.vectors ? (uint32_t)(c.cols / 8) : 1u), c.cols};
  const T *x = (const T*)c.x, *dy = (const T*)c.dy;
  T* out = (T*)c.out;
  const bool with = c.codes != nullptr;
#define ACT_FORWARD(GATED, SAVE) \
  act_forward_kernel<T, KIND, GATED, SAVE><<<grid, kActThreads, 0, c.stream>>>(x, out, c.codes, c.scale, c.numel, c.blocks, g)
#define ACT_BACKWARD(GATED, CODES) \
  act_backward_kernel<T, KIND, GATED, CODES><<<grid, kActThreads, 0, c.stream>>>(dy, x, c.codes, c.scale, out, c.numel, c.blocks, g)
  if (c.gated && !c.vectors) {
    if (c.forward) {
      if (with) glu_forward_any_kernel<T, KIND, true><<<grid, kActThreads, 0, c.stream>>>(x, out, c.codes, c.scale, c.numel, c.blocks, c.cols);
      else glu_forward_any_kernel<T, KIND, false><<<grid, kActThreads, 0, c.stream>>>(x, out, c.codes, c.scale, c.numel, c.blocks, c.cols);
    } else {
      if (with) glu_backward_any_kernel<T, KIND, true><<<grid, kActThreads, 0, c.stream>>>(dy, x, c.codes, c.scale, out, c.numel, c.blocks, c.cols);
      else glu_backward_any_kernel<T, KIND, false><<<grid, kActThreads, 0, c.stream>>>(dy, x, c.codes, c.scale, out, c.numel, c.blocks, c.cols);
    }
  } else if (c.gated) {
    if (c.forward) { if (with) ACT_FORWARD(true, true); else ACT_FORWARD(true, false); }
    else { if (with) ACT_BACKWARD(true, true); else ACT_BACKWARD(true, false); }
  } else {
    if (c.forward) { if (with) ACT_FORWARD(false, true); else ACT_FORWARD(false, false); }
    else { if (with) ACT_BACKWARD(false, true); else ACT_BACKWARD(false, false); }
  }
#undef ACT_FORWARD
#undef ACT_BACKWARD
  return check_launch();
}

template <typename T> int launch_kind(int kind, const ActCall& c) {
  switch (kind) {
    case kActNone: return launch<T, kActNone>(c);
    case kActRelu: return launch<T, kActRelu>(c);
    case kActSilu: return launch<T, kActSilu>(c);
    case kActGelu: return launch<T, kActGelu>(c);
    default: return launch<T, kActGeluTanh>(c);
  }
}

// Checks what both directions share and launches.  `io`: pointers of activations that the vector form reads 16 bytes at a time.
int act_call(ActCall& c, int gated, int kind, int dtype, const void* const* io, int n_io) {
  if (c.rows < 0 || c.cols < 0 || (c.cols > 0 && c.rows > ((int64_t)1 << 40) / c.cols)) return ACTNN_ERR_SHAPE;
  if (kind < 0 || kind >= kActKinds || gated < 0 || gated > 1) return ACTNN_ERR_ARG;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  c.numel = c.rows * c.cols;
  c.blocks = (c.numel + 255) / 256;
  c.gated = gated != 0;
  if (c.numel == 0) return ACTNN_OK;
  bool wide = true, typed = true;
  for (int i = 0; i < n_io; ++i) {
    if (!io[i]) return ACTNN_ERR_NULL;
    wide = wide && aligned(io[i], 16);
    typed = typed && aligned(io[i], dtype_size(dtype));
  }
  if (!typed) return ACTNN_ERR_ALIGN;
  if ((c.codes == nullptr) != (c.scale == nullptr)) return ACTNN_ERR_NULL;
  if (c.codes && (!aligned(c.codes, 8) || !aligned(c.scale, 4))) return ACTNN_ERR_ALIGN;
  if (c.blocks / kActWarps > 0x7ffffff0) return ACTNN_ERR_SHAPE;
  c.vectors = wide && c.cols % 8 == 0 && c.numel / 8 < 0x7fffffff;
  if (!c.gated) {
    if (!wide) return ACTNN_ERR_ALIGN;
    c.vectors = true;
  }
  switch (dtype) {
    case ACTNN_F32: return launch_kind<float>(kind, c);
    case ACTNN_F16: return launch_kind<__half>(kind, c);
    default: return launch_kind<__nv_bfloat16>(kind, c);
  }
}

}  // namespace
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_act_forward(const void* x, void* y, int8_t* codes, float* scale, int64_t rows, int64_t cols, int gated,
                                 int kind, int dtype, actnn_stream_t stream) {
  ActCall c{};
  c.x = x; c.out = y; c.codes = codes; c.scale = scale; c.rows = rows; c.cols = cols; c.forward = true;
  c.stream = (cudaStream_t)stream;
  const void* io[2] = {x, y};
  return act_call(c, gated, kind, dtype, io, 2);
}

extern "C" int actnn_act_backward(const void* grad_y, const void* x, const int8_t* codes, const float* scale, void* grad_x,
                                  int64_t rows, int64_t cols, int gated, int kind, int dtype, actnn_stream_t stream) {
  ActCall c{};
  c.x = x; c.dy = grad_y; c.out = grad_x; c.codes = (int8_t*)codes; c.scale = (float*)scale; c.rows = rows; c.cols = cols;
  c.stream = (cudaStream_t)stream;
  const void* io[3] = {grad_y, grad_x, codes ? grad_y : x};
  return act_call(c, gated, kind, dtype, io, 3);
}
