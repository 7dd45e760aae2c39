// A linear layer in 8-bit integers: tokens x [T, K] of a floating type by a weight kept as codes [N, K].
//
// Up to eight tokens (a serving loop's step) are one launch.  The weight is what has to be read, N * K bytes once, and every
// block needs all tokens' codes, so every block makes them again for itself: K elements a token from the L2, behind the
// block's own first weight loads, which are requested before.  A warp takes rows of the weight, two at a time; a lane multiplies
// 16 bytes of a row with the same place of each token by four-way integer dot products, and the 32 partial sums of a
// (row, token) are one redux instruction.  More tokens are two launches: codes of the rows into the workspace, then the
// product on the tensor cores.
//
// Measured on a B200: 1 x 2048 x 4096 4.0 us of which about 2 are the launch (1.3 for the weight's bytes), 1 x 8192 x 8192 14.2 (10.3).
#include "activation.cuh"

namespace actnn {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewTokens = 8;
constexpr int kFewRows = 2;                             // rows of the weight a warp has under way
constexpr int kFewAhead = 4;                            // pieces of 512 bytes of each that are requested at a time
constexpr int kFewSmem = 48 * 1024 - 512;               // codes of all tokens: what needs no opt-in, less a piece for `most_s` beside them

// 16 bytes of a row at `k`, zeros from K on; nothing behind K is read.
ACTNN_DEV uint4 weight_piece(const int8_t* row, int k, int K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k + 16 <= K) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + k));
  } else if (k < K) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K) w[i / 4] |= (uint32_t)__ldg(reinterpret_cast<const uint8_t*>(row) + k + i) << (8 * (i % 4));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}

// Eight elements that are read again soon: through the L1.
template <typename T> ACTNN_DEV Vec<T, 8> load_again(const T* p) {
  Vec<T, 8> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
    r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
  }
  return r;
}

// TOK: tokens the registers hold, T <= TOK.  Codes of a token in shared memory: `pieces` * 512 bytes, zeros from K on.
template <typename T, int TOK>
__global__ void __launch_bounds__(kFewThreads)
int8_few_kernel(const T* __restrict__ x, const int8_t* __restrict__ weights, const float* __restrict__ channel_scale,
                const T* __restrict__ bias, T* __restrict__ out, int tokens, int64_t N, int K, int64_t ldx, int64_t ldw, int pieces,
                bool vec) {
  extern __shared__ uint4 codes_s[];                    // [token][piece][lane]
  __shared__ uint32_t most_s[TOK];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t step = (int64_t)gridDim.x * kFewWarps * kFewRows;
  int64_t n = ((int64_t)blockIdx.x * kFewWarps + warp) * kFewRows;

  uint4 w[kFewRows][kFewAhead];                         // the first pieces, on their way while the tokens are coded
#pragma unroll
  for (int r = 0; r < kFewRows; ++r)
#pragma unroll
    for (int p = 0; p < kFewAhead; ++p)
      w[r][p] = n + r < N ? weight_piece(weights + (n + r) * ldw, p * 512 + lane * 16, K) : make_uint4(0, 0, 0, 0);

  // ---- codes: kFewThreads / TOK threads a token
  constexpr int kTeam = kFewThreads / TOK;
  const int t = threadIdx.x / kTeam, member = threadIdx.x % kTeam;
  if (threadIdx.x < TOK) most_s[threadIdx.x] = 0;
  __syncthreads();
  const T* p = x + t * ldx;
  auto load = [&](int e) {
    if (vec && e + 8 <= K) return load_again<T>(p + e);
    Vec<T, 8> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(v.w)[i] = e + i < K ? __ldg(p + e + i) : from_float<T>(0.f);
    return v;
  };
  if (t < tokens) {
    uint32_t most = 0;
#pragma unroll 8
    for (int e = member * 8; e < K; e += kTeam * 8) most = max(most, most_of(load(e)));
    most = __reduce_max_sync(kFull, most);
    if (lane == 0) atomicMax(&most_s[t], most);
  }
  __syncthreads();
  if (t < tokens) {
    const float inv = code_factor(largest(most_s[t]));
    int8_t* q = reinterpret_cast<int8_t*>(codes_s) + (size_t)t * pieces * 512;
#pragma unroll 4
    for (int e = member * 8; e < pieces * 512; e += kTeam * 8) {
      float2 f[4];
      unpack_vec(load(e), f);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = code_bits(f[i], make_float2(inv, inv));
      store_codes<8>(q + e, f);
    }
  }
  __syncthreads();

  // ---- products
  const float token_scale = lane < tokens ? code_step(largest(most_s[lane < TOK ? lane : 0])) : 0.f;
  for (bool first = true; n < N; n += step, first = false) {
    int acc[kFewRows][TOK] = {};
    for (int base = 0; base < pieces; base += kFewAhead) {
      if (!first || base > 0) {
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
#pragma unroll
          for (int q = 0; q < kFewAhead; ++q)
            w[r][q] = n + r < N ? weight_piece(weights + (n + r) * ldw, (base + q) * 512 + lane * 16, K) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int q = 0; q < kFewAhead; ++q) {
        if (base + q >= pieces) break;
#pragma unroll
        for (int k = 0; k < TOK; ++k) {
          if (k >= tokens) break;
          const uint4 c = codes_s[((size_t)k * pieces + base + q) * 32 + lane];
#pragma unroll
          for (int r = 0; r < kFewRows; ++r) {
            acc[r][k] = __dp4a((int)w[r][q].x, (int)c.x, acc[r][k]);
            acc[r][k] = __dp4a((int)w[r][q].y, (int)c.y, acc[r][k]);
            acc[r][k] = __dp4a((int)w[r][q].z, (int)c.z, acc[r][k]);
            acc[r][k] = __dp4a((int)w[r][q].w, (int)c.w, acc[r][k]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
      int mine = 0;
#pragma unroll
      for (int k = 0; k < TOK; ++k) {
        if (k >= tokens) break;
        const int sum = __reduce_add_sync(kFull, acc[r][k]);
        if (lane == k) mine = sum;
      }
      if (lane < tokens && n + r < N) {
        const float b = bias ? to_float(bias[n + r]) : 0.f;
        out[lane * N + n + r] = from_float<T>(fmaf((float)mine * token_scale, __ldg(channel_scale + n + r), b));
      }
    }
  }
}

struct FewCall {
  const void* x;
  const int8_t* weights;
  const float* channel_scale;
  const void* bias;
  void* out;
  int tokens, K, pieces;
  int64_t N, ldx, ldw;
  bool vec;
  cudaStream_t stream;
};
template <typename T, int TOK> int few(const FewCall& c) {
  auto* kernel = int8_few_kernel<T, TOK>;
  const size_t smem = (size_t)c.tokens * c.pieces * 512;
  const int64_t needed = (c.N + kFewWarps * kFewRows - 1) / (kFewWarps * kFewRows), most = (int64_t)device_info().sm_count * 4;
  kernel<<<(unsigned)(needed < most ? needed : most), kFewThreads, smem, c.stream>>>(
      (const T*)c.x, c.weights, c.channel_scale, (const T*)c.bias, (T*)c.out, c.tokens, c.N, c.K, c.ldx, c.ldw, c.pieces, c.vec);
  return check_launch();
}
template <typename T> int few_typed(const FewCall& c) {
  return c.tokens == 1 ? few<T, 1>(c) : c.tokens == 2 ? few<T, 2>(c) : c.tokens <= 4 ? few<T, 4>(c) : few<T, 8>(c);
}

// One launch for one token, and for up to eight while coding them in every block costs less than a launch of its own.  Measured,
// one launch against two, us, at N = 4096: K = 2048, 8 tokens 7.2 / 7.8; K = 4096, 1 token 6.1 / 10.6, 4 tokens 8.9 / 10.6, 8 tokens
// 11.5 / 10.6; N = K = 8192, 1 token 14.2 / 18.2, 2 tokens 20.5 / 18.2.
bool few_tokens(int64_t T, int64_t K) {
  return T <= kFewTokens && T * ((K + 511) / 512 * 512) <= kFewSmem && (T == 1 || (K <= 4096 && T * K <= 16384));
}
int64_t row_bytes(int64_t K) { return (K + 15) / 16 * 16; }

}  // namespace
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_int8_linear_workspace(int64_t T, int64_t K, int64_t* bytes) {
  if (!bytes) return ACTNN_ERR_NULL;
  if (T < 0 || K < 1 || K > 131072 || T > 0x7fffff00) return ACTNN_ERR_SHAPE;
  *bytes = few_tokens(T, K) ? 0 : T * row_bytes(K) + T * (int64_t)sizeof(float);
  return ACTNN_OK;
}

extern "C" int actnn_int8_linear(const void* x, const int8_t* weights, const float* channel_scale, const void* bias, void* out,
                                 int64_t T, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int dtype, void* workspace,
                                 int64_t workspace_bytes, actnn_stream_t stream) {
  if (T < 0 || N < 0 || K < 1 || K > 131072 || T > 0x7fffff00 || N > 0x7fffff00 || (T > 1 && ldx < K) || ldw < K ||
      ldw > ((int64_t)1 << 39)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (T == 0 || N == 0) return ACTNN_OK;
  if (!x || !weights || !channel_scale || !out) return ACTNN_ERR_NULL;
  const int size = dtype_size(dtype);
  if (!aligned(x, size) || !aligned(bias, size) || !aligned(out, size) || !aligned(channel_scale, 4) || !aligned(weights, 16) ||
      ldw % 16 != 0) return ACTNN_ERR_ALIGN;
  if (!few_tokens(T, K)) {
    const int64_t codes = T * row_bytes(K);
    if (!workspace) return ACTNN_ERR_NULL;
    if (!aligned(workspace, 16)) return ACTNN_ERR_ALIGN;
    if (workspace_bytes < codes + T * (int64_t)sizeof(float)) return ACTNN_ERR_CAPACITY;
    int8_t* c = (int8_t*)workspace;
    float* s = (float*)(c + codes);
    if (int st = actnn_row_codes(x, c, s, T, K, ldx, row_bytes(K), dtype, stream)) return st;
    return int8_matmul_impl(c, s, weights, channel_scale, bias, out, T, N, K, row_bytes(K), ldw, dtype, true, stream);
  }
  FewCall c{x, weights, channel_scale, bias, out, (int)T, (int)K, (int)((K + 511) / 512), N, ldx, ldw,
            ldx % 8 == 0 && aligned(x, 16), (cudaStream_t)stream};
  if (T == 1) c.vec = aligned(x, 16);
  switch (dtype) {
    case ACTNN_F32: return few_typed<float>(c);
    case ACTNN_F16: return few_typed<__half>(c);
    default: return few_typed<__nv_bfloat16>(c);
  }
}
