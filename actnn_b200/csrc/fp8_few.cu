// A linear layer in 8-bit floating point: tokens x [T, K] of a floating type by a weight kept as codes [N, K] with its scales.
//
// Up to eight tokens (a serving loop's step) are one launch.  The weight is what has to be read, once; every block makes the tokens'
// codes for itself, behind its own first weight loads.  A block has 16 channels, its warps the reduction's blocks of 128 in turn.  The sums
// of a block are four matrix instructions of 16 channels by 8 tokens by 32 values: an instruction's lanes may hold any 32 values as
// long as both operands agree, so a lane's 16 bytes of a row of the weight are its operand as they are loaded.  The scales multiply the
// sums of a block, the warps' sums are joined in order.  More tokens are two launches: codes of the rows into the workspace, then the
// product on the tensor memory's pipeline.  One f16 token by 2048 x 4096: 4.8 us, of which the weight's bytes are 1.3 at the copy rate; the
// rest is the launch, the coding of the token and one way to memory.
#include "fp8.cuh"

namespace actnn {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewTokens = 8;
constexpr int kFewChannels = 16;
constexpr int kFewAhead = 4;                            // blocks of 128 of its rows that a warp has under way
constexpr int kFewSmem = 40 * 1024;                     // codes of all tokens and their scales: with the joined sums within what needs no opt-in

// Bytes between the codes of two tokens: whole blocks, and 64 so that two tokens' 64 bytes lie in different banks.
static inline int few_stride(int64_t K) { return (int)((K + 127) / 128 * 128 + 64); }
static inline int64_t few_bytes(int64_t T, int64_t K) { return T * (few_stride(K) + (K + 511) / 512 * 4); }

// 16 bytes of a row at k, zeros from K on; nothing behind K is read.
ACTNN_DEV uint4 weight_bytes(const uint8_t* row, int k, int K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k + 16 <= K) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + k));
  } else if (k < K) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K) w[i / 4] |= load_one(row + k + i) << (8 * (i % 4));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
// c += A B of 16 channels by 8 tokens by 32 values.
ACTNN_DEV void mma16x8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// v * 2^e, e the sum of two scales' exponents: in two steps, each a factor that is a normal number.
ACTNN_DEV float scaled(float v, uint32_t byte_a, uint32_t byte_b) {
  const int e = (int)(byte_a + byte_b) - 254, half = e >> 1;
  return v * __uint_as_float((uint32_t)(half + 127) << 23) * __uint_as_float((uint32_t)(e - half + 127) << 23);
}

template <typename T>
__global__ void __launch_bounds__(kFewThreads)
fp8_few_kernel(const T* __restrict__ x, const uint8_t* __restrict__ weights, const uint8_t* __restrict__ scales, const T* __restrict__ bias,
               T* __restrict__ out, int tokens, int64_t N, int K, int64_t ldx, int64_t ldw, int stride, bool vec) {
  extern __shared__ uint4 dynamic_s[];                  // [token][stride] codes, [token][groups] words of scales
  __shared__ float sum_s[kFewWarps][kFewChannels * kFewTokens];
  uint8_t* codes_s = reinterpret_cast<uint8_t*>(dynamic_s);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int blocks = (K + kFpBlock - 1) / kFpBlock, groups = (blocks + 3) / 4;
  uint32_t* scale_s = reinterpret_cast<uint32_t*>(codes_s + tokens * stride);
  const int64_t n0 = (int64_t)blockIdx.x * kFewChannels, tiles = (N + 127) / 128;
  const int64_t row[2] = {min(n0 + g, N - 1), min(n0 + g + 8, N - 1)};          // rows behind the last are computed as it, and not written
  uint4 w[kFewAhead][2][2];                             // [block][row][half]
  auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int k = (first + i * kFewWarps) * kFpBlock + q * 16;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        w[i][r][0] = weight_bytes(weights + row[r] * ldw, k, K);
        w[i][r][1] = weight_bytes(weights + row[r] * ldw, k + 64, K);
      }
    }
  };
  load(warp);

  // ---- codes of the tokens: a warp takes 512 values of one
  for (int task = warp; task < tokens * groups; task += kFewWarps) {
    const int t = task / groups, j = task - t * groups;
    const T* p = x + t * ldx;
    Vec<T, 8> v[2];
    uint32_t byte[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) v[k] = vec ? fp8_load<T, true>(p, j * 512 + k * 256 + lane * 8, K) : fp8_load<T, false>(p, j * 512 + k * 256 + lane * 8, K);
    fp8_block_bits(v[0], v[1], byte);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = j * 512 + k * 256 + lane * 8;
      byte[k] = fp8_scale_byte(byte[k]);
      if (e < stride - 64) *reinterpret_cast<uint2*>(codes_s + t * stride + e) = fp8_codes8(v[k], fp8_factor(byte[k]));
    }
    const uint32_t mine = byte[0] | byte[1] << 16, other = __shfl_xor_sync(kFull, mine, 16);
    if (lane == 0) scale_s[t * groups + j] = mine | other << 8;
  }
  __syncthreads();

  // ---- sums: channels g and g + 8, tokens 2 q and 2 q + 1
  const uint8_t* token_scale = reinterpret_cast<const uint8_t*>(scale_s);
  const int t0 = min(2 * q, tokens - 1), t1 = min(2 * q + 1, tokens - 1);
  float acc[4] = {};
  for (int first = warp; first < blocks; first += kFewAhead * kFewWarps) {
    if (first != warp) load(first);
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int b = first + i * kFewWarps;
      if (b >= blocks) break;
      uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
      if (g < tokens) {
        const uint4* p = reinterpret_cast<const uint4*>(codes_s + g * stride + b * kFpBlock + q * 16);
        lo = p[0], hi = p[4];
      }
      float c[4] = {};
      mma16x8(c, w[i][0][0].x, w[i][1][0].x, w[i][0][0].y, w[i][1][0].y, lo.x, lo.y);
      mma16x8(c, w[i][0][0].z, w[i][1][0].z, w[i][0][0].w, w[i][1][0].w, lo.z, lo.w);
      mma16x8(c, w[i][0][1].x, w[i][1][1].x, w[i][0][1].y, w[i][1][1].y, hi.x, hi.y);
      mma16x8(c, w[i][0][1].z, w[i][1][1].z, w[i][0][1].w, w[i][1][1].w, hi.z, hi.w);
      const uint32_t s0 = __ldg(scales + fp8_scale_at(row[0], b, tiles)), s1 = __ldg(scales + fp8_scale_at(row[1], b, tiles));
      const uint32_t u0 = token_scale[t0 * groups * 4 + b], u1 = token_scale[t1 * groups * 4 + b];
      acc[0] += scaled(c[0], s0, u0);
      acc[1] += scaled(c[1], s0, u1);
      acc[2] += scaled(c[2], s1, u0);
      acc[3] += scaled(c[3], s1, u1);
    }
  }
  // [token][channel]
  sum_s[warp][2 * q * kFewChannels + g] = acc[0];
  sum_s[warp][(2 * q + 1) * kFewChannels + g] = acc[1];
  sum_s[warp][2 * q * kFewChannels + g + 8] = acc[2];
  sum_s[warp][(2 * q + 1) * kFewChannels + g + 8] = acc[3];
  __syncthreads();
  const int t = threadIdx.x / kFewChannels;
  const int64_t n = n0 + threadIdx.x % kFewChannels;
  if (t < tokens && n < N) {
    float s = sum_s[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < kFewWarps; ++k) s += sum_s[k][threadIdx.x];
    out[t * N + n] = from_float<T>(s + (bias ? to_float(bias[n]) : 0.f));
  }
}

bool few_tokens(int64_t T, int64_t K) { return T <= kFewTokens && few_bytes(T, K) <= kFewSmem; }
int64_t code_bytes(int64_t T, int64_t K) { return (T * fp8_row_bytes(K) + 255) / 256 * 256; }

template <typename T>
int few(const void* x, const uint8_t* weights, const uint8_t* scales, const void* bias, void* out, int64_t tokens, int64_t N, int64_t K,
        int64_t ldx, int64_t ldw, cudaStream_t s) {
  const bool vec = K % 8 == 0 && (ldx % 8 == 0 || tokens == 1) && aligned(x, 16);
  fp8_few_kernel<T><<<(unsigned)((N + kFewChannels - 1) / kFewChannels), kFewThreads, (size_t)few_bytes(tokens, K), s>>>(
      (const T*)x, weights, scales, (const T*)bias, (T*)out, (int)tokens, N, (int)K, ldx, ldw, few_stride(K), vec);
  return check_launch();
}

}  // namespace
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_fp8_linear_workspace(int64_t T, int64_t K, int64_t* bytes) {
  if (!bytes) return ACTNN_ERR_NULL;
  if (T < 0 || K < 1 || K > 0x7fffff00 || T > 0x7fffff00) return ACTNN_ERR_SHAPE;
  *bytes = few_tokens(T, K) ? 0 : code_bytes(T, K) + fp8_scale_bytes(T, K);
  return ACTNN_OK;
}

extern "C" int actnn_fp8_linear(const void* x, const uint8_t* weights, const uint8_t* weight_scales, const void* bias, void* out, int64_t T,
                                int64_t N, int64_t K, int64_t ldx, int64_t ldw, int dtype, void* workspace, int64_t workspace_bytes,
                                actnn_stream_t stream) {
  if (T < 0 || N < 0 || K < 1 || K > 0x7fffff00 || T > 0x7fffff00 || N > 0x7fffff00 || (T > 1 && ldx < K) || ldw < K ||
      ldw > ((int64_t)1 << 39)) return ACTNN_ERR_SHAPE;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (T == 0 || N == 0) return ACTNN_OK;
  if (!x || !weights || !weight_scales || !out) return ACTNN_ERR_NULL;
  const int size = dtype_size(dtype);
  if (!aligned(x, size) || !aligned(bias, size) || !aligned(out, size) || !aligned(weight_scales, 16) || !aligned(weights, 16) ||
      ldw % 16 != 0) return ACTNN_ERR_ALIGN;
  if (!few_tokens(T, K)) {
    const int64_t codes = code_bytes(T, K);
    if (!workspace) return ACTNN_ERR_NULL;
    if (!aligned(workspace, 16)) return ACTNN_ERR_ALIGN;
    if (workspace_bytes < codes + fp8_scale_bytes(T, K)) return ACTNN_ERR_CAPACITY;
    uint8_t *c = (uint8_t*)workspace, *s = c + codes;
    if (int st = actnn_fp8_row_codes(x, c, s, T, K, ldx, fp8_row_bytes(K), dtype, stream)) return st;
    return fp8_matmul_impl(c, s, weights, weight_scales, bias, out, T, N, K, fp8_row_bytes(K), ldw, dtype, true, stream);
  }
  const cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case ACTNN_F32: return few<float>(x, weights, weight_scales, bias, out, T, N, K, ldx, ldw, s);
    case ACTNN_F16: return few<__half>(x, weights, weight_scales, bias, out, T, N, K, ldx, ldw, s);
    default: return few<__nv_bfloat16>(x, weights, weight_scales, bias, out, T, N, K, ldx, ldw, s);
  }
}
