// Dropout without a mask: the backward pass draws the fields of the forward pass again (dropout.cuh), so both are this one kernel and
// nothing of an element is kept.  16384 x 8192 bf16: 84 us each way, the copy rate (82).
#include "dropout.cuh"

namespace actnn {
namespace {

constexpr int kDropThreads = 256;

// A thread has OCTS octets, kDropThreads apart.
template <typename T, int OCTS>
__global__ void __launch_bounds__(kDropThreads)
seeded_dropout_kernel(const T* __restrict__ x, T* __restrict__ y, int64_t numel, const DropKey drop) {
  const int64_t first = (int64_t)blockIdx.x * (kDropThreads * OCTS) + threadIdx.x;
  Vec<T, 8> v[OCTS];
#pragma unroll
  for (int k = 0; k < OCTS; ++k) {
    const int64_t e = (first + k * kDropThreads) * 8;
    if (e + 8 <= numel) {
      v[k] = load_vec<T, 8>(x + e);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(v[k].w)[i] = e + i < numel ? load_one(x + e + i) : from_float<T>(0.f);
    }
  }
  const NoiseKey key = drop_key(drop);
#pragma unroll
  for (int k = 0; k < OCTS; ++k) {
    const int64_t oct = first + k * kDropThreads, e = oct * 8;
    if (e >= numel) continue;
    float2 f[4];
    unpack_vec(v[k], f);
    drop_oct(f, noise_call(key, (uint64_t)oct), drop.least, drop.inv);
    if (e + 8 <= numel) {
      store_vec<T, 8, true>(y + e, f);
    } else {
      for (int i = 0; i < 8; ++i)
        if (e + i < numel) y[e + i] = from_float<T>(i & 1 ? f[i / 2].y : f[i / 2].x);
    }
  }
}

__global__ void philox_state_kernel(const int64_t* seed, const int64_t* offset, uint64_t more, int64_t* state) {
  state[0] = *seed;
  state[1] = (int64_t)((uint64_t)*offset + more);
}

template <typename T> int seeded_dropout(const void* x, void* y, int64_t numel, const DropKey& drop, cudaStream_t s) {
  constexpr int kMany = sizeof(T) == 4 ? 2 : 4;
  const int64_t octs = (numel + 7) / 8;
  const int each = octs >= (int64_t)device_info().sm_count * 2048 * kMany ? kMany : 1;
  const int64_t grid = (octs + kDropThreads * each - 1) / (kDropThreads * each);
  if (grid > 0x7fffffff) return ACTNN_ERR_SHAPE;
  (each > 1 ? seeded_dropout_kernel<T, kMany> : seeded_dropout_kernel<T, 1>)<<<(unsigned)grid, kDropThreads, 0, s>>>((const T*)x, (T*)y, numel, drop);
  return check_launch();
}

}  // namespace
}  // namespace actnn

using namespace actnn;

extern "C" int actnn_seeded_dropout(const void* x, void* y, int64_t numel, float p, int dtype, uint64_t seed, uint64_t offset,
                                    const int64_t* state, actnn_stream_t stream) {
  if (numel < 0) return ACTNN_ERR_SHAPE;
  if (!(p >= 0.f && p < 1.f)) return ACTNN_ERR_ARG;
  if (dtype < ACTNN_F32 || dtype > ACTNN_BF16) return ACTNN_ERR_DTYPE;
  if (numel == 0) return ACTNN_OK;
  if (!x || !y) return ACTNN_ERR_NULL;
  if (!aligned(x, 16) || !aligned(y, 16) || !aligned(state, 16)) return ACTNN_ERR_ALIGN;
  const DropKey drop = make_drop_key(p, seed, offset, state);
  switch (dtype) {
    case ACTNN_F32: return seeded_dropout<float>(x, y, numel, drop, (cudaStream_t)stream);
    case ACTNN_F16: return seeded_dropout<__half>(x, y, numel, drop, (cudaStream_t)stream);
    default: return seeded_dropout<__nv_bfloat16>(x, y, numel, drop, (cudaStream_t)stream);
  }
}

extern "C" int actnn_philox_state(const int64_t* seed, const int64_t* offset, uint64_t more, int64_t* state, actnn_stream_t stream) {
  if (!seed || !offset || !state) return ACTNN_ERR_NULL;
  if (!aligned(seed, 8) || !aligned(offset, 8) || !aligned(state, 16)) return ACTNN_ERR_ALIGN;
  philox_state_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(seed, offset, more, state);
  return check_launch();
}
